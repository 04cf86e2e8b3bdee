"""How the gradients' sums of window_attention are cut and what that takes: no GPU."""
import re

import pytest

from mlx_amd import _lib

F32, F16, BF16 = 0, 1, 2


def vjp_plan(*args, **kw):
    rc, plan = _lib.attention_vjp_plan(*args, **kw)
    assert rc == 0
    return plan


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
def test_gradients_without_query_heads_are_written(dtype):
    assert "attention_dkv" in vjp_plan(1, 0, 4, 100, 100, 64, dtype=dtype)
    assert vjp_plan(1, 0, 0, 100, 100, 64, dtype=dtype) == ""
    assert vjp_plan(0, 4, 4, 100, 100, 64, dtype=dtype) == ""
