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


def cuts(*args, **kw):
    """(runs of dq, runs of dk and dv, blocks of kept keys, their runs)"""
    plan = vjp_plan(*args, **kw)
    return tuple(int(x) for x in re.search(
        r"attention_dq\(dim=\d+,splits=(\d+)\)\+attention_dkv\(dim=\d+,splits=(\d+),kept=(\d+)x(\d+)\)",
        plan).groups())


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
def test_no_more_runs_than_there_are_tiles(dtype):
    # one tile of rows and of keys: one run, and nothing to sum
    for args in ((1, 4, 4, 1, 1, 64), (1, 32, 32, 16, 16, 128), (2, 8, 4, 7, 90, 256)):
        assert vjp_plan(*args, dtype=dtype).endswith("splits=1,kept=0x1)"), args
    # 64 rows or keys a run, the last one's excepted: a tile, or two of 32
    for args in ((1, 16, 16, 128, 128, 64), (1, 4, 1, 100, 100, 128), (1, 1, 1, 1000, 1000, 96),
                 (1, 8, 2, 3000, 3000, 64), (1, 2, 2, 200, 5000, 128)):
        for window, keep in ((1 << 30, 0), (64, 0), (200, 40)):
            dq, dkv, blocks, kept = cuts(*args, window=window, keep=keep, dtype=dtype)
            rows = args[1] // args[2] * args[3]
            assert dq == 1 or 64 * dq <= min(args[4], window + keep + 128)
            assert dkv == 1 or 64 * (dkv - 1) < min(rows, (window + 128) * args[1] // args[2])
            assert kept == 1 or 64 * (kept - 1) < rows


@pytest.mark.parametrize("B, Hq, Hkv, D, L, window, keep, dtype", (
    (1, 32, 8, 128, 8192, 64, 8192, BF16), (8, 32, 8, 128, 8192, 64, 4096, BF16),
    (8, 32, 32, 128, 8192, 128, 2048, BF16), (1, 32, 32, 128, 32768, 1024, 16384, F16),
    (4, 16, 16, 256, 4096, 100, 1000, F32), (1, 8, 1, 64, 20000, 256, 9000, BF16),
    (1, 64, 8, 128, 4096, 256, 4, BF16), (2, 28, 4, 128, 3000, 1 << 30, 0, F16)))
def test_the_sums_parts_are_bounded(B, Hq, Hkv, D, L, window, keep, dtype):
    """Parts are made for workgroups that fill the card, so there are at most as many as it takes
    twice over (1024 workgroups, each with the sums of 128 keys or rows, where there are parts)."""
    size = _lib.load().mlxrocm_window_attention_vjp_workspace_size(
        B, Hq, Hkv, L, L, D, window, keep, dtype)
    delta = 4 * B * Hq * L + 256
    of_keys, of_rows = 2 * 1024 * 128 * 2 * D * 4, 2 * 1024 * 128 * D * 4
    # (and the blocks of keys that are not kept have theirs)
    assert size <= delta + 2 * of_keys + of_rows


def test_float32_takes_the_cus_once():
    """A CU holds one workgroup of the kernel for few rows in float32."""
    for B, Hq, Hkv, D, Lq, Lk in ((3, 32, 8, 128, 1, 4600), (7, 32, 4, 128, 1, 2600),
                                  (1, 8, 2, 80, 100, 2200), (1, 4, 1, 128, 100, 1500),
                                  (100, 32, 8, 64, 1, 900)):
        rc, plan = _lib.attention_plan(B, Hq, Hkv, Lq, Lk, D, dtype=F32)
        rows, splits = re.match(r"attention_few\(dim=\d+,rows=(\d+),splits=(\d+)\)", plan).groups()
        blocks = -(-(Hq // Hkv * Lq) // int(rows)) * B * Hkv
        assert int(splits) == 1 or int(splits) * blocks <= 256
    # much work of many workgroups is the tiles'
    assert _lib.attention_plan(1, 8, 8, 1000, 1000, 80, dtype=F32)[1].startswith("attention_rows")
    assert _lib.attention_plan(1, 16, 16, 512, 512, 80, dtype=F32)[1].startswith("attention_few")
