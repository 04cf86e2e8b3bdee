"""window_attention, paged_attention and the cache's update at edges: no query heads, gradients of
any size, tangents, the versions of what is written in place."""
import math

import pytest
import torch

import mlx_amd
from tests.attention_util import pages_of, tensors
from tests.test_gpu_attention import BF16, F16, F32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("Lq, Lk, D", ((3, 5, 64), (200, 300, 128), (0, 40, 96)))
def test_gradients_without_query_heads(gpu, Lq, Lk, D, dtype):
    """Keys and values that no query reads have gradients of zero."""
    q = torch.zeros((2, 0, Lq, D), dtype=dtype, device=gpu).requires_grad_()
    k, v = (torch.randn((2, 3, Lk, D), device=gpu).to(dtype).requires_grad_() for _ in range(2))
    out = mlx_amd.window_attention(q, k, v, scale=0.1)
    assert out.shape == q.shape
    # memory that the gradients would find if nothing wrote them
    for _ in range(4):
        torch.full((2, 3, Lk, D), math.nan, dtype=dtype, device=gpu)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), torch.zeros_like(out))
    assert dq.shape == q.shape and not dk.any() and not dv.any()
