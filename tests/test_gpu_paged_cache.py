"""paged_cache_update, against the same copies one row at a time."""
import pytest
import torch

import mlx_amd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("B, H, L, D, page, lengths", (
    (1, 8, 1, 128, 16, [1]),
    (3, 2, 1, 64, 48, [200, 49, 0]),
    (2, 3, 100, 80, 32, [100, 33]),     # padding in front
    (2, 1, 37, 8, 16, [90, 37]),
    (1, 2, 5, 256, 64, [66]),           # over the end of a page
))
def test_update(gpu, B, H, L, D, page, lengths, dtype):
    g = torch.Generator(device=gpu).manual_seed(L)
    rand = lambda *s: torch.randn(s, generator=g, device=gpu).to(dtype)  # noqa: E731
    k, v = (rand(B, L, H, D).transpose(1, 2) for _ in range(2))
    per = max(1, -(-max(lengths) // page))
    table = torch.randperm(B * per + 2, device=gpu, generator=g)[:B * per].reshape(B, per).int()
    both = rand(2, B * per + 2, H, page, D)
    want = both.clone()
    for b, n in enumerate(lengths):
        for i in range(L):
            p = n - L + i
            if p >= 0:
                for w, x in enumerate((k, v)):
                    want[w, table[b, p // page], :, p % page] = x[b, :, i]
    n = torch.tensor(lengths, dtype=torch.int64, device=gpu)  # any integers will do
    got = mlx_amd.paged_cache_update(k, v, both[0], both[1], table, n)
    assert got[0].data_ptr() == both[0].data_ptr() and got[1].data_ptr() == both[1].data_ptr()
    assert torch.equal(both, want)


def test_pages_may_be_strided(gpu):
    """Keys and values of a page side by side in one allocation, a table that is a slice."""
    cache = torch.zeros((6, 2, 4, 32, 64), dtype=torch.bfloat16, device=gpu)
    k, v = (torch.randn((1, 4, 40, 64), device=gpu).to(torch.bfloat16) for _ in range(2))
    table = torch.tensor([[9, 9], [5, 3]], dtype=torch.int32, device=gpu)[1:]
    n = torch.tensor([40], dtype=torch.int32, device=gpu)
    mlx_amd.paged_cache_update(k, v, cache[:, 0], cache[:, 1], table, n)
    for w, x in enumerate((k, v)):
        assert torch.equal(cache[5, w], x[0, :, :32]) and torch.equal(cache[3, w, :, :8], x[0, :, 32:])
    out = mlx_amd.paged_attention(k, cache[:, 0], cache[:, 1], table, n, scale=0.1)
    assert torch.equal(out, mlx_amd.window_attention(k, k, v, scale=0.1))
