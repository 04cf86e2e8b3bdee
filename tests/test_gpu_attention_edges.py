"""window_attention, paged_attention and the cache's update at edges: no query heads, gradients of
any size, tangents, the versions of what is written in place."""
import math

import pytest
import torch

import mlx_amd
from tests.attention_util import pages_of, tensors, visible
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


@pytest.mark.parametrize("size", (2.0 ** 11, 1.0, 1e-3, 1e-4, 1e-5))
@pytest.mark.parametrize("L, D, window", ((2048, 128, None), (300, 64, None), (1500, 96, 200),
                                          (700, 256, None)))
def test_gradients_of_any_size_in_float16(gpu, L, D, window, size):
    """In the mean as far off as with probabilities and their gradients rounded to eleven bits, the
    results to float16 (as in test_gpu_attention_tiles.py, with its tenth more): float16's few
    exponents may cost nothing beside.  2^11: gradients of the probabilities are beyond its range."""
    q, k, v, do = tensors(1, 4, 2, D, L, L, F16, gpu, seed=L, grad=True)
    do = (do.float() * size).to(F16)
    scale = D ** -0.5 if size <= 1 else D ** -1.5
    if size > 1:
        v = v * 16
    x, y, z, dout = (t.double() for t in (q, k, v, do))
    y, z = (t.repeat_interleave(2, 1) for t in (y, z))

    def eleven(t):  # bits
        m, e = torch.frexp(t)
        return torch.ldexp((m * 2048).round(), e - 11)

    seen = visible(L, L, [L], window, 0, gpu)
    p = torch.softmax((scale * x @ y.transpose(2, 3)).masked_fill(~seen, -math.inf), -1)
    exact_ds = p * (dout @ z.transpose(2, 3) - (dout * (p @ z)).sum(-1, keepdim=True))
    ds = eleven(p * (dout @ z.transpose(2, 3) - (dout * (eleven(p) @ z)).sum(-1, keepdim=True)))
    two = lambda t: t.unflatten(1, (2, 2)).sum(2)  # noqa: E731  (heads that share one)
    want = dict(dq=scale * exact_ds @ y, dk=two(scale * exact_ds.transpose(2, 3) @ x),
                dv=two(p.transpose(2, 3) @ dout))
    model = dict(dq=scale * ds @ y, dk=two(scale * ds.transpose(2, 3) @ x),
                 dv=two(eleven(p).transpose(2, 3) @ dout))
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = mlx_amd.window_attention(*leaves, scale=scale, window=window)
    for name, t in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, do)):
        off = float((t.double() - want[name]).norm())
        by_design = float((model[name].half().double() - want[name]).norm())
        assert by_design < math.inf
        assert off <= 1.1 * by_design, (name, off / by_design)


def test_forward_mode_is_refused(gpu):
    from torch.autograd import forward_ad

    q, k, v = tensors(2, 4, 2, 64, 3, 40, BF16, gpu)
    k_pages, v_pages, table = pages_of(k, v, 16)
    n = torch.tensor([40, 7], dtype=torch.int32, device=gpu)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for args in ((dual(q), k, v), (q, dual(k), v), (q.clone().requires_grad_(), k, dual(v))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                mlx_amd.window_attention(*args, scale=0.1)
        with pytest.raises(NotImplementedError, match="no gradients"):
            mlx_amd.paged_attention(dual(q), k_pages, v_pages, table, n, scale=0.1)
        with pytest.raises(NotImplementedError, match="no gradients"):
            mlx_amd.paged_cache_update(dual(k), v, k_pages, v_pages, table, n)
        mlx_amd.window_attention(q, k, v, scale=0.1)  # (what has no tangent is computed)


def test_an_update_is_seen_by_graphs(gpu):
    """Pages that a graph has saved have been written to when its gradients are wanted."""
    k, v = tensors(2, 4, 2, 64, 3, 40, BF16, gpu)[1:]
    n = torch.tensor([40, 7], dtype=torch.int32, device=gpu)
    for make in (lambda t: t, lambda t: t.long()):  # by the native host path, and not
        k_pages, v_pages, table = pages_of(k, v, 16)
        x = torch.ones((), dtype=BF16, device=gpu, requires_grad=True)
        saved = [(x * pages).sum() for pages in (k_pages, v_pages)]
        before = [pages._version for pages in (k_pages, v_pages)]
        mlx_amd.paged_cache_update(k, v, k_pages, v_pages, table, make(n))
        assert [pages._version for pages in (k_pages, v_pages)] == [b + 1 for b in before]
        for s in saved:
            with pytest.raises(RuntimeError, match="inplace"):
                s.backward()
    with torch.inference_mode():
        pages = [p.clone() for p in (k_pages, v_pages)]
        mlx_amd.paged_cache_update(k, v, *pages, table, n)
    mlx_amd.paged_cache_update(k, v, *pages, table, n)  # (these have no version)
    assert torch.equal(pages[0], k_pages) and torch.equal(pages[1], v_pages)


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("Lq, Lk, page, window, keep, lengths", (
    (1, 512, 16, None, 0, [512, 77]), (5, 960, 48, 300, 7, [960, 400]), (40, 2048, 128, 64, 0, [2048, 9]),
    (300, 768, 32, None, 0, [768, 300]), (500, 1024, 64, 200, 3, [1024, 1000])))
@pytest.mark.parametrize("D", (64, 96, 256))
def test_pages_give_the_bits_of_contiguous_keys(gpu, Lq, Lk, page, window, keep, lengths, D, dtype):
    """Where the table has room for these keys alone, so that both are cut alike."""
    q, k, v = tensors(2, 8, 2, D, Lq, Lk, dtype, gpu, seed=D + Lq)
    n = torch.tensor(lengths, dtype=torch.int32, device=gpu)
    args = dict(scale=D ** -0.5, window=window, keep=keep)
    out = mlx_amd.paged_attention(q, *pages_of(k, v, page, fill=math.nan), n, **args)
    assert torch.equal(out, mlx_amd.window_attention(q, k, v, lengths=n, **args))


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("fill", (math.nan, math.inf, -math.inf))
@pytest.mark.parametrize("D, keep", ((64, 0), (128, 3), (256, 0)))
def test_rows_that_are_not_finite_reach_their_keys_alone(gpu, D, keep, fill, dtype):
    """One row of q or of dout: the other rows' and the keys' that it does not see are what they are
    with zeros there, bit for bit (and finite)."""
    L, window = 300, 20
    q, k, v, do = tensors(1, 4, 2, D, L, L, dtype, gpu, seed=D, grad=True)
    j = torch.arange(L, device=gpu)
    apart = ((j > 90) | (j <= 90 - window)) & (j >= keep)
    for which in range(2):
        results = []
        for value in (fill, 0.0):
            x = [q.clone(), do.clone()]
            x[which][0, :, 90] = value
            leaves = [t.clone().requires_grad_() for t in (x[0], k, v)]
            out = mlx_amd.window_attention(*leaves, scale=D ** -0.5, window=window, keep=keep)
            results.append((out.detach(), *torch.autograd.grad(out, leaves, x[1])))
        for i, (a, b) in enumerate(zip(*results)):
            rows = j != 90 if i < 2 else apart
            assert torch.isfinite(a[:, :, rows].float()).all(), (which, i)
            assert torch.equal(a[:, :, rows], b[:, :, rows]), (which, i)
