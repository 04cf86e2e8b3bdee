"""window_attention and paged_attention against the formulas in 64 bits, and the gradients
against theirs and against differences."""
import math

import pytest
import torch

import mlx_amd
from tests.attention_util import check, pages_of, reference, tensors

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16

# (B, Hq, Hkv, D, Lq, Lk, window, keep, lengths): head sizes and shared heads, one token to many,
# windows, kept tokens, ragged lengths, rows that see nothing
SHAPES = (
    (1, 4, 4, 64, 1, 1, None, 0, None),
    (2, 8, 2, 128, 1, 77, None, 0, [77, 5]),
    (3, 4, 1, 80, 1, 300, 100, 3, [300, 0, 101]),
    (2, 6, 6, 40, 3, 130, 16, 1, [130, 2]),
    (1, 7, 1, 128, 5, 1000, 300, 70, None),       # 35 rows
    (2, 16, 2, 96, 8, 333, None, 0, [333, 8]),    # 64 rows
    (1, 2, 1, 256, 9, 65, 33, 0, None),
    (2, 8, 2, 64, 100, 100, None, 0, None),
    (2, 4, 2, 128, 129, 257, 64, 5, [257, 100]),  # padding in front
    (1, 3, 3, 8, 65, 65, 1, 0, None),             # each token sees itself alone
    (1, 4, 1, 136, 200, 200, 90, 200, None),      # everything is kept
    (2, 2, 2, 256, 70, 90, 17, 2, [90, 0]),
    (1, 5, 1, 96, 333, 500, 128, 40, None),
    (1, 1, 1, 80, 200, 7, None, 0, None),         # more queries than keys
)


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("shape", SHAPES)
def test_window_attention(gpu, shape, dtype):
    B, Hq, Hkv, D, Lq, Lk, window, keep, lengths = shape
    q, k, v = tensors(B, Hq, Hkv, D, Lq, Lk, dtype, gpu, seed=D + Lk)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=gpu)
    out = mlx_amd.window_attention(q, k, v, scale=D ** -0.5, window=window, keep=keep, lengths=n)
    assert out.dtype == dtype and out.stride() == q.stride()
    want, bound = reference(q, k, v, D ** -0.5, window, keep, lengths)
    check(out, want["out"], bound["out"], "out")


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("shape", SHAPES)
def test_gradients(gpu, shape, dtype):
    B, Hq, Hkv, D, Lq, Lk, window, keep, lengths = shape
    q, k, v, do = tensors(B, Hq, Hkv, D, Lq, Lk, dtype, gpu, seed=D + Lk, grad=True)
    for x in (q, k, v):
        x.requires_grad_()
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=gpu)
    out = mlx_amd.window_attention(q, k, v, scale=D ** -0.5, window=window, keep=keep, lengths=n)
    grads = torch.autograd.grad(out, (q, k, v), do)
    want, bound = reference(q, k, v, D ** -0.5, window, keep, lengths, do)
    check(out.detach(), want["out"], bound["out"], "out")
    for name, x, of in zip(("dq", "dk", "dv"), grads, (q, k, v)):
        assert x.dtype == dtype and x.shape == of.shape
        check(x, want[name], bound[name], name)


def test_gradients_against_differences(gpu):
    """(f(x + h d) - f(x - h d)) / 2h along random directions, f = sum(out * do) in 64 bits.
    float32 results are off by some 2^-22 each (scores of a few units), so f by about
    sqrt(n) 2^-22 with n results of unit size times do, the quotient by that over h; the
    third derivative leaves h^2 times a few."""
    B, Hq, Hkv, D, Lq, Lk = 2, 4, 2, 64, 90, 120
    q, k, v, do = tensors(B, Hq, Hkv, D, Lq, Lk, F32, gpu, seed=5, grad=True)
    lengths = torch.tensor([120, 60], dtype=torch.int32, device=gpu)
    args = dict(scale=D ** -0.5, window=50, keep=4, lengths=lengths)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(mlx_amd.window_attention(*leaves, **args), leaves, do)
    h = 1e-2
    noise = 8 * math.sqrt(do.numel()) * 2.0 ** -22 / h
    g = torch.Generator(device=gpu).manual_seed(9)
    for i in range(3):
        d = torch.randn(leaves[i].shape, generator=g, device=gpu)
        ends = []
        for sign in (1, -1):
            x = [q, k, v]
            x[i] = x[i] + sign * h * d
            ends.append((mlx_amd.window_attention(*x, **args).double() * do).sum())
        got = (grads[i].double() * d).sum()
        want = (ends[0] - ends[1]) / (2 * h)
        size = (grads[i].double() * d).square().sum().sqrt()
        assert abs(float(got - want)) <= noise + 10 * h * h * float(size) + 1e-3 * float(size)


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("page", (16, 48, 128))
@pytest.mark.parametrize("shape", SHAPES)
def test_paged_attention(gpu, shape, dtype, page):
    """Against the formulas; and bit for bit what window_attention gives on the same keys where
    the two are cut alike (they are when the tables have room for the keys alone)."""
    B, Hq, Hkv, D, Lq, Lk, window, keep, lengths = shape
    q, k, v = tensors(B, Hq, Hkv, D, Lq, Lk, dtype, gpu, seed=D + Lk)
    k_pages, v_pages, table = pages_of(k, v, page, fill=math.nan)
    n = torch.tensor(lengths or [Lk] * B, dtype=torch.int32, device=gpu)
    args = dict(scale=-0.7 * D ** -0.5, window=window, keep=keep)
    out = mlx_amd.paged_attention(q, k_pages, v_pages, table, n, **args)
    assert out.dtype == dtype and out.stride() == q.stride()
    want, bound = reference(q, k, v, args["scale"], window, keep, lengths)
    check(out, want["out"], bound["out"], "out")


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("Lq", (1, 6, 40))
def test_split_over_the_cache(gpu, Lq, dtype):
    """Few rows over a long cache: many runs of keys, joined; lengths far below the table's."""
    B, Hq, Hkv, D, Lk = 2, 8, 2, 128, 9000
    q, k, v = tensors(B, Hq, Hkv, D, Lq, Lk, dtype, gpu, seed=3)
    lengths = [9000, 700]
    n = torch.tensor(lengths, dtype=torch.int32, device=gpu)
    k_pages, v_pages, table = pages_of(k, v, 64, fill=math.inf)
    for window, keep in ((None, 0), (3000, 10), (100, 0)):
        args = dict(scale=D ** -0.5, window=window, keep=keep)
        want, bound = reference(q, k, v, D ** -0.5, window, keep, lengths)
        out = mlx_amd.paged_attention(q, k_pages, v_pages, table, n, **args)
        check(out, want["out"], bound["out"], f"paged, window {window}")
        out = mlx_amd.window_attention(q, k, v, lengths=n, **args)
        check(out, want["out"], bound["out"], f"contiguous, window {window}")


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("value", (math.nan, math.inf, -math.inf))
@pytest.mark.parametrize("Lq, D", ((3, 128), (150, 64), (150, 256), (20, 96)))
def test_what_is_not_seen_does_not_reach_a_row(gpu, Lq, D, value, dtype):
    """Bit for bit the result with zeros in those places, forward and backward: keys past a
    sequence's length, keys before every window, and keys and rows that others see."""
    B, Hq, Hkv, Lk, window = 2, 4, 2, 160, 24
    lengths = [160, 100]
    n = torch.tensor(lengths, dtype=torch.int32, device=gpu)
    q, k, v, do = tensors(B, Hq, Hkv, D, Lq, Lk, dtype, gpu, seed=1, grad=True)
    # key 95 of sequence 0 and all from 100 on of sequence 1 are spoilt
    spoilt = [x.clone() for x in (k, v)]
    clean = [x.clone() for x in (k, v)]
    for x, fill in ((spoilt, value), (clean, 0.0)):
        for t in x:
            t[0, :, 95] = fill
            t[1, :, 100:] = fill
            t[1, :, 0] = fill if Lq < 70 else t[1, :, 0]  # before every window
    results = []
    for kv in (spoilt, clean):
        leaves = [x.clone().requires_grad_() for x in (q, *kv)]
        out = mlx_amd.window_attention(*leaves, scale=D ** -0.5, window=window, lengths=n)
        results.append((out.detach(), *torch.autograd.grad(out, leaves, do)))
        page = pages_of(*kv, 16, fill=value)
        results[-1] += (mlx_amd.paged_attention(q, *page, n, scale=D ** -0.5, window=window),)
    p = torch.arange(Lq, device=gpu) + 160 - Lq
    sees = (p >= 95) & (p - 95 < window)  # rows of sequence 0 that see key 95
    for i in (0, 1, 4):  # out, dq, and out over pages
        a, b = results[0][i], results[1][i]
        assert torch.equal(a[1], b[1]), i
        assert torch.equal(a[0][:, ~sees], b[0][:, ~sees]), i
        assert not torch.isfinite(a[0][:, sees].float()).all() or not sees.any()
    # keys that no row that sees key 95 sees: before the window of the first, after the last
    first, last = max(95, 160 - Lq), min(159, 95 + window - 1)
    j = torch.arange(Lk, device=gpu)
    apart = (j <= first - window) | (j > last)
    for i in (2, 3):  # dk, dv
        a, b = results[0][i], results[1][i]
        assert torch.equal(a[1], b[1]), i
        assert torch.equal(a[0][:, apart], b[0][:, apart]), i


def test_rows_that_are_not_finite_reach_their_keys_alone(gpu):
    """The same for q and dout: padding in front, and rows that a key is not seen by."""
    B, Hq, Hkv, D, L, window = 2, 4, 1, 128, 200, 20
    n = torch.tensor([200, 120], dtype=torch.int32, device=gpu)
    q, k, v, do = tensors(B, Hq, Hkv, D, L, L, BF16, gpu, seed=2, grad=True)
    results = []
    for fill in (math.nan, 0.0):
        x, y = q.clone(), do.clone()
        for t in (x, y):
            t[0, :, 90] = fill
            t[1, :, :80] = fill
        leaves = [t.clone().requires_grad_() for t in (x, k, v)]
        out = mlx_amd.window_attention(*leaves, scale=D ** -0.5, window=window, lengths=n)
        results.append((out.detach(), *torch.autograd.grad(out, leaves, y)))
    j = torch.arange(L, device=gpu)
    apart = (j > 90) | (j <= 90 - window)
    for i in range(4):
        a, b = results[0][i], results[1][i]
        assert torch.equal(a[1], b[1]), i
        rows = j != 90 if i < 2 else apart
        assert torch.equal(a[0][:, rows], b[0][:, rows]), i


def test_strides_and_broadcasts(gpu):
    """Slices of one fused projection, a sliced token dimension, expanded keys (whose gradient is
    the sum over what they were expanded to), unaligned and mixed types."""
    B, L, Hq, Hkv, D = 2, 70, 4, 2, 64
    g = torch.Generator(device=gpu).manual_seed(0)
    fused = torch.randn((B, L, (Hq + 2 * Hkv) * D), generator=g, device=gpu).to(BF16)
    q, k, v = (x.unflatten(-1, (-1, D)).transpose(1, 2)
               for x in fused.split((Hq * D, Hkv * D, Hkv * D), -1))
    args = dict(scale=0.1, window=30, keep=2)
    dense = mlx_amd.window_attention(*(x.contiguous() for x in (q, k, v)), **args)
    assert torch.equal(mlx_amd.window_attention(q, k, v, **args), dense)
    every = mlx_amd.window_attention(q[:, :, ::2], k, v, **args)
    assert torch.equal(every, mlx_amd.window_attention(q[:, :, ::2].contiguous(), k, v, **args))
    off = torch.empty(q.numel() + 1, dtype=BF16, device=gpu)[1:].view(q.shape).copy_(q)
    assert off.data_ptr() % 16 and torch.equal(mlx_amd.window_attention(off, k, v, **args), dense)
    last = q.transpose(2, 3).contiguous().transpose(2, 3)  # the head dimension is strided
    assert torch.equal(mlx_amd.window_attention(last, k, v, **args), dense)
    # one key head and one batch for all
    k1, v1 = (x[:1, :1].clone().requires_grad_() for x in (k, v))
    out = mlx_amd.window_attention(q, k1.expand(B, Hkv, L, D), v1.expand(B, Hkv, L, D), **args)
    do = torch.randn(out.shape, generator=g, device=gpu).to(BF16)
    dk1, dv1 = torch.autograd.grad(out, (k1, v1), do)
    k2, v2 = (x.detach().expand(B, Hkv, L, D).contiguous().requires_grad_() for x in (k1, v1))
    dk2, dv2 = torch.autograd.grad(mlx_amd.window_attention(q, k2, v2, **args), (k2, v2), do)
    for a, b in ((dk1, dk2), (dv1, dv2)):
        assert torch.equal(a, b.sum((0, 1), keepdim=True))
    # a gradient that is itself expanded, and a type of each operand's own
    leaf = q.float().requires_grad_()
    out = mlx_amd.window_attention(leaf, k, v, **args)
    assert out.dtype == F32
    (dq,) = torch.autograd.grad(out.sum(), leaf)
    want, bound = reference(leaf, k.float(), v.float(), **args,
                            dout=torch.ones_like(out))
    check(dq, want["dq"], bound["dq"], "dq")


def test_offsets_beyond_32_bits(gpu):
    """Pages whose elements lie past 2^32 bytes and 2^31 elements."""
    Hkv, page, D = 2, 64, 128
    pages = (1 << 31) // (Hkv * page * D) + 200
    k_pages, v_pages = (torch.empty((pages, Hkv, page, D), dtype=BF16, device=gpu)
                        for _ in range(2))
    q, k, v = tensors(1, 4, Hkv, D, 2, 600, BF16, gpu, seed=8)
    table = torch.arange(pages - 1, pages - 11, -1, dtype=torch.int32, device=gpu)[None]
    n = torch.tensor([600], dtype=torch.int32, device=gpu)
    mlx_amd.paged_cache_update(k, v, k_pages, v_pages, table, n)
    want, bound = reference(q, k, v, 0.1, 500, 3)
    out = mlx_amd.paged_attention(q, k_pages, v_pages, table, n, scale=0.1, window=500, keep=3)
    check(out, want["out"], bound["out"], "few rows")
    q = tensors(1, 4, Hkv, D, 100, 600, BF16, gpu, seed=9)[0]
    want, bound = reference(q, k, v, 0.1, 500, 3)
    out = mlx_amd.paged_attention(q, k_pages, v_pages, table, n, scale=0.1, window=500, keep=3)
    check(out, want["out"], bound["out"], "many rows")


@pytest.mark.parametrize("Lq", (1, 100))
def test_large_scores_and_scales(gpu, Lq):
    """Scores of hundreds, where the maximum moves; scale zero; a negative one."""
    B, Hq, Hkv, D, Lk = 1, 4, 2, 64, 500
    q, k, v = tensors(B, Hq, Hkv, D, Lq, Lk, F32, gpu, seed=4)
    k = k * torch.linspace(0.1, 4, Lk, device=gpu)[None, None, :, None]
    for scale in (1.0, -1.0, 0.0, 0.125):
        out = mlx_amd.window_attention(q, k, v, scale=scale)
        want, bound = reference(q, k, v, scale)
        check(out, want["out"], bound["out"], f"scale {scale}")


def test_replays_from_a_graph_and_on_another_stream(gpu):
    """One step of decoding, captured: the cache's update and the attention over it."""
    B, Hq, Hkv, D, page = 2, 8, 2, 128, 32
    q, k, v = tensors(B, Hq, Hkv, D, 1, 3000, BF16, gpu, seed=6)
    k_pages, v_pages, table = pages_of(k, v, page)
    lengths = torch.tensor([2000, 150], dtype=torch.int32, device=gpu)
    new_k, new_v = (torch.empty((B, Hkv, 1, D), dtype=BF16, device=gpu) for _ in range(2))

    def step():
        mlx_amd.paged_cache_update(new_k, new_v, k_pages, v_pages, table, lengths)
        return mlx_amd.paged_attention(q, k_pages, v_pages, table, lengths, scale=0.1)

    new_k.normal_(), new_v.normal_()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step()
    for i in range(3):
        lengths += 1
        new_k.normal_(), new_v.normal_()
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        assert torch.equal(replayed, step()), i


def test_same_results_every_time(gpu):
    q, k, v, do = tensors(2, 8, 2, 64, 300, 300, BF16, gpu, seed=7, grad=True)
    first = None
    for _ in range(3):
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        out = mlx_amd.window_attention(*leaves, scale=0.2, window=100, keep=2)
        got = (out.detach(), *torch.autograd.grad(out, leaves, do))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_empty_and_refused(gpu):
    z = lambda *s, dtype=BF16: torch.zeros(s, dtype=dtype, device=gpu)  # noqa: E731
    ints = lambda *s: torch.zeros(s, dtype=torch.int32, device=gpu)  # noqa: E731
    assert mlx_amd.window_attention(z(0, 4, 3, 64), z(0, 2, 3, 64), z(0, 2, 3, 64), scale=1).shape == (0, 4, 3, 64)
    assert mlx_amd.window_attention(z(2, 4, 0, 64), z(2, 2, 3, 64), z(2, 2, 3, 64), scale=1).shape == (2, 4, 0, 64)
    q, k, v = (x.requires_grad_() for x in (z(2, 4, 3, 64), z(2, 2, 0, 64), z(2, 2, 0, 64)))
    out = mlx_amd.window_attention(q, k, v, scale=1)
    assert torch.equal(out, torch.zeros_like(out))
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    assert torch.equal(dq, torch.zeros_like(q)) and dk.shape == k.shape and dv.shape == v.shape
    out = mlx_amd.paged_attention(z(2, 4, 1, 64), z(3, 2, 16, 64), z(3, 2, 16, 64), ints(2, 0), ints(2), scale=1)
    assert torch.equal(out, torch.zeros_like(out))
    # entries of the table and lengths beyond what exists are brought back to it
    wild = torch.tensor([[7, -5], [1 << 30, 2]], dtype=torch.int32, device=gpu)
    long = torch.tensor([1000, -3], dtype=torch.int32, device=gpu)
    pages = torch.ones((3, 2, 16, 64), dtype=BF16, device=gpu)
    for Lq in (1, 100):
        out = mlx_amd.paged_attention(z(2, 4, Lq, 64), pages, pages, wild, long, scale=1)
        rows = torch.arange(Lq, device=gpu) >= Lq - 32
        assert (out[0][:, rows] == 1).all() and not out[0][:, ~rows].any() and not out[1].any()
    before = pages.clone()
    mlx_amd.paged_cache_update(z(2, 2, 1, 64), z(2, 2, 1, 64), pages, pages, wild, long)
    assert torch.equal(pages, before)
    x = z(1, 2, 16, 64).requires_grad_()
    with pytest.raises(NotImplementedError):
        mlx_amd.paged_attention(x, pages, pages, ints(1, 1), ints(1), scale=1)
    with pytest.raises(ValueError):  # pages that start off a 16-byte boundary
        off = torch.zeros(3 * 2 * 16 * 64 + 1, dtype=BF16, device=gpu)[1:].view(3, 2, 16, 64)
        mlx_amd.paged_attention(z(1, 2, 1, 64), off, off, ints(1, 1), ints(1), scale=1)
