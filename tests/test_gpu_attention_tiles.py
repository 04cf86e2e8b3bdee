"""The kernel of 128-row tiles at the small shapes of test_gpu_attention: as many copies of the batch
as it takes for that kernel to be the one that runs, one of them against the formulas, the others
against that one."""
import math

import pytest
import torch

import mlx_amd
from mlx_amd import _lib, ops
from tests.attention_util import check, pages_of, reference, tensors, visible
from tests.test_gpu_attention import BF16, F16, F32, SHAPES

pytestmark = pytest.mark.gpu


def copies_for_tiles(B, Hq, Hkv, Lq, Lk, D, window, keep, dtype):
    for n in (1, 4, 16, 64, 256, 1024):
        rc, plan = _lib.attention_plan(n * B, Hq, Hkv, Lq, Lk, D, window or 1 << 30, keep,
                                       ops._DTYPE_CODE[dtype])
        assert rc == 0
        if plan.startswith("attention_rows"):
            return n
    return 0


def test_there_are_shapes_for_both(gpu):
    n = [copies_for_tiles(*s[:3], s[4], s[5], s[3], s[6], s[7], F16) for s in SHAPES]
    assert 0 in n and sum(x > 0 for x in n) >= 8  # 16 rows at most are always few


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("shape", SHAPES)
def test_many_copies(gpu, shape, dtype):
    B, Hq, Hkv, D, Lq, Lk, window, keep, lengths = shape
    copies = copies_for_tiles(B, Hq, Hkv, Lq, Lk, D, window, keep, dtype)
    if copies == 0:
        copies = 3  # (the kernel for few rows)
    q, k, v = tensors(B, Hq, Hkv, D, Lq, Lk, dtype, gpu, seed=D + Lk)
    want, bound = reference(q, k, v, D ** -0.5, window, keep, lengths)
    n = torch.tensor(lengths or [Lk] * B, dtype=torch.int32, device=gpu)
    k_pages, v_pages, table = pages_of(k, v, 48, fill=math.nan)
    args = dict(scale=D ** -0.5, window=window, keep=keep)
    every = [x.repeat(copies, 1, 1, 1) for x in (q, k, v)]
    outs = (mlx_amd.window_attention(*every, lengths=n.repeat(copies), **args),
            mlx_amd.paged_attention(every[0], k_pages, v_pages, table.repeat(copies, 1),
                                    n.repeat(copies), **args))
    for out, what in zip(outs, ("contiguous", "paged")):
        out = out.unflatten(0, (copies, B))
        check(out[0], want["out"], bound["out"], what)
        assert torch.equal(out, out[:1].expand_as(out)), what


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("value", (math.nan, math.inf, -math.inf))
@pytest.mark.parametrize("Lq, D", ((150, 64), (150, 256), (20, 96), (150, 128)))
def test_what_is_not_seen_does_not_reach_a_row(gpu, Lq, D, value, dtype):
    B, Hq, Hkv, Lk, window = 2, 4, 2, 160, 24
    copies = max(1, copies_for_tiles(B, Hq, Hkv, Lq, Lk, D, window, 0, dtype))
    n = torch.tensor([160, 100], dtype=torch.int32, device=gpu).repeat(copies)
    q, k, v = tensors(B, Hq, Hkv, D, Lq, Lk, dtype, gpu, seed=1)
    results = []
    for fill in (value, 0.0):
        kv = [x.clone() for x in (k, v)]
        for t in kv:
            t[0, :, 95] = fill
            t[1, :, 100:] = fill
        k_pages, v_pages, table = pages_of(*kv, 16, fill=value)
        q_all, *kv = (x.repeat(copies, 1, 1, 1) for x in (q, *kv))
        args = dict(scale=D ** -0.5, window=window)
        results.append((
            mlx_amd.window_attention(q_all, *kv, lengths=n, **args),
            mlx_amd.paged_attention(q_all, k_pages, v_pages, table.repeat(copies, 1), n, **args)))
    p = torch.arange(Lq, device=gpu) + 160 - Lq
    sees = (p >= 95) & (p - 95 < window)  # rows of the first sequence that see key 95
    for a, b in zip(*results):
        a, b = a.unflatten(0, (copies, B)), b.unflatten(0, (copies, B))
        assert torch.equal(a[:, 1], b[:, 1])
        assert torch.equal(a[:, 0][:, :, ~sees], b[:, 0][:, :, ~sees])
        assert not sees.any() or not torch.isfinite(a[:, 0][:, :, sees].float()).any(-1).all()


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("keep", (5, 130))
def test_gradients_of_kept_keys(gpu, keep, dtype):
    """Keys that all rows see, whose sums are cut, beside keys whose are not."""
    B, Hq, Hkv, D, L, window = 2, 22, 11, 72, 1500, 64
    if dtype == F32:
        window = 40  # (168 rows of two heads: not cut either)
        Hq = 11
    rc, plan = _lib.attention_vjp_plan(B, Hq, Hkv, L, L, D, window, keep, ops._DTYPE_CODE[dtype])
    assert rc == 0 and "attention_dkv(dim=96,splits=1,kept=" in plan and plan.endswith("+attention_sum")
    q, k, v, do = tensors(B, Hq, Hkv, D, L, L, dtype, gpu, seed=6, grad=True)
    lengths = [L, 700]
    want, bound = reference(q, k, v, 0.1, window, keep, lengths, do)
    for x in (q, k, v):
        x.requires_grad_()
    n = torch.tensor(lengths, dtype=torch.int32, device=gpu)
    out = mlx_amd.window_attention(q, k, v, scale=0.1, window=window, keep=keep, lengths=n)
    for name, x in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), do)):
        check(x, want[name], bound[name], name)


@pytest.mark.parametrize("dtype", (F16, BF16))
@pytest.mark.parametrize("B, H, L, D, window", ((8, 8, 23, 64, None), (2, 4, 235, 80, None),
                                                (2, 4, 900, 128, 6), (16, 8, 3, 64, None)))
def test_gradients_of_tokens_that_see_few(gpu, B, H, L, D, window, dtype):
    """In the mean the gradients are as far off as the formulas are with those numbers rounded that
    the kernels round: probabilities, their gradients and the results (the result that delta is
    formed from is not).  A tenth more: the kernels round probabilities before they are divided
    by their sum, so the errors are others of the same size, and of three tokens not many."""
    q, k, v, do = tensors(B, H, H, D, L, L, dtype, gpu, seed=L, grad=True)
    want, _ = reference(q, k, v, D ** -0.5, window, 0, None, do)
    seen = visible(L, L, [L] * B, window, 0, gpu)
    x, y, z, dout = (t.double() for t in (q, k, v, do))
    rounded = lambda t: t.to(dtype).double()  # noqa: E731
    p = torch.softmax((D ** -0.5 * x @ y.transpose(2, 3)).masked_fill(~seen, -math.inf), -1)
    delta = (dout * (rounded(p) @ z)).sum(-1, keepdim=True)
    ds = rounded(p * (dout @ z.transpose(2, 3) - delta)) * D ** -0.5
    model = dict(dq=ds @ y, dk=ds.transpose(2, 3) @ x, dv=rounded(p).transpose(2, 3) @ dout)
    for t in (q, k, v):
        t.requires_grad_()
    out = mlx_amd.window_attention(q, k, v, scale=D ** -0.5, window=window)
    for name, t in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), do)):
        off = float((t.double() - want[name]).norm())
        by_design = float((rounded(model[name]) - want[name]).norm())
        assert off <= 1.1 * by_design, (name, off / by_design)


def test_what_the_gradients_keep():
    lib = _lib.load()
    size = lambda Lk, window, dtype: lib.mlxrocm_window_attention_lse_size(  # noqa: E731
        2, 4, 2, 30, Lk, 64, window, 4, ops._DTYPE_CODE[dtype])
    sums, low = 1024, 2 * 4 * 30 * 64 * 2
    assert size(2048, 1 << 30, BF16) == size(9000, 2044, F16) == sums + low
    assert size(2049, 1 << 30, BF16) == size(100, 1 << 30, F32) == sums
