"""The native host path of attention, its cache and the drafts' verification against their own
Python bodies: the same results to the bit where it takes a call, and nothing taken that the bodies
have to convert, copy, differentiate or refuse."""
import pytest
import torch

import mlx_amd
from mlx_amd import _lib
from test_gpu_fast_ops import _x, both  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache(pages=7, heads=2, page=16, dim=64, dtype=torch.bfloat16):
    return _x(pages, heads, page, dim, dtype=dtype), _x(pages, heads, page, dim + 1, dtype=dtype)[
        ..., :dim].contiguous()


TABLE, LENGTHS = [[4, 0, 2], [1, 6, 3]], [37, 20]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 5, 33])
def test_window_attention(both, rows, dtype):  # noqa: F811
    q, k, v = _x(2, rows, 4, 64, dtype=dtype).transpose(1, 2), *(
        _x(2, 2, 60, 64 * n, dtype=dtype)[..., :64] for n in (1, 2))
    for kw in (dict(scale=0.125), dict(scale=0.1, window=9, keep=2, lengths=_int([60, 12]))):
        assert _lib.load_fast().window_attention(
            q, k, v, kw["scale"], kw.get("window"), kw.get("keep", 0), kw.get("lengths")) is not None
        both(lambda: mlx_amd.window_attention(q, k, v, **kw))


@pytest.mark.parametrize("rows", [1, 3, 30])
def test_paged(both, rows):  # noqa: F811
    table, lengths = _int(TABLE), _int(LENGTHS)
    wide = _int([row + [99] for row in TABLE])[:, :3]  # a slice of a wider table
    pages = _cache()
    q, k, v = _x(2, 4, rows, 64), _x(2, 2, rows, 64), _x(2, rows, 2, 64).transpose(1, 2)
    for t in (table, wide):
        both(lambda: mlx_amd.paged_attention(q, *pages, t, lengths, scale=0.125, window=8, keep=1))
        both(lambda: mlx_amd.paged_cache_update(k, v, *(p.clone() for p in pages), t, lengths))
    fast = _lib.load_fast()
    assert fast.paged_attention(q, *pages, wide, lengths, 0.125, None, 0) is not None
    assert fast.paged_cache_update(k, v, *(p.clone() for p in pages), wide, lengths) is True


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_verify_draft(both, dtype):  # noqa: F811
    p, q = (torch.softmax(_x(3, n, 1001, dtype=torch.float32), -1).to(dtype) for n in (5, 4))
    draft = torch.randint(0, 1001, (3, 4), dtype=torch.int32, device="cuda")
    u = torch.rand((3, 5), device="cuda")
    args = (draft, p, q, u[:, :4].contiguous(), u[:, 4].contiguous())
    assert _lib.load_fast().verify_draft(*args, None) is not None
    both(lambda: mlx_amd.verify_draft(*args))
    both(lambda: mlx_amd.verify_draft(draft, p, None, *args[3:], lengths=_int([4, 0, 2])))
    # what the body has to convert or copy
    assert _lib.load_fast().verify_draft(draft.long(), *args[1:], None) is None
    assert _lib.load_fast().verify_draft(draft, p, q, u[:, :4], u[:, 4], None) is None
    both(lambda: mlx_amd.verify_draft(draft.long(), p, q, u[:, :4], u[:, 4]))


def test_what_is_left_to_the_bodies(both):  # noqa: F811
    fast = _lib.load_fast()
    q, k, v = _x(2, 4, 5, 64), _x(2, 2, 40, 64), _x(2, 2, 40, 64)
    rest = (0.125, None, 0, None)
    assert fast.window_attention(q, k, v, *rest) is not None
    for args in (
            (q.float(), k, v, *rest), (q.cpu(), k, v, *rest), (q, k[:1], v[:1], *rest),
            (q, k, v[..., :32], *rest), (q, k[:, :, :0], v[:, :, :0], *rest),
            (q[..., ::2], k[..., ::2], v[..., ::2], *rest), (q[..., 4:36], k[..., :32], v[..., :32], *rest),
            (q[..., :60], k[..., :60], v[..., :60], *rest), (q[:, :3], k, v, *rest),
            (q, k, v, 1, None, 0, None), (q, k, v, float("inf"), None, 0, None),
            (q, k, v, 0.125, 0, 0, None), (q, k, v, 0.125, None, -1, None),
            (q, k, v, 0.125, True, 0, None), (q, k, v, 0.125, None, 0, _int([40])),
            (q, k, v, 0.125, None, 0, _int([40, 40]).long())):
        assert fast.window_attention(*args) is None
    both(lambda: mlx_amd.window_attention(q.float(), k, v, scale=0.125))
    both(lambda: mlx_amd.window_attention(q[..., 4:36], k[..., :32], v[..., :32], scale=1))
    both(lambda: mlx_amd.window_attention(q, k[:, :, :0], v[:, :, :0], scale=0.125))
    leaf = q.clone().requires_grad_()
    assert fast.window_attention(leaf, k, v, *rest) is None
    both(lambda: mlx_amd.window_attention(leaf, k, v, scale=0.125))
    with torch.no_grad():
        assert fast.window_attention(leaf, k, v, *rest) is not None


def test_what_cannot_be_written_to(both):  # noqa: F811
    table, lengths = _int(TABLE), _int(LENGTHS)
    k_pages, v_pages = _cache()
    k, v = _x(2, 2, 3, 64), _x(2, 2, 3, 64)
    shared = k_pages[:1].expand(7, -1, -1, -1)
    with pytest.raises(ValueError, match="share memory"):
        mlx_amd.paged_cache_update(k, v, shared, v_pages, table, lengths)
    for args in ((k.clone().requires_grad_(), v, k_pages), (k, v, k_pages.clone().requires_grad_())):
        with pytest.raises(NotImplementedError, match="no gradients"):
            mlx_amd.paged_cache_update(*args, v_pages, table, lengths)
        with torch.no_grad():
            mlx_amd.paged_cache_update(*args, v_pages, table, lengths)


def test_on_another_stream():
    table, lengths, pages = _int(TABLE), _int(LENGTHS), _cache()
    q = _x(2, 8, 1, 64)
    want = mlx_amd.paged_attention(q, *pages, table, lengths, scale=0.125)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = [mlx_amd.paged_attention(q, *pages, table, lengths, scale=0.125) for _ in range(20)]
    stream.synchronize()
    assert all(torch.equal(t, want) for t in got)


def _leaves(dtype=torch.bfloat16, length=40):
    fused = _x(2, length, 8, 64, dtype=dtype)  # four heads of q, two of k, two of v, side by side
    return [t.transpose(1, 2).detach().requires_grad_() for t in fused.split((4, 2, 2), 2)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths", [None, [40, 13]])
def test_gradients(both, lengths, dtype):  # noqa: F811
    n = None if lengths is None else _int(lengths)
    cotangent = _x(2, 40, 4, 64, dtype=dtype).transpose(1, 2)

    def run(cotangent):
        leaves = _leaves(dtype)
        out = mlx_amd.window_attention(*leaves, scale=0.125, window=9, keep=2, lengths=n)
        grads = torch.autograd.grad(out, leaves, cotangent)
        assert [g.stride() for g in grads] == [torch.empty_like(t).stride() for t in leaves]
        return (out.detach(), *grads)

    both(lambda: run(cotangent))
    both(lambda: run(cotangent[:, :, :1].expand(2, 4, 40, 64)))
    both(lambda: run(cotangent[..., :1].expand(2, 4, 40, 64)))  # not dense
    assert _lib.load_fast().window_attention_recorded(*_leaves(dtype), 0.125, 9, 2, n) is not None


def test_what_is_recorded():
    fast = _lib.load_fast()
    q, k, v = _leaves()
    rest = (0.125, None, 0, None)
    plain = [t.detach() for t in (q, k, v)]
    assert fast.window_attention_recorded(*plain, *rest) is None
    assert fast.window_attention_recorded(q.float(), k, v, *rest) is None
    with torch.no_grad():
        assert fast.window_attention_recorded(q, k, v, *rest) is None
    # a gradient of one operand, twice from one graph, and added up
    out = fast.window_attention_recorded(*plain[:2], v, *rest)
    assert out.requires_grad and out.grad_fn is not None
    (dv,) = torch.autograd.grad(out.sum(), v, retain_graph=True)
    out.sum().backward()
    assert torch.equal(v.grad, dv) and q.grad is None
    with pytest.raises(RuntimeError, match="second time"):
        out.sum().backward()
    # once differentiable
    out = fast.window_attention_recorded(q, k, v, *rest)
    (dq,) = torch.autograd.grad(out.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        dq.float().sum().backward()
    # what it needs was written to
    x = q * 1
    out = fast.window_attention_recorded(x, k, v, *rest)
    x.zero_()
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()


def test_gradients_on_another_stream():
    want = None
    for stream in (None, torch.cuda.Stream()):
        leaves = _leaves(length=300)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            out = mlx_amd.window_attention(*leaves, scale=0.125)
            grads = torch.autograd.grad(out, leaves, torch.ones_like(out))
        torch.cuda.synchronize()
        want = grads if want is None else want
        assert all(torch.equal(a, b) for a, b in zip(grads, want))
