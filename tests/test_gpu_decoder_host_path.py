"""The native host path of rotary positions, routing and adapters against their own Python bodies:
the same results and gradients to the bit where it takes a call, whichever operands are left out, and
nothing taken that the bodies have to convert, copy or refuse."""
import itertools

import pytest
import torch

import mlx_amd
from mlx_amd import _lib
from test_gpu_fast_ops import _x, both  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu

TYPES = (torch.float32, torch.float16, torch.bfloat16)


def _int(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _plus(t, n):
    return (t.float() + n).to(t.dtype)


# ---------------------------------------------------------------- adapters
def adapted(dtype, adapters, L=5):
    x, y = _x(3, L, 96, dtype=dtype), _x(3, L, 80, dtype=dtype)
    return x, _x(adapters, 16, 96, dtype=dtype), _x(adapters, 80, 16, dtype=dtype), y


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("indices", (None, [2, -1, 0], [[0, 1, 2, -1, 0], [7, 0, 0, 1, 1], [2, 2, 2, 2, 2]]), ids=str)
@pytest.mark.parametrize("beside", (False, True))
def test_adapter_matmul(both, dtype, indices, beside):  # noqa: F811
    x, a, b, y = adapted(dtype, 1 if indices is None else 3)
    y = y if beside else None
    of = None if indices is None else _int(indices)
    assert _lib.load_fast().adapter_matmul(x, a, b, of, 1.5, y) is not None
    both(lambda: mlx_amd.adapter_matmul(x, a, b, of, scale=1.5, y=y))
    operands = [x, a, b] + ([y] if beside else [])
    dout = _x(3, 5, 80, dtype=dtype)
    for wanted in itertools.product((False, True), repeat=len(operands)):
        if not any(wanted):
            continue
        leaves = [t.detach().requires_grad_(is_) for t, is_ in zip(operands, wanted)]

        def step(dout=dout):
            out = mlx_amd.adapter_matmul(*leaves[:3], of, scale=1.5, y=leaves[3] if beside else None)
            grads = torch.autograd.grad(out, [t for t in leaves if t.requires_grad], dout)
            return (out, *(t.contiguous() for t in grads))

        assert _lib.load_fast().adapter_matmul(*leaves[:3], of, 1.5, leaves[3] if beside else None) is not None
        both(step)
    both(lambda: step(dout[:1, :, :1].expand(3, 5, 80)))
    both(lambda: step(dout.transpose(0, 1).contiguous().transpose(0, 1)))


@pytest.mark.parametrize("L", (1, 40))
def test_adapter_matmul_of_parts_of_rows(both, L):  # noqa: F811
    """Rows that lie apart, and rows of one element."""
    x, a, b, y = adapted(torch.bfloat16, 3, L)
    of = _int([1, 1, 0])
    wide_x, wide_y = _x(3, L, 200), _x(3, L, 90)
    for u, v in ((wide_x[..., 8:104], wide_y[..., 5:85]), (wide_x[:1, :1, :96].expand(3, L, 96), None)):
        u = u.detach().requires_grad_()
        assert _lib.load_fast().adapter_matmul(u, a, b, of, 2.0, v) is not None

        def step():
            out = mlx_amd.adapter_matmul(u, a, b, of, scale=2.0, y=v)
            return (out, *torch.autograd.grad(out, u, y))

        both(step)
    both(lambda: mlx_amd.adapter_matmul(x[0, 0], a, b, _int(2)))
    both(lambda: mlx_amd.adapter_matmul(x[..., :1], a[..., :1].contiguous(), b[:, :1].contiguous(), of))
    assert _lib.load_fast().adapter_matmul(x[0, 0], a, b, _int(2), 1.0, None) is not None


def test_adapters_left_to_the_body(both):  # noqa: F811
    x, a, b, y = adapted(torch.bfloat16, 3)
    of = _int([1, 0, 2])
    fast = _lib.load_fast()
    for args in ((x, a, b, of.long(), 1.0, y), (x.float(), a, b, of, 1.0, None), (x, a, b, None, 1.0, y),
                 (x, a, b, of, torch.ones(3), y), (x, a, b, of, float("inf"), y), (x, a, b, of, 1.0, y[:1]),
                 (x, a[:2], b, of, 1.0, y), (x, a.transpose(1, 2), b, of, 1.0, y), (x.cpu(), a, b, of, 1.0, y),
                 (x[..., :95], a, b, of, 1.0, y), (x, a, b, _int([1, 0]), 1.0, y), (x[:0], a, b, of[:0], 1.0, None),
                 (x, a[0], b[0], None, 1.0, y), (x, a, b, of, 1.0, y.double())):
        assert fast.adapter_matmul(*args) is None


# ---------------------------------------------------------------- positions
ROTATIONS = (dict(), dict(dims=32), dict(traditional=True), dict(base=500.0, scale=0.5), dict(freqs=True),
             dict(sections=(8, 12, 12)), dict(sections=(32,)), dict(dims=16, sections=(0, 8), traditional=True))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("options", ROTATIONS, ids=str)
def test_rope(both, dtype, options):  # noqa: F811
    options = dict(options)
    if options.get("freqs"):
        options["freqs"] = torch.arange(1, 33, device="cuda").float()
    sections = options.get("sections")
    fast = _lib.load_fast()
    for kind in (torch.int32, torch.int64):
        at = torch.randint(-9, 3000, ((len(sections),) if sections else ()) + (2, 7), device="cuda").to(kind)
        for x in (_x(2, 7, 3, 64, dtype=dtype).transpose(1, 2), _x(2, 3, 7, 70, dtype=dtype)[..., 3:67]):
            plain = (x, at, options.get("dims"), options.get("traditional", False), options.get("base"),
                     options.get("scale", 1.0), options.get("freqs"), sections)
            assert fast.rope(*plain) is not None
            both(lambda: mlx_amd.rope(x, at, **options))
            x = x.detach().requires_grad_()
            up = _x(2, 3, 7, 64, dtype=dtype).requires_grad_()

            def step(up=up):
                out = mlx_amd.rope(x, at, **options)
                dx, = torch.autograd.grad(out, x, up, create_graph=True)
                if not up.requires_grad:
                    return out, dx
                return out, dx, *torch.autograd.grad(dx.float().square().sum(), up)

            assert fast.rope(x, *plain[1:]) is not None
            both(step)
            both(lambda: step(up.detach()[:, :1, :, :1].expand(2, 3, 7, 64)))
            both(lambda: step(up.detach().transpose(2, 3).contiguous().transpose(2, 3)))


@pytest.mark.parametrize("options", ROTATIONS, ids=str)
def test_rope_cache_update(both, options):  # noqa: F811
    options = dict(options)
    if options.get("freqs"):
        options["freqs"] = torch.arange(1, 33, device="cuda").float()
    sections = options.get("sections")
    at = None if sections is None else torch.randint(0, 90, (len(sections), 2, 5), device="cuda")
    q, k, v = _x(2, 5, 4, 64).transpose(1, 2), _x(2, 2, 5, 64), _x(2, 2, 5, 66)[..., :64]
    pages = _x(7, 2, 16, 64), _plus(_x(7, 2, 16, 64), 1)
    table, lengths = _int([[4, 0, 2, 9], [1, 6, 3, 9]])[:, :3], _int([37, 3])
    plain = (q, k, v, *(p.clone() for p in pages), table, lengths, at, options.get("dims"),
             options.get("traditional", False), options.get("base"), options.get("scale", 1.0),
             options.get("freqs"), sections)
    assert _lib.load_fast().rope_cache_update(*plain) is not None
    both(lambda: mlx_amd.rope_cache_update(q, k, v, *(p.clone() for p in pages), table, lengths, positions=at,
                                           **options))


def test_positions_left_to_the_body(both):  # noqa: F811
    fast = _lib.load_fast()
    x, at = _x(2, 3, 7, 64), torch.zeros((2, 7), dtype=torch.int32, device="cuda")
    for args in ((x, at.to(torch.uint32), None, False, None, 1.0, None, None), (x, None, None, False, None, 1.0, None, None),
                 (x, at, 63, False, None, 1.0, None, None), (x, at, None, False, -1.0, 1.0, None, None),
                 (x, at, None, False, None, 1.0, None, [32]), (x, at, None, False, None, 1.0, None, (32,)),
                 (x, at, None, False, 5.0, 1.0, torch.ones(32, device="cuda"), None),
                 (x, at, None, False, None, 1.0, torch.ones(32, device="cuda").half(), None),
                 (x.transpose(2, 3), at, None, False, None, 1.0, None, None), (x.double(), at, None, False, None, 1.0, None, None),
                 (x, at.cpu(), None, False, None, 1.0, None, None), (x, at, None, False, None, float("nan"), None, None)):
        assert fast.rope(*args) is None


# ---------------------------------------------------------------- experts
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scoring", ("softmax", "sigmoid"))
@pytest.mark.parametrize("normalize", (False, True))
def test_route_experts(both, dtype, scoring, normalize):  # noqa: F811
    bias = _x(48, dtype=torch.float32)
    fast = _lib.load_fast()
    for logits in (_x(5, 48, dtype=dtype), _x(2, 3, 60, dtype=dtype)[..., 5:53], _x(48, dtype=dtype)):
        for more in (dict(), dict(bias=bias), dict(groups=4, top_groups=2, group_best=2), dict(groups=3, scale=-2.0)):
            options = dict(scoring=scoring, normalize=normalize, **more)
            plain = (6, scoring, more.get("bias"), more.get("groups", 1), more.get("top_groups"),
                     more.get("group_best", 1), normalize, more.get("scale", 1.0))
            assert fast.route_experts(logits, *plain) is not None
            both(lambda: mlx_amd.route_experts(logits, 6, **options))
            leaf = logits.detach().requires_grad_()
            up = _x(*logits.shape[:-1], 6, dtype=dtype)

            def step(up=up):
                indices, weights = mlx_amd.route_experts(leaf, 6, **options)
                return indices, weights, *torch.autograd.grad(weights, leaf, up)

            assert fast.route_experts(leaf, *plain) is not None
            both(step)
            both(lambda: step(up[..., :1].expand(up.shape)))
            if up.dim() > 1:
                both(lambda: step(up.transpose(0, -1).contiguous().transpose(0, -1)))
    for args in ((logits.double(), *plain), (logits.cpu(), *plain), (logits, 0, *plain[1:]), (logits, 49, *plain[1:]),
                 (logits, 6, "relu", *plain[2:]), (logits, 6, scoring, bias[:47], *plain[3:]),
                 (logits, 6, scoring, bias.half(), *plain[3:]), (logits, 6, scoring, None, 5, *plain[4:])):
        assert fast.route_experts(*args) is None


def test_twice_is_refused_and_unused_results_have_no_gradient(both):  # noqa: F811
    x, a, b, y = (t.requires_grad_() for t in adapted(torch.float32, 3))
    logits = _x(5, 48, dtype=torch.float32).requires_grad_()

    def twice():
        for out, leaf in ((mlx_amd.adapter_matmul(x, a, b, _int([0, 1, 2]), y=y), x),
                          (mlx_amd.adapter_matmul(x, a, b, _int([0, 1, 2])), b),
                          (mlx_amd.route_experts(logits, 4)[1], logits)):
            grad, = torch.autograd.grad(out.square().sum(), leaf, create_graph=True)
            with pytest.raises(RuntimeError, match="once_differentiable"):
                grad.sum().backward()
        indices, weights = mlx_amd.route_experts(logits, 4)
        assert not indices.requires_grad and weights.requires_grad
        return indices, weights

    both(twice)


def test_every_launch_is_on_the_tensors_device(monkeypatch):
    """The bodies make the tensors' device the current one before they convert, copy or compute: an
    operand may be on another."""
    from mlx_amd import _copy, ops, rotary
    from test_gpu_fast_ops import _Nothing

    inside = []
    device, copy, lib = torch.cuda.device, _copy.copy, _lib.load()

    class Device(device):
        def __enter__(self):
            inside.append(self)
            return super().__enter__()

        def __exit__(self, *args):
            inside.pop()
            return super().__exit__(*args)

    def copied(*args):
        assert inside, "a copy"
        return copy(*args)

    class Checked:
        def __getattr__(self, name):
            if not name.endswith("_size") and name != "mlxrocm_last_error":
                assert inside, name
            return getattr(lib, name)

    x, a, b, y = adapted(torch.bfloat16, 3)
    q, k = _x(2, 7, 4, 64).transpose(1, 2), _x(2, 2, 64, 7).transpose(2, 3)
    at = torch.arange(7, device="cuda").expand(2, 7)
    pages = _x(7, 2, 16, 64), _x(7, 2, 16, 64)
    freqs = torch.arange(1, 33, device="cuda").half()
    logits = _x(5, 96)[:, ::2]
    monkeypatch.setattr(ops, "_fast", _Nothing())
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(_copy, "copy", copied)
    monkeypatch.setattr(rotary, "_copy", copied)
    monkeypatch.setattr(_lib, "load", Checked)
    mlx_amd.adapter_matmul(x, a.float(), b, _int([1, 0, -1], torch.int64), y=y, scale=torch.ones(3, device="cuda").half())
    mlx_amd.adapter_matmul(x[..., ::2].transpose(0, 1), a[..., :48], b, _int([1, 0, 1, 2, 0]))
    mlx_amd.rope(k, at.to(torch.uint32), freqs=freqs)
    mlx_amd.rope_cache_update(q, k, k, *pages, _int([[4, 0], [1, 6]], torch.int64), _int([7, 3], torch.int64), freqs=freqs)
    mlx_amd.route_experts(logits, 4, bias=_x(48))
    leaves = [t.requires_grad_() for t in (x, a, b, q, logits)]
    out = (mlx_amd.adapter_matmul(x, a, b, _int([1, 0, 2], torch.int64)), mlx_amd.rope(q, at),
           mlx_amd.route_experts(logits, 4)[1])
    torch.autograd.grad(sum(t.float().sum() for t in out), leaves)
