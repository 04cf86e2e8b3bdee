"""Where rotary positions, routing and adapters end: what lies around their results and workspaces stays
as it was, offsets pass 32 bits, runs of tokens are as long as they get."""
import ctypes

import pytest
import torch

import mlx_amd
from mlx_amd import _lib, nn
from test_gpu_adapter_matmul import case, check, close, reference

pytestmark = pytest.mark.gpu

TYPES = (torch.float32, torch.float16, torch.bfloat16)
CODE = {torch.float32: _lib.FLOAT32, torch.float16: _lib.FLOAT16, torch.bfloat16: _lib.BFLOAT16}
PATTERN = 0xA5
MARGIN = 4096


class Guarded:
    """Memory of exactly `nbytes` in the middle of a pattern."""

    def __init__(self, nbytes):
        self.nbytes = nbytes
        self.buffer = torch.full((nbytes + 2 * MARGIN,), PATTERN, dtype=torch.uint8, device="cuda")

    def ptr(self):
        return self.buffer.data_ptr() + MARGIN

    def as_(self, dtype, *shape):
        return self.buffer[MARGIN:MARGIN + self.nbytes].view(dtype).view(shape)

    def check(self, name):
        for part in (self.buffer[:MARGIN], self.buffer[MARGIN + self.nbytes:]):
            assert (part == PATTERN).all(), name


def stream():
    return torch.cuda.current_stream().cuda_stream


def call(name, *args):
    lib = _lib.load()
    status = getattr(lib, name)(*args)
    assert status == _lib.OK, lib.mlxrocm_last_error()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B, L, K, N, r, adapters", (
    (1, 1, 33, 1001, 5, 1), (3, 7, 33, 1001, 5, 2), (70, 1, 40, 17, 16, 3), (2, 50, 1001, 33, 200, 2),
    (1, 300, 264, 130, 16, 1), (5, 41, 72, 100, 130, 4), (100, 3, 36, 20, 33, 6), (2, 1, 8, 8, 1, 70)))
def test_adapters_write_their_results_only(gpu, dtype, B, L, K, N, r, adapters):
    args, dout = case(B, L, K, N, r, adapters, dtype)
    x, a, b, y = (args[n] for n in ("x", "a", "b", "y"))
    indices = args["indices"].int()
    scales = torch.linspace(-1.0, 2.0, adapters).cuda()
    T, size, code = B * L, x.element_size(), CODE[dtype]
    sizes = (T, B, adapters, r, K, N)
    lib = _lib.load()
    out, h = Guarded(T * N * size), Guarded(lib.mlxrocm_adapter_matmul_h_size(*sizes, code))
    need = lib.mlxrocm_adapter_matmul_workspace_size(*sizes, code)
    ws = Guarded(need)
    call("mlxrocm_adapter_matmul", x.data_ptr(), a.data_ptr(), b.data_ptr(), indices.data_ptr(), scales.data_ptr(),
         y.data_ptr(), out.ptr(), h.ptr(), *sizes, K, N, 1.5, code, ws.ptr(), need, stream())
    want = reference(**{**args, "scale": 1.5 * scales.double()}, dout=dout)
    for name, g in (("out", out), ("h", h), ("workspace", ws)):
        g.check(name)
    close(out.as_(dtype, B, L, N), want["out"], "out")
    # h: with both factors, rows filled up to 16 ranks by zeros; rows without an adapter are left as they were
    padded = -(-r // 16) * 16
    of = indices.long().repeat_interleave(L)
    has = (of >= 0) & (of < adapters)
    held = h.as_(torch.float32, T, padded)
    i = of.clamp(0, adapters - 1)
    s = (1.5 * scales.double())[i][:, None]
    x64, a64 = x.double().view(T, K), a.double()[i]
    exact = s * torch.einsum("tk,trk->tr", x64, a64)
    off = (K + 4) * 2.0 ** -24 * s.abs() * torch.einsum("tk,trk->tr", x64.abs(), a64.abs())
    assert ((held[:, :r].double() - exact).abs() <= off)[has].all()
    assert (held[has][:, r:] == 0).all()
    assert (held[~has].view(torch.uint8) == PATTERN).all()
    # gradients: all of them, and each alone
    need = lib.mlxrocm_adapter_matmul_vjp_workspace_size(*sizes, code)
    for wanted in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1)):
        grads = [Guarded(t.numel() * size) if is_ else None for t, is_ in zip((x, a, b), wanted)]
        ws = Guarded(need)
        call("mlxrocm_adapter_matmul_vjp", x.data_ptr(), a.data_ptr(), b.data_ptr(), indices.data_ptr(),
             scales.data_ptr(), h.ptr(), dout.data_ptr(), *(g and g.ptr() for g in grads), *sizes, K, N, 1.5, code,
             ws.ptr(), need, stream())
        ws.check("workspace")
        for name, like, g in zip(("dx", "da", "db"), (x, a, b), grads):
            if g is not None:
                g.check(name)
                close(g.as_(dtype, *like.shape), want[name], name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, experts, k, groups", ((1, 1, 1, 1), (17, 33, 5, 1), (33, 130, 32, 13), (3, 60, 4, 3),
                                                      (16, 1024, 8, 8), (5, 1000, 31, 1), (37, 9, 2, 1)))
def test_routing_writes_its_results_only(gpu, dtype, rows, experts, k, groups):
    g = torch.Generator().manual_seed(rows)
    stride = experts + 3
    logits = torch.randn((rows, stride), generator=g).to(dtype).cuda()[:, :experts]
    bias = torch.randn((experts,), generator=g).cuda()
    grad = torch.randn((rows, k), generator=g).to(dtype).cuda()
    size = logits.element_size()
    for sigmoid, b in ((0, None), (1, bias), (0, bias)):
        indices, weights, out = Guarded(rows * k * 4), Guarded(rows * k * size), Guarded(rows * experts * size)
        top = -(-groups // 2)
        call("mlxrocm_route_experts", logits.data_ptr(), b if b is None else b.data_ptr(), indices.ptr(), weights.ptr(),
             rows, stride, experts, min(k, top * experts // groups), sigmoid, groups, top, 1, 1, 1.0, CODE[dtype],
             stream())
        used = min(k, top * experts // groups)
        for name, got in (("indices", indices), ("weights", weights)):
            got.check(name)
        flat = indices.as_(torch.int32, -1)[:rows * used].view(rows, used)
        want = mlx_amd.route_experts(logits, used, scoring="sigmoid" if sigmoid else "softmax", bias=b, groups=groups,
                                     top_groups=top)
        assert torch.equal(flat, want[0])
        assert torch.equal(weights.as_(dtype, -1)[:rows * used].view(rows, used), want[1])
        call("mlxrocm_route_experts_vjp", logits.data_ptr(), indices.ptr(), grad.data_ptr(), out.ptr(), rows, stride,
             k, experts, used, sigmoid, 1, 1.0, CODE[dtype], stream())
        out.check("gradient")
        assert out.as_(dtype, rows, experts).isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D, dims, traditional", ((64, 64, 0), (18, 6, 0), (18, 6, 1), (80, 40, 1), (2, 2, 0), (300, 256, 0)))
def test_rope_writes_its_result_only(gpu, dtype, D, dims, traditional):
    for B, H, L in ((1, 1, 1), (3, 5, 7), (1, 3, 2100)):
        x = torch.randn((B, H, L, D), generator=torch.Generator().manual_seed(D)).to(dtype).cuda()
        at = torch.arange(L, device="cuda").expand(B, L)
        out = Guarded(x.numel() * x.element_size())
        strides = (ctypes.c_int64 * 6)(*x.stride()[:3], *x.stride()[:3])
        call("mlxrocm_rope", x.data_ptr(), out.ptr(), B, H, L, D, strides, at.data_ptr(),
             (ctypes.c_int64 * 3)(0, 0, 1), 1, 1, None, dims, traditional, 1e4, 1.0, None, 0, CODE[dtype], stream())
        out.check("out")
        assert torch.equal(out.as_(dtype, B, H, L, D), mlx_amd.rope(x, at, dims=dims, traditional=bool(traditional)))


# ---------------------------------------------------------------- offsets beyond 32 bits
def test_logits_and_gradients_far_apart(gpu):
    rows, E = 5, 64
    apart = 2 ** 31 // 4 + 8 * 131
    g = torch.Generator().manual_seed(1)
    dense = torch.randn((rows, E), generator=g).to(torch.bfloat16).cuda()
    far = torch.empty(apart * rows, dtype=torch.bfloat16, device="cuda").as_strided((rows, E), (apart, 1))
    far.copy_(dense)
    bias = torch.randn((E,), generator=g).cuda()
    for options in (dict(), dict(scoring="sigmoid", bias=bias, groups=4, top_groups=2, group_best=2),
                    dict(normalize=False)):
        results = []
        for logits in (dense, far):
            leaf = logits.detach().requires_grad_()
            indices, weights = mlx_amd.route_experts(leaf, 6, **options)
            results.append((indices, weights.detach(), *torch.autograd.grad(weights.float().square().sum(), leaf)))
        for one, two in zip(*results):
            assert torch.equal(one, two)


def test_a_cache_beyond_32_bits(gpu):
    """Pages, queries, keys and values that lie far apart hold what near ones do."""
    g = torch.Generator().manual_seed(4)

    def normal(*shape):
        return torch.randn(shape, generator=g).to(torch.bfloat16).cuda()

    def far(t):
        apart = 8 * (2 ** 28 // (t.shape[0] - 1) + 131)  # (pages are aligned)
        buffer = torch.empty(apart * t.shape[0], dtype=t.dtype, device="cuda")
        return buffer.as_strided(t.shape, (apart, *t.stride()[1:])).copy_(t)

    q, k, v = normal(3, 4, 5, 64), normal(3, 2, 5, 64), normal(3, 2, 5, 64)
    pages = normal(6, 2, 16, 64), normal(6, 2, 16, 64)
    table = torch.tensor([[5, 0], [1, 4], [3, 2]], dtype=torch.int32).cuda()
    lengths = torch.tensor([18, 30, 3], dtype=torch.int32).cuda()
    other = [far(t) for t in (q, k, v, *pages)]
    assert other[3].stride(0) * 5 > 2 ** 31
    near = mlx_amd.rope_cache_update(q, k, v, *pages, table, lengths)
    for one, two in zip(near, mlx_amd.rope_cache_update(*other, table, lengths)):
        assert torch.equal(one, two)


@pytest.mark.parametrize("L", (1, 40))
def test_rows_of_adapters_far_apart(gpu, L):
    args, dout = case(5, L, 96, 80, 16, 3, torch.bfloat16, [0, 2, -1, 2, 1])
    apart = 2 ** 31 // (4 * L) + 8 * 131
    far = {}
    for name, t in (("x", args["x"]), ("y", args["y"]), ("dout", dout)):
        n = t.shape[-1]
        buffer = torch.empty(apart * 5 * L, dtype=torch.bfloat16, device="cuda")
        far[name] = buffer.as_strided((5, L, n), (L * apart, apart, 1)).copy_(t)
    check({**args, "x": far["x"], "y": far["y"]}, far["dout"])


def test_adapters_beyond_32_bits(gpu):
    """1024 adapters whose elements pass 2**31: the first and the last of them, and none for the others."""
    adapters, r, K, N = 1024, 128, 17000, 16896
    assert adapters * r * min(K, N) > 2 ** 31
    used = [1023, 0, 1023, -1, 1000]
    g = torch.Generator(device="cuda").manual_seed(2)
    a = torch.empty((adapters, r, K), dtype=torch.bfloat16, device="cuda")
    b = torch.empty((adapters, N, r), dtype=torch.bfloat16, device="cuda")
    for i in set(used) - {-1}:
        a[i] = torch.randn((r, K), generator=g, device="cuda") * K ** -0.5
        b[i] = torch.randn((N, r), generator=g, device="cuda") * r ** -0.5
    x = torch.randn((5, 3, K), generator=g, device="cuda").to(torch.bfloat16)
    dout = torch.randn((5, 3, N), generator=g, device="cuda").to(torch.bfloat16)
    few = [0, 1000, 1023]
    small = dict(a=a[few], b=b[few], indices=torch.tensor([few.index(i) if i >= 0 else -1 for i in used],
                                                          dtype=torch.int32).cuda())
    leaves = [t.requires_grad_() for t in (x, a, b)]
    out = mlx_amd.adapter_matmul(*leaves, torch.tensor(used, dtype=torch.int32).cuda())
    want = reference(x.detach(), **small, dout=dout)
    close(out, want["out"], "out")
    dx, da, db = torch.autograd.grad(out, leaves, dout)
    close(dx, want["dx"], "dx")
    close(da[few], want["da"], "da")
    close(db[few], want["db"], "db")
    for grad in (da, db):
        for first in range(0, adapters, 128):
            part = grad[first:first + 128].flatten(1).any(1).nonzero().flatten().tolist()
            assert [first + i for i in part] == [i for i in few if first <= i < first + 128]


# ---------------------------------------------------------------- runs of tokens, groups
@pytest.mark.parametrize("dtype", TYPES)
def test_the_longest_runs_of_tokens(gpu, dtype):
    """So many tokens that a workgroup has 2048 of an adapter's sum.  Whole numbers: the sums are exact."""
    T, K, N, r = 140007, 1280, 1300, 4
    g = torch.Generator(device="cuda").manual_seed(3)

    def signs(*shape):
        return torch.randint(-1, 2, shape, generator=g, device="cuda").to(dtype)

    x, a, b, dout = signs(T, K), signs(2, r, K), signs(2, N, r), signs(T, N)
    leaves = [t.requires_grad_() for t in (a, b)]
    # a few rows of the first adapter, the others of the second
    indices = torch.ones(T, dtype=torch.int32, device="cuda")
    indices[::1777] = 0
    indices[5::50000] = -1
    grads = torch.autograd.grad(mlx_amd.adapter_matmul(x, *leaves, indices), leaves, dout)
    for i in range(2):
        mine = indices == i
        x64, d64 = x[mine].double(), dout[mine].double()
        h, back = x64 @ a[i].detach().double().T, d64 @ b[i].detach().double()
        for got, left, right in ((grads[0][i], back.T, x64), (grads[1][i], d64.T, h)):
            assert float((left.abs() @ right.abs()).max()) < 2 ** 24
            assert torch.equal(got, (left @ right).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B, L, adapters", ((65, 3, 2), (100, 7, 40), (130, 33, 5), (70, 2, 1)))
def test_many_requests_of_several_tokens(gpu, dtype, B, L, adapters):
    args, dout = case(B, L, 72, 100, 16, adapters, dtype, seed=B)
    args["indices"] = args["indices"].int()
    check(args, dout)
    check({**args, "y": None}, dout)


@pytest.mark.parametrize("dtype", TYPES)
def test_native_sizes(gpu, dtype):
    """The sizes of the other tests by indices of 32 bits, which the native path takes."""
    from test_gpu_adapter_matmul import SIZES

    for B, L, K, N, r, adapters in SIZES:
        args, dout = case(B, L, K, N, r, adapters, dtype)
        args["indices"] = args["indices"].int()
        check(args, dout)
        check({**args, "y": None}, dout)


# ---------------------------------------------------------------- the layer
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mode", ("affine", "mxfp4", "mxfp8", "nvfp4", None))
def test_lora_linear_beside_every_projection(gpu, dtype, mode):
    torch.manual_seed(0)
    if mode is None:
        base = torch.nn.Linear(128, 192, device="cuda", dtype=dtype)
    else:
        base = nn.QuantizedLinear(128, 192, bias=False, mode=mode, device="cuda", dtype=dtype)
    layer = nn.LoRALinear(base, rank=8, adapters=3, scale=2.0, dtype=dtype)
    assert layer.lora_a.dtype == layer.lora_b.dtype == dtype
    assert layer.lora_a.shape == (3, 8, 128) and layer.lora_b.shape == (3, 192, 8)
    x = torch.randn(4, 5, 128, device="cuda").to(dtype)
    indices = torch.tensor([2, -1, 0, 2], dtype=torch.int32).cuda()
    assert torch.equal(layer(x, indices), base(x))
    with torch.no_grad():
        layer.lora_b.normal_()
    close(layer(x, indices), reference(x, layer.lora_a, layer.lora_b, indices, 2.0, base(x))["out"])
    dout = torch.randn(4, 5, 192, device="cuda").to(dtype)
    grads = torch.autograd.grad(layer(x, indices), (layer.lora_a, layer.lora_b), dout)
    want = reference(x, layer.lora_a, layer.lora_b, indices, 2.0, base(x), dout)
    for name, got in zip(("da", "db"), grads):
        close(got, want[name], name)
