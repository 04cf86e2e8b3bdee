"""adapter_matmul and its gradients against 64 bits."""
import math

import pytest
import torch

import mlx_amd
from mlx_amd import nn

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8,
             torch.float64: 2.0 ** -53}  # (the last where differences are taken of the formulas)
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133,
            torch.float64: 0.0}
# of the narrow operand where it is the sum of two numbers: relative to itself (bfloat16), to the
# largest of its token (float16)
HELD = {torch.float64: 0.0, torch.float32: 0.0, torch.float16: 2.0 ** -21, torch.bfloat16: 2.0 ** -17}
TYPES = (torch.float32, torch.float16, torch.bfloat16)
F = 2.0 ** -24


def reference(x, a, b, indices=None, scale=1.0, y=None, dout=None):
    """{name: (value, bound)}: out, and dx, da, db where dout is given.

    A sum of n products in 32 bits is off by at most (n + 2) 2**-24 of the sum of their magnitudes; h
    and g carry that into the products they go into, beside how they are held there; sums over
    tokens hold them, and float16's x and dout, as two bfloat16 numbers (the product of the lower
    parts is left out: 2**-16 in all)."""
    dtype = x.dtype
    K, N = a.shape[2], b.shape[1]
    rows = x.detach().double().reshape(-1, K)
    n = len(rows)
    if indices is None:
        of = torch.zeros(n, dtype=torch.long, device=x.device)
    else:
        of = indices.long().reshape(-1, 1).expand(-1, n // max(indices.numel(), 1)).reshape(-1)
    has = (of >= 0) & (of < a.shape[0])
    of = torch.where(has, of, 0)
    scales = torch.as_tensor(scale, dtype=torch.float64, device=x.device).expand(a.shape[0])
    s = torch.where(has, scales[of], 0.0)[:, None]
    a, b = a.detach().double(), b.detach().double()
    A, B = a[of], b[of]
    rows = torch.where(has[:, None], rows, 0.0)
    h = s * torch.einsum("tk,trk->tr", rows, A)
    h_size = s.abs() * torch.einsum("tk,trk->tr", rows.abs(), A.abs())
    r = a.shape[1]
    u, tiny = HALF_STEP[dtype], SMALLEST[dtype]

    def held(v):
        return HELD[dtype] * (v.abs() if dtype != torch.float16 else v.abs().amax(1, keepdim=True))

    h_off = (K + 4) * F * h_size
    delta = torch.einsum("tr,tnr->tn", h, B)
    off = torch.einsum("tr,tnr->tn", h_off + held(h) + (2 * r + 4) * F * (h.abs() + h_off), B.abs())
    base = torch.zeros_like(delta) if y is None else y.detach().double().reshape(-1, N)
    out = base + delta
    shape = (*x.shape[:-1], N)
    results = {"out": (out.reshape(shape), (off + (u + 2 * F) * (out.abs() + off) + tiny).reshape(shape))}
    if dout is not None:
        d = torch.where(has[:, None], dout.detach().double().reshape(-1, N), 0.0)
        g = s * torch.einsum("tn,tnr->tr", d, B)
        g_off = (N + 4) * F * s.abs() * torch.einsum("tn,tnr->tr", d.abs(), B.abs())
        dx = torch.einsum("tr,trk->tk", g, A)
        off = torch.einsum("tr,trk->tk", g_off + held(g) + (2 * r + 4) * F * (g.abs() + g_off), A.abs())
        results["dx"] = (dx.reshape(x.shape), (off + (u + 2 * F) * (dx.abs() + off) + tiny).reshape(x.shape))
        pair = 0.0 if dtype == torch.float32 else 2.0 ** -16
        for name, like, p, p_off, q, turned in (("da", a, g, g_off, rows, False),
                                                ("db", b, h, h_off, d, True)):
            value, bound = torch.zeros_like(like), torch.zeros_like(like)
            for i in range(len(like)):
                mine = has & (of == i)
                m = int(mine.sum())
                v = p[mine].T @ q[mine]
                e = (p_off[mine] + (pair + (m + 4) * F) * (p[mine].abs() + p_off[mine])).T @ q[mine].abs()
                value[i], bound[i] = (v.T, e.T) if turned else (v, e)
            results[name] = (value, bound + (u + 2 * F) * (value.abs() + bound) + tiny)
    return results


def close(got, want, name=""):
    value, bound = want
    assert got.shape == value.shape, (name, got.shape, value.shape)
    # Beyond the type's largest value lies infinity: 94031 is more than float16's 65504 and half a
    # step of 32, 65520, from which on values round to infinity; within the bound of that, either
    most = torch.finfo(got.dtype).max * (1 + HALF_STEP[got.dtype])
    got = got.detach().double()
    infinite = got == value.sign() * math.inf
    assert infinite[value.abs() - bound >= most].all()
    beyond = infinite & (value.abs() + bound >= most)
    off = torch.where(beyond, 0.0, (got - value).abs() - bound)
    assert float(off.max()) <= 0, (name, float(off.max()))


def case(B, L, K, N, r, adapters, dtype, indices=None, seed=0, y=True):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g) * std).to(dtype).cuda()

    if indices is None:
        indices = torch.randint(-1, adapters, (B,), generator=g)
    return dict(x=normal(B, L, K), a=normal(adapters, r, K, std=K ** -0.5),
                b=normal(adapters, N, r, std=r ** -0.5), indices=torch.as_tensor(indices).cuda(),
                scale=1.5, y=normal(B, L, N) if y else None), normal(B, L, N)


def check(args, dout=None):
    names = ("x", "a", "b")
    if dout is None:
        close(mlx_amd.adapter_matmul(**args), reference(**args)["out"], "out")
        return
    want = reference(**args, dout=dout)
    leaves = {n: args[n].detach().requires_grad_() for n in names}
    if args.get("y") is not None:
        leaves["y"] = args["y"].detach().requires_grad_()
    out = mlx_amd.adapter_matmul(**{**args, **leaves})
    close(out, want["out"], "out")
    assert torch.equal(out.detach(), mlx_amd.adapter_matmul(**args))
    grads = torch.autograd.grad(out, list(leaves.values()), dout)
    for name, got in zip(leaves, grads):
        if name == "y":
            assert torch.equal(got, dout)
        else:
            close(got, want["d" + name], "d" + name)


SIZES = (
    (1, 1, 64, 64, 8, 1), (1, 1, 4096, 512, 16, 3), (7, 1, 256, 100, 4, 3), (64, 1, 128, 96, 64, 9),
    (65, 1, 128, 96, 16, 9), (3, 5, 96, 130, 12, 2), (2, 33, 72, 1001, 1, 4), (1, 100, 1056, 48, 32, 1),
    (5, 64, 160, 272, 128, 3), (2, 17, 40, 33, 200, 2), (3, 40, 64, 24, 256, 2), (6, 1, 33, 17, 5, 4),
    (4, 70, 512, 600, 33, 6), (300, 1, 64, 80, 16, 40), (1, 500, 320, 520, 16, 1), (2, 31, 8, 8, 16, 70),
)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B, L, K, N, r, adapters", SIZES)
def test_adapter_matmul_and_its_gradients(gpu, dtype, B, L, K, N, r, adapters):
    args, dout = case(B, L, K, N, r, adapters, dtype)
    check(args, dout)
    check({**args, "y": None})


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("indices", ([-1] * 6, [0] * 6, [2, 0, 2, 1, 0, 2], [5, -3, 1 << 30, 2, 3, -1 << 31]),
                         ids=str)
@pytest.mark.parametrize("L", (1, 21))
def test_requests_with_and_without_adapters(gpu, dtype, indices, L):
    args, dout = case(6, L, 128, 144, 16, 4, dtype, indices)
    none = torch.tensor([i < 0 or i >= 4 for i in indices])
    out = mlx_amd.adapter_matmul(**args)
    assert torch.equal(out[none], args["y"][none])
    assert (mlx_amd.adapter_matmul(**{**args, "y": None})[none] == 0).all()
    check(args, dout)
    unused = [i for i in range(4) if i not in indices]
    a = args["a"].requires_grad_()
    da, = torch.autograd.grad(mlx_amd.adapter_matmul(**args), a, dout)
    assert (da[unused] == 0).all()


def test_one_adapter_and_matrices(gpu):
    args, dout = case(2, 30, 96, 64, 8, 1, torch.bfloat16)
    args["indices"] = None
    check(args, dout)
    a, b = args["a"][0].requires_grad_(), args["b"][0].requires_grad_()
    out = mlx_amd.adapter_matmul(args["x"], a, b, scale=1.5, y=args["y"])
    assert torch.equal(out.detach(), mlx_amd.adapter_matmul(**args))
    da, db = torch.autograd.grad(out, (a, b), dout)
    assert da.shape == a.shape and db.shape == b.shape


def test_indices_of_tokens_and_of_all(gpu):
    args, dout = case(3, 50, 64, 80, 16, 5, torch.float16)
    g = torch.Generator().manual_seed(3)
    for dtype in (torch.int32, torch.int64, torch.uint8):
        args["indices"] = torch.randint(0, 6, (3, 50), generator=g).to(dtype).cuda()  # 5: none
        check(args, dout)
    args["indices"] = torch.tensor(3).cuda()
    check(args, dout)
    flat = {**args, "x": args["x"][0, 0], "y": args["y"][0, 0]}
    check(flat, dout[0, 0])


def test_scales_of_each_adapter(gpu):
    for dtype in TYPES:
        args, dout = case(5, 9, 64, 80, 16, 3, dtype)
        args["scale"] = torch.tensor([0.5, -2.0, 0.0]).cuda()
        check(args, dout)
    args["scale"] = torch.tensor(2.0)
    check({**args, "scale": torch.tensor(2.0)})


def test_strides_and_types(gpu):
    args, dout = case(4, 6, 128, 96, 16, 3, torch.bfloat16)
    side = torch.randn(4, 6, 3 * 128, device="cuda").to(torch.bfloat16)
    args["x"] = side[..., 128:256]  # a part of a wider product
    args["y"] = torch.randn(4, 6, 200, device="cuda").to(torch.bfloat16)[..., 3:99]
    check(args, dout)
    check(args, torch.randn(6, 4, 96, device="cuda").to(torch.bfloat16).transpose(0, 1))
    args["a"] = args["a"].transpose(1, 2).contiguous().transpose(1, 2)
    args["x"] = args["x"].transpose(0, 1).contiguous().transpose(0, 1)
    check(args, dout)
    check({**args, "y": args["y"][:1, :1].expand(4, 6, 96)}, dout[:1, :, :1].expand(4, 6, 96))
    # adapters in float32 beside activations in bfloat16: all in float32
    mixed = {**args, "a": args["a"].float().requires_grad_(), "b": args["b"].float()}
    out = mlx_amd.adapter_matmul(**mixed)
    assert out.dtype == torch.float32
    wide = {n: t.float() if n in "xaby" else t for n, t in args.items()}
    assert torch.equal(out.detach(), mlx_amd.adapter_matmul(**wide))
    x = args["x"].detach().requires_grad_()
    dx, = torch.autograd.grad(mlx_amd.adapter_matmul(**{**mixed, "x": x}), x, dout.float())
    assert dx.dtype == torch.bfloat16


def test_only_some_gradients(gpu):
    args, dout = case(3, 20, 64, 80, 16, 3, torch.bfloat16)
    every = {n: args[n].detach().requires_grad_() for n in ("x", "a", "b", "y")}
    want = dict(zip(every, torch.autograd.grad(
        mlx_amd.adapter_matmul(**{**args, **every}), list(every.values()), dout)))
    for name in every:
        leaf = args[name].detach().requires_grad_()
        got, = torch.autograd.grad(mlx_amd.adapter_matmul(**{**args, name: leaf}), leaf, dout)
        assert torch.equal(got, want[name])


def test_empty(gpu):
    args, dout = case(3, 0, 64, 80, 16, 3, torch.bfloat16)
    leaves = {n: args[n].detach().requires_grad_() for n in ("x", "a", "b")}
    out = mlx_amd.adapter_matmul(**{**args, **leaves})
    assert out.shape == (3, 0, 80)
    for leaf, got in zip(leaves.values(), torch.autograd.grad(out, list(leaves.values()), dout)):
        assert got.shape == leaf.shape and (got == 0).all()
    args, _ = case(0, 4, 64, 80, 16, 3, torch.float32, indices=torch.zeros(0, dtype=torch.int32))
    assert mlx_amd.adapter_matmul(**args).shape == (0, 4, 80)


def test_small_and_large_float16(gpu):
    """h beyond float16's range, and far below it, still counts."""
    for size in (2.0 ** -12, 2.0 ** 11):
        args, dout = case(5, 3, 256, 64, 16, 2, torch.float16, y=False)
        args["x"] = args["x"] * size
        args["a"] = (args["a"] * 16 * size).to(torch.float16)
        args["scale"] = size ** -2
        check(args, dout)
    args, dout = case(3, 40, 256, 64, 16, 2, torch.float16)
    check(args, dout * 2.0 ** -18)


def test_rows_do_not_touch_each_other(gpu):
    """What is not finite in one request, or in its adapter, stays there."""
    for L in (1, 20):
        args, dout = case(5, L, 96, 64, 16, 4, torch.bfloat16, indices=[0, 1, 2, 1, -1])
        clean = mlx_amd.adapter_matmul(**args)
        args["x"][0, 0, 5] = math.inf
        args["x"][4] = math.nan  # no adapter reads it
        args["a"][2, 3, 7] = math.nan
        out = mlx_amd.adapter_matmul(**args)
        assert not out[0, 0].isfinite().any() and out[2].isnan().all()
        assert torch.equal(out[0, 1:], clean[0, 1:]) and torch.equal(out[[1, 3, 4]], clean[[1, 3, 4]])


def test_the_same_bits_again_and_rows_behind(gpu):
    args, dout = case(9, 70, 256, 300, 16, 4, torch.bfloat16)
    leaves = {n: args[n].detach().requires_grad_() for n in ("x", "a", "b")}
    runs = []
    for _ in range(2):
        out = mlx_amd.adapter_matmul(**{**args, **leaves})
        runs.append((out.detach(), *torch.autograd.grad(out, list(leaves.values()), dout)))
    for one, two in zip(*runs):
        assert torch.equal(one, two)


def test_many_rows_of_one_and_of_many_adapters(gpu):
    """Sums over tokens that are cut and joined, tiles that end inside requests."""
    for adapters, L in ((1, 3000), (3, 999)):
        args, dout = case(4, L, 520, 264, 16, adapters, torch.bfloat16,
                          indices=[i % adapters for i in range(4)])
        check(args, dout)


def test_gradient_against_differences(gpu):
    args, dout = case(3, 4, 40, 24, 8, 2, torch.float32)
    args["indices"] = torch.tensor([1, 0, 1]).cuda()
    leaves = {n: args[n].detach().requires_grad_() for n in ("x", "a", "b")}
    grads = torch.autograd.grad(mlx_amd.adapter_matmul(**{**args, **leaves}), list(leaves.values()), dout)
    g = torch.Generator().manual_seed(11)
    for (name, leaf), grad in zip(leaves.items(), grads):
        step = torch.randn(leaf.shape, generator=g).cuda().double()
        e = 1e-3  # (linear in each of them: the differences have no error of their own)
        at = [float((reference(**{**args, name: leaf.double() + s * e * step})["out"][0]
                     * dout.double()).sum()) for s in (1, -1)]
        size = float((grad.double().abs() * step.abs()).sum())
        assert abs(float((grad.double() * step).sum()) - (at[0] - at[1]) / (2 * e)) <= 200 * F * size + 1e-9


def test_captured_training_and_decoding(gpu):
    args, dout = case(6, 1, 128, 96, 16, 4, torch.bfloat16)
    rows, drows = case(3, 90, 128, 96, 16, 4, torch.bfloat16, seed=1)

    def step(args, dout):
        x, a, b = args["x"], args["a"], args["b"]
        out = mlx_amd.adapter_matmul(**args)
        return (out, *torch.autograd.grad(out, (x, a, b), dout))

    for args, dout in ((args, dout), (rows, drows)):
        held = {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in args.items()}
        for n in "xab":
            held[n].requires_grad_()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step(held, dout)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(held, dout)
        for n in range(4):
            new = {**args, "x": torch.randn_like(args["x"]), "indices": args["indices"].roll(n)}
            with torch.no_grad():
                held["x"].copy_(new["x"])
                held["indices"].copy_(new["indices"])
            graph.replay()
            for name in "xab":
                new[name] = new[name].detach().requires_grad_()
            want = step(new, dout)
            torch.cuda.synchronize()
            for one, two in zip(got, want):
                assert torch.equal(one, two)


def test_beside_a_quantized_projection(gpu):
    """The layer: its product and its gradients are the projection's and the adapters' together."""
    torch.manual_seed(0)
    base = nn.QuantizedLinear(128, 192, bias=False, device="cuda", dtype=torch.bfloat16)
    layer = nn.LoRALinear(base, rank=8, adapters=3, scale=2.0)
    x = torch.randn(4, 5, 128, device="cuda").to(torch.bfloat16)
    indices = torch.tensor([2, -1, 0, 2]).cuda()
    assert torch.equal(layer(x, indices), base(x))  # b starts at zero
    with torch.no_grad():
        layer.lora_b.normal_()
    out = layer(x, indices)
    assert torch.equal(out, mlx_amd.adapter_matmul(x, layer.lora_a, layer.lora_b, indices, scale=2.0,
                                                   y=base(x)))
    assert torch.equal(out[1], base(x)[1])
    x.requires_grad_()
    dout = torch.randn_like(out)
    dx, da, db = torch.autograd.grad(layer(x, indices), (x, layer.lora_a, layer.lora_b), dout)
    alone, = torch.autograd.grad(base(x), x, dout)
    assert torch.equal(dx[1], alone[1]) and not torch.equal(dx[0], alone[0])
    assert (da[1] == 0).all() and (db[1] == 0).all() and (da[0] != 0).any()
    names = {n for n, p in layer.named_parameters()}
    assert names == {"lora_a", "lora_b"}  # the projection is frozen


@pytest.mark.parametrize("dtype", (torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64, torch.uint16,
                                   torch.uint32, torch.uint64))
def test_indices_of_every_type(gpu, dtype):
    """No adapter is what lies outside of them in the indices' own type."""
    args, _ = case(6, 2, 64, 48, 8, 3, torch.float32)
    most = torch.iinfo(dtype).max
    indices = [0, min(2 ** 32, most), 2, min(2 ** 32 + 1, most), min(2 ** 63, most), 1]
    got = mlx_amd.adapter_matmul(**{**args, "indices": torch.tensor(indices, dtype=dtype).cuda()})
    want = mlx_amd.adapter_matmul(
        **{**args, "indices": torch.tensor([0, -1, 2, -1, -1, 1], dtype=torch.int32).cuda()})
    assert torch.equal(got, want)


def whole(*shape, most, g, dtype):
    return torch.randint(0, most + 1, shape, generator=g).to(dtype).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T, r, odd", ((1, 8, 0), (3, 16, 1), (40, 16, 0), (40, 30, 0), (70, 64, 1), (70, 64, 0),
                                       (40, 128, 0), (5, 130, 0), (40, 256, 1)))
def test_sums_over_ranks_and_tokens_keep_their_32_bits(gpu, dtype, T, r, odd):
    """Whole numbers whose sums 32 bits hold (below 2**24; 2**23, where float16 keeps 23 bits of a
    token's h): what stays when they cancel is right to the last bit, and rounded once."""
    g = torch.Generator().manual_seed(T + r)
    half = dtype == torch.float16
    K = (64 if half else 256) + odd
    small, large = 255, 511 if half else 255

    def exactly(got, want):
        assert torch.equal(got.detach(), want.to(dtype)), float((got.detach().double() - want).abs().max())

    # out: h[n % r] 2**-10 beside a y that is nearly its opposite
    N = 2 * r + odd
    x, a = whole(T, K, most=large, g=g, dtype=dtype), whole(1, r, K, most=small, g=g, dtype=dtype)
    h = (x.double() @ a[0].double().T)[:, torch.arange(N) % r] * 2.0 ** -10
    assert float(h.max()) < 2.0 ** (13 if half else 14) and float(h.max()) > 2.0 ** 10
    b = torch.zeros((1, N, r), dtype=dtype, device="cuda")
    b[0, torch.arange(N), torch.arange(N) % r] = 2.0 ** -10
    y = -h.to(torch.bfloat16).to(dtype)
    exactly(mlx_amd.adapter_matmul(x, a, b, y=y), h + y.double())
    # h[2 j] - h[2 j + 1], whose rows of a differ in one place
    even = r - r % 2
    a = whole(1, r, K, most=small - 1, g=g, dtype=dtype)
    a[0, 1:even:2] = a[0, :even:2]
    a[0, 1:even:2, K // 3] += 1
    b = torch.zeros((1, N, r), dtype=dtype, device="cuda")
    b[0, torch.arange(N), torch.arange(N) % (even // 2) * 2] = 1.0
    b[0, torch.arange(N), torch.arange(N) % (even // 2) * 2 + 1] = -1.0
    exactly(mlx_amd.adapter_matmul(x, a, b), x.double() @ a[0].double().T @ b[0].double().T)
    # dx: g[2 j] - g[2 j + 1], whose columns of b differ in one place
    x, a = torch.ones((T, 2 * r + odd), dtype=dtype, device="cuda"), torch.zeros((1, r, 2 * r + odd), dtype=dtype)
    n = torch.arange(even)
    a[0, n, n // 2] = 1.0 - 2.0 * (n % 2).to(dtype)
    b = whole(1, K, r, most=small - 1, g=g, dtype=dtype)
    b[0, :, 1:even:2] = b[0, :, :even:2]
    b[0, K // 3, 1:even:2] += 1
    a = a.cuda()
    dout = whole(T, K, most=large, g=g, dtype=dtype)
    x.requires_grad_()
    dx, = torch.autograd.grad(mlx_amd.adapter_matmul(x, a, b), x, dout)
    exactly(dx, dout.double() @ b[0].double() @ a[0].double())
    # da and db: pairs of tokens that cancel but for one place; 16 tokens that are not zero, of 2**20 each
    T = max(T, 16)
    at = torch.randperm(T, generator=g)[:16].cuda()
    sign = torch.zeros((T, 1), dtype=dtype, device="cuda")
    sign[at[:8]], sign[at[8:]] = 1.0, -1.0
    pairs = whole(T, 256, most=63, g=g, dtype=dtype)
    pairs[at[8:]] = pairs[at[:8]]
    pairs[at[8:], 7] += 1
    weights = whole(1, 256, r, most=63, g=g, dtype=dtype)
    x, a = (sign * torch.ones((1, 40 + odd), dtype=dtype, device="cuda")), whole(1, r, 40 + odd, most=3, g=g, dtype=dtype)
    a.requires_grad_()
    da, = torch.autograd.grad(mlx_amd.adapter_matmul(x, a, weights), a, pairs)
    exactly(da[0], (pairs.double() @ weights[0].double()).T @ x.double())
    b = torch.zeros((1, 40 + odd, r), dtype=dtype, device="cuda", requires_grad=True)
    a = weights.transpose(1, 2).contiguous()
    db, = torch.autograd.grad(mlx_amd.adapter_matmul(pairs, a, b), b, sign.expand(T, 40 + odd))
    exactly(db[0], sign.expand(T, 40 + odd).double().T @ (pairs.double() @ a[0].double().T))
