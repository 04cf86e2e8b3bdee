"""rope and rope_cache_update against rotations in 64 bits."""
import ctypes
import math

import pytest
import torch

import mlx_amd
from mlx_amd import _lib

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
TYPES = (torch.float32, torch.float16, torch.bfloat16)


def reference(x, positions, dims=None, traditional=False, base=10000.0, scale=1.0, freqs=None,
              sections=None, sign=1.0):
    """(value, bound) in 64 bits.  Cosine and sine are off by 3 * 2**-24 at most (two units of
    values up to 1, and the rounding of the angle that is left), each product and the sum by
    2**-24 of their size, the result by half a step of the type."""
    dtype, x = x.dtype, x.detach().double()
    D = x.shape[-1]
    dims = D if dims is None else dims
    half = dims // 2
    if positions.dim() == 2:
        positions, sections = positions[None], (half,)
    axis = [i for i, n in enumerate(sections) for _ in range(n)]
    if freqs is None:
        freqs = [base ** (i / half) for i in range(half)]
    freqs = torch.as_tensor(freqs, dtype=torch.float64, device=x.device)
    angle = positions.double()[axis].permute(1, 2, 0)[:, None] * scale / freqs
    cos, sin = angle.cos(), sign * angle.sin()
    one, two = (slice(0, dims, 2), slice(1, dims, 2)) if traditional else \
        (slice(0, half), slice(half, dims))
    a, b = x[..., one], x[..., two]
    out, size = x.clone(), torch.zeros_like(x)
    out[..., one], out[..., two] = a * cos - b * sin, b * cos + a * sin
    size[..., one] = size[..., two] = a.abs() + b.abs()
    turned = size > 0
    bound = 5 * 2.0 ** -24 * size + torch.where(
        turned, HALF_STEP[dtype] * out.abs() + SMALLEST[dtype], 0.0)
    return out, bound


def close(got, want):
    value, bound = want
    assert got.isfinite().all()
    off = (got.detach().double() - value).abs() - bound
    assert float(off.max()) <= 0, float(off.max())


def normal(*shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).cuda()


def positions_of(B, L, axes=None, first=0, seed=0):
    g = torch.Generator().manual_seed(seed + 77)
    shape = (B, L) if axes is None else (axes, B, L)
    return (first + torch.randint(0, 5000, shape, generator=g)).cuda()


OPTIONS = (
    dict(D=128),
    dict(D=64, traditional=True),
    dict(D=80, dims=40, traditional=True),
    dict(D=80, dims=32),
    dict(D=96, dims=12, scale=0.25, base=500.0),
    dict(D=18, dims=6),
    dict(D=6, dims=2),
    dict(D=2, traditional=True),
    dict(D=256, sections=(32, 48, 48)),
    dict(D=128, sections=(1, 0, 30, 33), traditional=True),
    dict(D=64, dims=64, freqs=True),
    dict(D=300, dims=256),
)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("options", OPTIONS, ids=str)
@pytest.mark.parametrize("B, H, L", ((1, 1, 1), (3, 5, 7), (2, 32, 1), (1, 3, 2100)))
def test_rope_and_its_gradient(gpu, dtype, options, B, H, L):
    options = dict(options)
    D, sections = options.pop("D"), options.get("sections")
    if options.get("freqs"):
        options["freqs"] = torch.logspace(0, 3, 32, dtype=torch.float32).cuda()
    x, dout = normal(B, H, L, D, dtype=dtype), normal(B, H, L, D, dtype=dtype, seed=1)
    at = positions_of(B, L, sections and len(sections))
    x.requires_grad_()
    out = mlx_amd.rope(x, at, **options)
    assert out.shape == x.shape and out.dtype == dtype
    close(out, reference(x, at, **options))
    dx, = torch.autograd.grad(out, x, dout)
    close(dx, reference(dout, at, **options, sign=-1.0))


@pytest.mark.parametrize("dtype", (torch.int32, torch.int64, torch.uint32))
def test_far_and_negative_positions(gpu, dtype):
    at = torch.tensor([[0, 1, 2 ** 20 + 3, 2 ** 31 - 1]])
    if dtype != torch.uint32:
        at = torch.cat((at, torch.tensor([[-5, -2 ** 31]])), 1)
    x = normal(1, 2, at.shape[1], 64, dtype=torch.float32)
    # Angles up to 2**31 are off by some five roundings of 2**-53 on each side: 10 * 2**-22 at most,
    # which each of a pair's columns feels
    value, bound = reference(x, at.cuda())
    far = 10 * 2.0 ** -22 * 2 * float(x.abs().max())
    close(mlx_amd.rope(x, at.to(dtype).cuda()), (value, bound + far))
    near = at.abs() <= 2 ** 21
    got = mlx_amd.rope(x, at.to(dtype).cuda())[:, :, near[0]]
    close(got, (value[:, :, near[0]], bound[:, :, near[0]]))


def test_strides_and_memory_order(gpu):
    at = positions_of(2, 9)
    base = normal(2, 9, 6, 3, 64, dtype=torch.bfloat16)  # queries, keys and values side by side
    x = base[:, :, :, 1].transpose(1, 2)
    want = reference(x, at)
    out = mlx_amd.rope(x, at)
    close(out, want)
    dense = x.transpose(1, 2).contiguous().transpose(1, 2)
    out = mlx_amd.rope(dense, at)
    assert out.stride() == dense.stride()
    close(out, want)
    odd = normal(2, 6, 9, 67, dtype=torch.bfloat16)[..., 1:65]  # rows that are not aligned
    close(mlx_amd.rope(odd, at), reference(odd, at))
    columns = normal(2, 6, 64, 9, dtype=torch.float16).transpose(2, 3)  # columns that are not dense
    close(mlx_amd.rope(columns, at), reference(columns, at))
    shared = normal(1, 1, 9, 64, dtype=torch.float32).expand(2, 6, 9, 64)
    close(mlx_amd.rope(shared, at), reference(shared, at))
    one = torch.arange(9).cuda().expand(2, 9)  # positions shared by the sequences
    close(mlx_amd.rope(x, one), reference(x, one))


def test_derivatives_of_derivatives_and_differences(gpu):
    x = normal(1, 2, 5, 32, dtype=torch.float32).requires_grad_()
    at = positions_of(1, 5)
    out = mlx_amd.rope(x, at, dims=16)
    d = normal(1, 2, 5, 32, dtype=torch.float32, seed=2).requires_grad_()
    dx, = torch.autograd.grad(out, x, d, create_graph=True)
    back, = torch.autograd.grad(dx, d, torch.ones_like(dx))
    close(back, reference(torch.ones_like(x), at, dims=16))
    # linear: differences of any size are the derivative
    step = normal(1, 2, 5, 32, dtype=torch.float32, seed=3)
    up, down = (reference(x + s * step, at, dims=16)[0] for s in (1, -1))
    want = float(((up - down) / 2 * d.double()).sum())
    size = float((x.abs().double() + step.abs().double()).sum() * d.abs().max())
    assert abs(float((dx.double() * step.double()).sum()) - want) <= 20 * 2.0 ** -24 * size


def test_values_that_are_not_finite_stay_in_their_pairs(gpu):
    x = normal(1, 2, 3, 64, dtype=torch.float16)
    clean = mlx_amd.rope(x, positions_of(1, 3))
    x[0, 1, 2, 5] = math.inf
    x[0, 0, 1, 40] = math.nan
    out = mlx_amd.rope(x, positions_of(1, 3))
    hit = torch.zeros_like(x, dtype=torch.bool)
    hit[0, 1, 2, [5, 37]] = hit[0, 0, 1, [8, 40]] = True
    assert not out[hit].isfinite().any() and torch.equal(out[~hit], clean[~hit])


def test_empty(gpu):
    for shape in ((0, 2, 3, 8), (2, 0, 3, 8), (2, 2, 0, 8)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        out = mlx_amd.rope(x, torch.zeros((shape[0], shape[2]), dtype=torch.int64, device="cuda"))
        assert out.shape == x.shape
        assert torch.autograd.grad(out.sum(), x)[0].shape == x.shape


def test_offsets_beyond_32_bits(gpu):
    rows, D = 3, 64
    apart = 2 ** 31 // 2 + 8 * 131
    buffer = torch.zeros(apart * rows, dtype=torch.bfloat16, device="cuda")
    x = buffer.as_strided((1, 2, rows, D), (0, D, apart, 1))
    x.copy_(normal(1, 2, rows, D, dtype=torch.bfloat16))
    close(mlx_amd.rope(x, positions_of(1, rows)), reference(x, positions_of(1, rows)))


# ---------------------------------------------------------------- into the cache
def update_case(dtype, B, Hq, Hkv, L, D, page, lengths, seed=0):
    width = max(1, -(-max(max(lengths), L) // page))
    pages = B * width + 3
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(pages, generator=g)[:B * width].reshape(B, width).to(torch.int32).cuda()
    q, k, v = (normal(B, L, h, D, dtype=dtype, seed=seed + i).transpose(1, 2)
               for i, h in enumerate((Hq, Hkv, Hkv)))
    k_pages, v_pages = (normal(pages, Hkv, page, D, dtype=dtype, seed=seed + 3 + i) for i in range(2))
    return dict(q=q, k=k, v=v, k_pages=k_pages, v_pages=v_pages, block_table=table,
                lengths=torch.tensor(lengths, dtype=torch.int32).cuda())


def check_update(case, got, before, positions=None, **options):
    """Rotated queries and pages; whatever is not written stays bit for bit."""
    q, k_pages, v_pages = got
    L, page = case["q"].shape[2], before[0].shape[2]
    lengths = case["lengths"].tolist()
    slots = torch.tensor([[n - L + i for i in range(L)] for n in lengths]).cuda()
    at = slots if positions is None else positions
    value, bound = reference(case["q"], at, **options)
    padding = (slots < 0)[:, None, :, None].expand_as(q)
    assert (q[padding] == 0).all()
    close(torch.where(padding, 0, q), (value.masked_fill(padding, 0), bound))
    keys, off = reference(case["k"], at, **options)
    want_k, off_k, want_v = before[0].double(), torch.zeros_like(before[0], dtype=torch.float64), before[1].clone()
    for b in range(len(lengths)):
        for i in range(L):
            s = int(slots[b, i])
            if 0 <= s < case["block_table"].shape[1] * page:
                to = int(case["block_table"][b, s // page])
                if 0 <= to < want_v.shape[0]:
                    want_k[to, :, s % page], off_k[to, :, s % page] = keys[b, :, i], off[b, :, i]
                    want_v[to, :, s % page] = case["v"][b, :, i]
    assert torch.equal(v_pages, want_v)
    close(k_pages, (want_k, off_k))


UPDATES = (
    (1, 1, 1, 1, 64, 16, [1]),
    (2, 8, 2, 1, 128, 16, [17, 1]),
    (3, 4, 4, 7, 80, 48, [7, 3, 100]),
    (4, 6, 3, 33, 96, 32, [40, 0, 33, 5]),
    (1, 40, 8, 3, 256, 64, [200]),
    (2, 3, 1, 2049, 32, 128, [2049, 70]),
)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B, Hq, Hkv, L, D, page, lengths", UPDATES)
def test_rope_cache_update(gpu, dtype, B, Hq, Hkv, L, D, page, lengths):
    case = update_case(dtype, B, Hq, Hkv, L, D, page, lengths)
    before = case["k_pages"].clone(), case["v_pages"].clone()
    versions = case["k_pages"]._version, case["v_pages"]._version
    got = mlx_amd.rope_cache_update(**case, base=500.0)
    assert got[1] is case["k_pages"] and got[2] is case["v_pages"]
    assert (got[1]._version, got[2]._version) == tuple(n + 1 for n in versions)
    check_update(case, got, before, base=500.0)


@pytest.mark.parametrize("options", (dict(dims=40, traditional=True), dict(sections=(10, 14, 16)),
                                     dict(sections=(40,), scale=0.5)), ids=str)
def test_rope_cache_update_options(gpu, options):
    case = update_case(torch.bfloat16, 2, 4, 2, 9, 80, 16, [30, 5])
    before = case["k_pages"].clone(), case["v_pages"].clone()
    sections = options.get("sections")
    positions = positions_of(2, 9, sections and len(sections))
    check_update(case, mlx_amd.rope_cache_update(**case, positions=positions, **options), before,
                 positions, **options)


def test_it_is_rope_and_paged_cache_update(gpu):
    """Bit for bit what the two operators give one after the other; attention reads it."""
    for dtype in TYPES:
        case = update_case(dtype, 3, 8, 2, 5, 64, 16, [40, 5, 17])
        two = [case["k_pages"].clone(), case["v_pages"].clone()]
        at = case["lengths"][:, None].long() - 5 + torch.arange(5, device="cuda")
        q = mlx_amd.rope(case["q"], at)
        mlx_amd.paged_cache_update(mlx_amd.rope(case["k"], at), case["v"], *two, case["block_table"],
                                   case["lengths"])
        got = mlx_amd.rope_cache_update(**case)
        for x, y in zip(got, (q, *two)):
            assert torch.equal(x, y)
        out = [mlx_amd.paged_attention(x, *pages, case["block_table"], case["lengths"], scale=0.125)
               for x, pages in ((got[0], got[1:]), (q, two))]
        assert torch.equal(*out)


def test_places_that_do_not_exist(gpu):
    """Lengths past the table's room and pages that are none: nothing is written there."""
    case = update_case(torch.float16, 3, 2, 2, 4, 64, 16, [16, 16, 16])
    case["lengths"] = torch.tensor([18, 16, 400], dtype=torch.int32, device="cuda")
    case["block_table"][1, 0] = -7
    before = case["k_pages"].clone(), case["v_pages"].clone()
    check_update(case, mlx_amd.rope_cache_update(**case), before)
    case["block_table"][1, 0] = 1 << 20
    before = case["k_pages"].clone(), case["v_pages"].clone()
    check_update(case, mlx_amd.rope_cache_update(**case), before)


def test_a_cache_without_pages(gpu):
    """Queries turn, nothing is written, and neither table nor pages are read: they may be null."""
    case = update_case(torch.bfloat16, 2, 4, 2, 3, 64, 16, [5, 3])
    out = torch.full_like(case["q"], math.nan)
    strides = (ctypes.c_int64 * 19)(*(s for t in (case["q"], case["k"], case["v"], out) for s in t.stride()[:3]))
    at = case["lengths"][:, None].long() - 3 + torch.arange(3, device="cuda")
    for pages, width in ((0, 7), (0, 0), (5, 0)):
        status = _lib.load().mlxrocm_rope_cache_update(
            *(case[n].data_ptr() for n in "qkv"), out.data_ptr(), None, None, None, case["lengths"].data_ptr(),
            2, 4, 2, 3, 64, pages, 16, width, strides, None, None, 0, 1, None, 64, 0, 1e4, 1.0, None, 2,
            torch.cuda.current_stream().cuda_stream)
        assert status == _lib.OK
        close(out, reference(case["q"], at))
        out.fill_(math.nan)
    empty = {**case, "k_pages": case["k_pages"][:0], "v_pages": case["v_pages"][:0]}
    close(mlx_amd.rope_cache_update(**empty)[0], reference(case["q"], at))


def test_strided_pages_and_tables(gpu):
    case = update_case(torch.bfloat16, 2, 4, 2, 6, 64, 32, [40, 6])
    n, _, page, D = case["k_pages"].shape
    both = normal(n, 2, 2, page, D, dtype=torch.bfloat16)  # keys and values of a page together
    case["k_pages"], case["v_pages"] = both[:, 0], both[:, 1]
    wide = torch.zeros((2, 9), dtype=torch.int64, device="cuda")
    wide[:, :2] = case["block_table"]
    case["block_table"] = wide[:, :2]
    before = case["k_pages"].clone(), case["v_pages"].clone()
    check_update(case, mlx_amd.rope_cache_update(**case), before)


def test_captured_steps(gpu):
    """A captured step moves on with the lengths on the device, beside eager work of the same program."""
    case = update_case(torch.bfloat16, 2, 4, 2, 1, 64, 16, [20, 33])
    state = {n: t.clone() for n, t in case.items()}
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        mlx_amd.rope_cache_update(**state)  # (what is loaded at the first call is loaded)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, *_ = mlx_amd.rope_cache_update(**state)
        state["lengths"].add_(1)
    state["k_pages"].copy_(case["k_pages"])
    state["v_pages"].copy_(case["v_pages"])
    state["lengths"].fill_(0).add_(case["lengths"])
    for _ in range(4):
        graph.replay()
        want = mlx_amd.rope_cache_update(**case)
        torch.cuda.synchronize()
        assert torch.equal(out, want[0])
        case["lengths"].add_(1)
    assert torch.equal(state["k_pages"], case["k_pages"])
    assert torch.equal(state["v_pages"], case["v_pages"])


def test_another_stream(gpu):
    x = normal(2, 8, 300, 64, dtype=torch.bfloat16)
    at = positions_of(2, 300)
    want = mlx_amd.rope(x, at)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = mlx_amd.rope(x, at)
    stream.synchronize()
    assert torch.equal(out, want)
