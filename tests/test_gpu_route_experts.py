"""route_experts against scores in 64 bits: indices are equal, weights and gradients as far off as
their roundings."""
import math

import pytest
import torch

import mlx_amd
from mlx_amd import nn

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
TYPES = (torch.float32, torch.float16, torch.bfloat16)
F = 2.0 ** -24


def reference(logits, k, scoring="softmax", bias=None, groups=1, top_groups=None, group_best=1,
              normalize=True, scale=1.0, grad=None):
    """indices, weights and the gradient of the logits, one row after the other in 64 bits (CPU)."""
    rows = logits.detach().double().cpu().reshape(-1, logits.shape[-1])
    E = rows.shape[1]
    top_groups = groups if top_groups is None else top_groups
    indices, weights, grads = [], [], []
    for n, l in enumerate(rows):
        if scoring == "sigmoid":
            s = torch.sigmoid(l)
        else:
            m = float(l.max())
            s = torch.zeros_like(l) if m == -math.inf else torch.exp(l - m) / torch.exp(l - m).sum()
        choice = (l if bias is None and not (group_best > 1 and top_groups < groups) else s).clone()
        if bias is not None:
            choice += bias.double().cpu()
        choice[l == -math.inf] = -math.inf
        order = choice.tolist()
        size = E // groups
        marks = [sum(sorted(order[g * size:(g + 1) * size], reverse=True)[:group_best])
                 for g in range(groups)]
        open_ = sorted(range(groups), key=lambda g: (-marks[g], g))[:top_groups]
        left = [e for e in range(E) if e // size in open_]
        chosen = sorted(left, key=lambda e: (-order[e], e))[:k]
        c = s[chosen]
        total = c.sum() if normalize else torch.ones(())
        w = c / total if total > 0 else torch.zeros_like(c)
        indices.append(chosen)
        weights.append(w * scale)
        if grad is not None:
            g = torch.zeros_like(l)
            up = grad.double().cpu().reshape(-1, k)[n] * scale
            if normalize:
                up = (up - (up * w).sum()) / total if total > 0 else torch.zeros_like(up)
            g[chosen] = up
            if scoring == "sigmoid":
                grads.append(g * s * torch.sigmoid(-l))
            else:
                grads.append(s * (g - (g * s).sum()))
    shape = (*logits.shape[:-1], k)
    out = [torch.tensor(indices, dtype=torch.int32).reshape(shape), torch.stack(weights).reshape(shape)]
    if grad is not None:
        out.append(torch.stack(grads).reshape(logits.shape))
    return out


def relative(logits):
    """How far a weight may be off before it is rounded: e^x by the rounding of x (differences up to the
    spread of the logits) and two units, for itself and for the sum; the sum by an addition for each
    of a lane's up to 64 values and the four steps over lanes, and four more operations."""
    finite = logits.detach().double()[logits.isfinite()]
    spread = float(finite.max() - finite.min()) if finite.numel() else 0.0
    return (2 * (spread + 4) + 64 + 4 + 4) * F


def check(logits, k, seed=5, **options):
    dtype = logits.dtype
    g = torch.Generator().manual_seed(seed)
    grad = torch.randn((*logits.shape[:-1], k), generator=g).to(dtype).cuda()
    logits = logits.cuda().requires_grad_()
    indices, weights = mlx_amd.route_experts(logits, k, **options)
    assert indices.dtype == torch.int32 and weights.dtype == dtype and not indices.requires_grad
    plain = mlx_amd.route_experts(logits.detach(), k, **options)
    assert torch.equal(plain[0], indices) and torch.equal(plain[1], weights.detach())
    dl, = torch.autograd.grad(weights, logits, grad)
    want = reference(logits, k, grad=grad, **options)
    assert torch.equal(indices.cpu(), want[0])
    off = (weights.detach().cpu().double() - want[1]).abs()
    bound = (relative(logits) + HALF_STEP[dtype]) * want[1].abs() + SMALLEST[dtype]
    assert float((off - bound).max()) <= 0, float((off - bound).max())
    # each term of the gradient is a product of at most three such numbers; a sum of k terms
    scale = abs(options.get("scale", 1.0))
    size = k * scale * float(grad.abs().max())
    off = (dl.cpu().double() - want[2]).abs()
    bound = (3 * relative(logits) + (k + 8) * F) * 2 * size + HALF_STEP[dtype] * want[2].abs() + SMALLEST[dtype]
    assert float((off - bound).max()) <= 0, float((off - bound).max())
    return indices, weights, dl


def logits_of(*shape, dtype, std=2.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype)


SHAPES = ((1, 1, 1, 1, 1), (3, 2, 1, 1, 1), (5, 8, 2, 1, 1), (17, 60, 4, 1, 1), (33, 64, 6, 4, 2),
          (9, 256, 8, 8, 4), (16, 160, 6, 8, 3), (2, 384, 8, 1, 1), (2, 1024, 32, 16, 5),
          (4, 48, 17, 3, 2), (3, 45, 20, 5, 5), (2, 16, 1, 16, 1), (7, 33, 33 - 1, 1, 1),
          (3, 130, 9, 13, 4), (2, 1000, 10, 1, 1))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows, experts, k, groups, top", SHAPES)
@pytest.mark.parametrize("scoring", ("softmax", "sigmoid"))
def test_route_experts_and_its_gradient(gpu, dtype, rows, experts, k, groups, top, scoring):
    logits = logits_of(rows, experts, dtype=dtype)
    bias = torch.randn((experts,), generator=torch.Generator().manual_seed(1)).mul(50).round() * 0.001
    best = 2 if experts // groups > 1 else 1
    for options in (dict(), dict(normalize=False), dict(bias=bias.cuda(), scale=2.5),
                    dict(group_best=best, scale=-0.5), dict(bias=bias.cuda(), group_best=best,
                                                            normalize=False)):
        check(logits, k, scoring=scoring, groups=groups, top_groups=top, **options)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scoring", ("softmax", "sigmoid"))
def test_equal_ones_go_by_index(gpu, dtype, scoring):
    logits = torch.randint(-2, 3, (40, 96), generator=torch.Generator().manual_seed(2)).to(dtype)
    logits[0] = 0
    logits[1] = torch.tensor([0.0, -0.0] * 48)
    bias = torch.randint(0, 2, (96,), generator=torch.Generator().manual_seed(3)).float().cuda()
    for options in (dict(), dict(bias=bias), dict(groups=8, top_groups=3),
                    dict(groups=8, top_groups=3, group_best=2, bias=bias)):
        indices, *_ = check(logits, 12, scoring=scoring, **options)
    assert mlx_amd.route_experts(logits[:2].cuda(), 5)[0].tolist() == [[0, 1, 2, 3, 4]] * 2


def test_choices_that_differ_in_the_last_bits(gpu):
    """Choices apart by less than 32 bits hold: their order is that of 64 bits."""
    base = 0.25
    logits = torch.zeros((1, 64))
    bias = torch.full((64,), base)
    order = torch.randperm(64, generator=torch.Generator().manual_seed(4))
    # sigmoid(l) near 1/2 moves by l / 4: logits a few 2**-30 apart, scores 2**-32 apart
    logits[0, order] = torch.arange(64, dtype=torch.float32) * 2.0 ** -30
    indices, _ = mlx_amd.route_experts(logits.cuda(), 32, scoring="sigmoid", bias=bias.cuda())
    assert indices[0].tolist() == order.flip(0)[:32].tolist()
    logits = torch.tensor([[1.0, 1.0 - 2.0 ** -24, 1.0 - 2.0 ** -23, 0.0] * 4])
    check(logits, 9, bias=torch.zeros(16, device="cuda"))


@pytest.mark.parametrize("k", (1, 3, 8, 15, 16, 20))
@pytest.mark.parametrize("near", (2.0 ** -21, 2.0 ** -24, 2.0 ** -27, 0.0))
def test_choices_in_near_pairs(gpu, k, near):
    """Two or three choices, or groups, nearer to each other than 32 bits can tell: in 64 they have an
    order, whichever way that is found."""
    g = torch.Generator().manual_seed(k)
    E, rows = 64, 24
    logits = (torch.randn((rows, E), generator=g) * 2).float()
    logits[:, 1::2] = logits[:, ::2]  # pairs of one score
    logits[4:8, 2::4] = logits[4:8, ::4]  # threes and fours
    bias = (torch.randn((E,), generator=g) * 0.1).float()
    bias[1::2] = (bias[::2].double() + near * torch.randn((E // 2,), generator=g).double()).float()
    bias[2::4] = bias[::4]
    logits[8:12, 32:] = logits[8:12, :32]  # groups that are alike but for that
    bias[32:] = bias[:32] + near
    for options in (dict(), dict(groups=4, top_groups=2), dict(groups=4, top_groups=2, group_best=2),
                    dict(groups=16, top_groups=8, group_best=2), dict(groups=2, top_groups=1, group_best=2)):
        for scoring in ("sigmoid", "softmax"):
            for b in (bias, bias * 64):  # (choices far from 1 have fewer bits behind the point)
                check(logits, k, scoring=scoring, bias=b.cuda(), **options)
    check(logits, k)
    check(logits * 2.0 ** -20, k, groups=4, top_groups=2)
    check(logits * 2.0 ** 20, k)


def test_masked_and_empty_rows(gpu):
    for dtype in TYPES:
        logits = logits_of(6, 32, dtype=dtype)
        logits[0] = -math.inf
        logits[1, 3:] = -math.inf
        logits[2, :30] = -math.inf
        logits[3] = torch.finfo(dtype).min
        bias = logits_of(32, dtype=torch.float32, std=0.1, seed=8).cuda()
        for options in (dict(), dict(normalize=False), dict(scoring="sigmoid"), dict(bias=bias),
                        dict(scoring="sigmoid", bias=bias, groups=4, top_groups=4, group_best=2)):
            indices, weights = mlx_amd.route_experts(logits.cuda(), 5, **options)
            want = reference(logits, 5, **options)
            assert torch.equal(indices.cpu(), want[0])
            assert (weights[0] == 0).all() and (weights[1, 3:] == 0).all()
            if options.get("scoring") != "sigmoid":
                off = (weights.cpu().double() - want[1]).abs()
                assert float((off - (relative(logits[4:]) + HALF_STEP[dtype]) * want[1]).max()) <= 0
            leaf = logits.cuda().requires_grad_()
            weights = mlx_amd.route_experts(leaf, 5, **options)[1]
            dl, = torch.autograd.grad(weights.float().square().sum(), leaf)
            assert dl.isfinite().all() and (dl[0] == 0).all() and (dl[1, 3:] == 0).all()


def test_tiny_sigmoids_keep_their_ratios(gpu):
    logits = torch.tensor([[-200.0, -201.0, -200.5, -300.0], [-95.0, 3.0, -95.0, -95.0]])
    _, weights = mlx_amd.route_experts(logits.cuda(), 2, scoring="sigmoid")
    w = 1 / (1 + math.exp(-0.5))
    assert weights[0].tolist() == pytest.approx([w, 1 - w], rel=1e-6)
    assert weights[1].tolist() == pytest.approx([1.0, 0.0], abs=1e-30)


def test_infinities_and_nan(gpu):
    inf, nan = math.inf, math.nan
    logits = torch.tensor([[0.0, inf, 1.0, inf, 2.0, 3.0], [0.0, nan, 1.0, 5.0, 2.0, 3.0],
                           [nan] * 6, [0.0, 1.0, 2.0, 3.0, 4.0, 5.0]]).cuda()
    indices, weights = mlx_amd.route_experts(logits, 3)
    assert indices.tolist() == [[1, 3, 5], [3, 5, 4], [0, 1, 2], [5, 4, 3]]
    assert weights[0].tolist() == [0.5, 0.5, 0.0] and weights[2].isnan().all()
    assert weights[1].isfinite().all()  # depends on the chosen logits alone
    clean = mlx_amd.route_experts(logits[3:], 3)[1]
    assert torch.equal(weights[3:], clean)
    whole = mlx_amd.route_experts(logits, 3, normalize=False)[1]
    assert whole[1].isnan().all() and whole[3].isfinite().all()
    indices, weights = mlx_amd.route_experts(logits, 6, scoring="sigmoid", normalize=False)
    assert indices.tolist()[1] == [3, 5, 4, 2, 0, 1] and weights[1].isnan().tolist() == [False] * 5 + [True]
    bias = torch.tensor([0.0, 0.0, nan, inf, -inf, 0.0], device="cuda")
    for row in (1, 3):
        indices, _ = mlx_amd.route_experts(logits[row:row + 1], 6, scoring="sigmoid", bias=bias)
        assert indices.tolist() == [[3, 5, 0, 1, 2, 4] if row == 1 else [3, 5, 1, 0, 2, 4]]


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_of_every_type(gpu, dtype):
    inf, nan = math.inf, math.nan
    logits = torch.tensor([[nan] * 6, [0.0, nan, 1.0, 5.0, 2.0, 3.0], [-inf, nan, -inf, 1.0, -inf, -inf],
                           [0.0, 1.0, 2.0, 3.0, 4.0, 5.0]], dtype=dtype).cuda().requires_grad_()
    for scoring in ("softmax", "sigmoid"):
        indices, weights = mlx_amd.route_experts(logits, 6, scoring=scoring)
        assert indices.tolist() == [[0, 1, 2, 3, 4, 5], [3, 5, 4, 2, 0, 1], [3, 0, 1, 2, 4, 5],
                                    [5, 4, 3, 2, 1, 0]]
        assert weights[:3].isnan().all() and weights[3].isfinite().all()
        dl, = torch.autograd.grad(weights.sum(), logits)
        assert dl[:3].isnan().any(1).all() and dl[3].isfinite().all()
        indices, weights = mlx_amd.route_experts(logits, 2, scoring=scoring)
        assert weights[0].isnan().all() and weights[[1, 3]].isfinite().all()
        assert weights[2].tolist() == [1.0, 0.0]  # the second is masked, index 0
    weights = mlx_amd.route_experts(logits, 6, scoring="sigmoid", normalize=False)[1]
    assert weights.isnan().tolist() == [[True] * 6, [False] * 5 + [True],
                                        [False, False, True, False, False, False], [False] * 6]


@pytest.mark.parametrize("dtype", TYPES)
def test_choices_that_all_are_nan_go_by_index(gpu, dtype):
    """One NaN makes NaN of a softmax: no choice that has such a score is before another."""
    logits = torch.tensor([[0.0, math.nan, 1.0, 5.0, 2.0, 3.0], [0.0, 1.0, 2.0, 3.0, 4.0, 5.0]],
                          dtype=dtype).cuda()
    bias = torch.tensor([0.0, 0.5, 3.0, 1.0, 4.0, 2.0], device="cuda")
    for options in (dict(bias=bias), dict(bias=bias, groups=2, top_groups=1),
                    dict(groups=2, top_groups=1, group_best=2)):
        indices, _ = mlx_amd.route_experts(logits, 3, **options)
        assert indices[0].tolist() == [0, 1, 2], options
        indices, _ = mlx_amd.route_experts(logits[1:], 3, **options)
        assert indices.tolist() == ([[4, 2, 5]] if options == dict(bias=bias) else
                                    [[4, 5, 3]] if "bias" in options else [[5, 4, 3]])


def test_shapes_strides_and_empties(gpu):
    wide = logits_of(2, 3, 5, 70, dtype=torch.bfloat16).cuda()
    want = reference(wide[..., 3:67], 4)
    indices, weights = mlx_amd.route_experts(wide[..., 3:67], 4)
    assert indices.shape == weights.shape == (2, 3, 5, 4) and torch.equal(indices.cpu(), want[0])
    turned = wide.transpose(0, 2)[..., :64]
    assert torch.equal(mlx_amd.route_experts(turned, 4)[0].cpu(), reference(turned, 4)[0])
    columns = wide.transpose(2, 3)
    assert torch.equal(mlx_amd.route_experts(columns, 2)[0].cpu(), reference(columns, 2)[0])
    shared = wide[0, 0, :1].expand(9, 70)
    assert torch.equal(mlx_amd.route_experts(shared, 4)[0].cpu(), reference(shared, 4)[0])
    assert mlx_amd.route_experts(wide[0, 0, 0], 4)[0].shape == (4,)
    leaf = wide[:, :0].detach().requires_grad_()
    indices, weights = mlx_amd.route_experts(leaf, 4)
    assert indices.shape == (2, 0, 5, 4)
    assert torch.autograd.grad(weights.sum(), leaf)[0].shape == leaf.shape


def test_gradient_against_differences(gpu):
    logits = logits_of(6, 24, dtype=torch.float32).cuda().requires_grad_()
    step = logits_of(6, 24, dtype=torch.float32, std=1.0, seed=9).cuda()
    for options in (dict(), dict(normalize=False), dict(scoring="sigmoid"),
                    dict(scoring="sigmoid", normalize=False, scale=3.0)):
        _, weights = mlx_amd.route_experts(logits, 5, **options)
        up = torch.cos(torch.arange(5, device="cuda") + 1.0)
        dl, = torch.autograd.grad((weights * up).sum(), logits)
        e = 1e-5
        at = [(reference(logits.detach().double() + s * e * step.double(), 5, **options)[1]
               * up.double().cpu()).sum() for s in (1, -1)]
        want = float(at[0] - at[1]) / (2 * e)
        # 32-bit gradients of 144 terms, and differences of third order in e
        assert abs(float((dl.double() * step.double()).sum()) - want) <= 144 * 64 * F + 1e-8


def test_rows_beyond_a_grid_of_blocks_and_the_gradient_of_expanded_ones(gpu):
    logits = logits_of(70001, 8, dtype=torch.float16).cuda().requires_grad_()
    indices, weights = mlx_amd.route_experts(logits, 2)
    top = torch.sort(logits.detach().float(), dim=-1, descending=True, stable=True)
    assert torch.equal(indices.long(), top[1][:, :2])
    want = torch.softmax(top[0][:, :2].double(), -1)
    assert float((weights.double() - want).abs().max()) <= 2.0 ** -11 + 100 * F
    dl, = torch.autograd.grad(weights.sum(), logits)  # an expanded gradient: the weights sum to 1
    assert float(dl.abs().max()) <= 2.0 ** -11


def test_replays_and_experts(gpu):
    """The router in front of the experts, captured and replayed on new hidden states."""
    torch.manual_seed(0)
    glu = nn.SwitchGLU(128, 192, 16, device="cuda", dtype=torch.bfloat16)
    gate = torch.randn(16, 128, device="cuda", dtype=torch.bfloat16) * 0.1
    x = torch.randn(12, 128, device="cuda", dtype=torch.bfloat16)

    def block(x):
        indices, weights = mlx_amd.route_experts(torch.nn.functional.linear(x, gate), 4)
        return indices, weights, (glu(x, indices) * weights[..., None]).sum(-2)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        block(x)
    torch.cuda.current_stream().wait_stream(stream)
    held = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(held)
    for _ in range(4):
        x = torch.randn_like(x)
        held.copy_(x)
        graph.replay()
        want = block(x)
        torch.cuda.synchronize()
        for got, ref in zip(out, want):
            assert torch.equal(got, ref)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("second, third", ((20.0, 18.0), (18.0, 20.0)))
def test_second_choices_of_a_group_that_are_equal_in_32_bits(gpu, dtype, second, third):
    """Sigmoids of 18, 19 and 20 are one number there: groups go by the larger of neighbours in 64."""
    logits = torch.full((1, 32), -10.0, dtype=dtype)
    logits[0, [0, 2, 3]] = torch.tensor([0.0, second, third], dtype=dtype)
    logits[0, [16, 18]] = torch.tensor([0.0, 19.0], dtype=dtype)
    bias = torch.zeros(32, device="cuda")
    bias[[0, 16]] = 1.0
    options = dict(scoring="sigmoid", bias=bias, groups=2, top_groups=1, group_best=2)
    indices, *_ = check(logits, 1, **options)
    assert indices.tolist() == [[0]]
    check(logits, 5, **options)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("experts, groups", ((32, 2), (48, 3), (256, 8), (240, 5), (1024, 4)))
def test_saturated_choices_of_groups(gpu, dtype, experts, groups):
    """One choice of each group stands out, the others are equal in 32 bits or masked out."""
    g = torch.Generator().manual_seed(experts)
    some = torch.tensor([-10.0, -10.0, -10.0, 17.0, 17.5, 18.0, 19.0, 20.0, -math.inf], dtype=dtype)
    logits = some[torch.randint(0, len(some), (33, experts), generator=g)]
    bias = torch.zeros(experts, device="cuda")
    size = experts // groups
    logits[:, ::size] = 0.0
    bias[::size] = 1.0
    for best in (1, 2):
        for k in (1, 8):
            check(logits, k, scoring="sigmoid", bias=bias, groups=groups, top_groups=groups // 2,
                  group_best=best)


@pytest.mark.parametrize("scoring", ("sigmoid", "softmax"))
@pytest.mark.parametrize("experts", (16, 256, 1024))
@pytest.mark.parametrize("size", (2.0 ** 17, 2097150.0, 2.0 ** 21, 3e6, 2.0 ** 24, 2.0 ** 33, 1e30))
def test_large_biases_keep_the_order_of_64_bits(gpu, scoring, experts, size):
    """A bias that forces experts leaves 32 bits nothing of their scores."""
    g = torch.Generator().manual_seed(experts)
    logits = torch.randn((12, experts), generator=g)
    bias = torch.zeros(experts, device="cuda")
    bias[:6] = size
    bias[6:9] = -size
    logits[:, 0], logits[:, 1] = 0.49, 0.532  # sigmoids of 0.62 and 0.63
    for k in (1, 2, 4, 9):
        check(logits, k, scoring=scoring, bias=bias)
    check(logits, 3, scoring=scoring, bias=bias, groups=4, top_groups=2, group_best=2)
    check(logits, 3, scoring=scoring, bias=-bias)


@pytest.mark.parametrize("experts, groups, top", ((48, 3, 2), (9, 1, 1), (36, 4, 2), (45, 5, 3), (130, 13, 6),
                                                  (96, 12, 5), (54, 6, 6)))
def test_groups_that_leave_lanes_without_experts(gpu, experts, groups, top):
    """No power of two of groups, or of experts of one; experts that are masked in front of a group."""
    g = torch.Generator().manual_seed(experts)
    logits = torch.randn((24, experts), generator=g) * 2
    logits[:8, 1::2] = logits[:8, :-1:2]  # pairs of one score
    size = experts // groups
    logits[6:12, ::size] = -math.inf
    logits[10:14, 1::size] = math.nan
    logits[12:18] += 20  # sigmoids that 32 bits do not tell apart
    bias = (torch.randn((experts,), generator=g) * 0.1).cuda()
    rows = [n for n in range(24) if not 10 <= n < 14]
    for scoring in ("sigmoid", "softmax"):
        for best in (1, 2):
            for b in (bias, bias.round(), None):
                options = dict(scoring=scoring, bias=b, groups=groups, top_groups=top, group_best=best)
                check(logits[rows], min(5, top * size), **options)
                # what is NaN is as if it were masked where others are left
                if scoring == "sigmoid" and size > 5:
                    got = mlx_amd.route_experts(logits.cuda(), 3, **options)[0]
                    assert torch.equal(got.cpu(), reference(logits.nan_to_num(-math.inf, math.inf, -math.inf),
                                                            3, **options)[0])
