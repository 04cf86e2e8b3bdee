"""What else stands around a decoder's quantized projections, as cases that can be timed.

A case is a dict of plain values.  ``listed()`` gives the ones that are looked at
first, ``draw(rng)`` one more of the same ranges, ``prepare`` what a program holds
before the call, ``run`` one pass -- through the package's operators where ``own``
is true, else in elementary torch operations in 32 bits (angles, and scores that
decide between experts, in 64) -- ``work`` the bytes and operations a pass cannot do
without and ``exact`` the same results in 64 bits.

The kinds of case:

* ``route``: ``route_experts``, the experts of each token and their weights; with
  ``train`` the gradient of the logits.
* ``rope``: ``rope``, queries rotated by their positions along one or more axes; with
  ``train`` the gradient.
* ``append``: ``rope_cache_update``, queries and keys rotated and keys and values
  written into the pages of a cache.
* ``adapt``: ``adapter_matmul``, what a low-rank adapter of each request adds to a
  shared projection; with ``train`` the gradients of x and of the adapters.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}

# (query heads, key heads, head size)
HEADS = ((32, 8, 128), (28, 4, 128), (32, 8, 64), (64, 8, 128), (32, 32, 128), (16, 16, 80),
         (8, 1, 256), (12, 4, 96))
# (inputs, outputs) of a projection
LAYERS = ((4096, 4096), (4096, 1024), (4096, 14336), (14336, 4096), (3584, 512), (2048, 512),
          (8192, 1024), (2048, 1408), (1056, 2080), (1024, 1001))
# (experts, chosen, groups, chosen groups)
EXPERTS = ((8, 2, 1, 1), (64, 6, 1, 1), (64, 8, 1, 1), (60, 4, 1, 1), (128, 8, 1, 1),
           (160, 6, 8, 3), (256, 8, 8, 4), (16, 1, 1, 1), (384, 8, 1, 1), (512, 10, 1, 1))


def listed():
    return [
        # one token of one chat chooses its experts: latency is all
        {"name": "route, 1 token", "kind": "route", "rows": 1, "experts": 64, "chosen": 6,
         "groups": 1, "top_groups": 1, "scoring": "softmax", "bias": False, "normalize": True,
         "train": False, "dtype": "bfloat16"},
        # prompts: sigmoid scores, a bias for balance, half of the groups
        {"name": "route, prompts, groups", "kind": "route", "rows": 16384, "experts": 256,
         "chosen": 8, "groups": 8, "top_groups": 4, "scoring": "sigmoid", "bias": True,
         "normalize": True, "train": False, "dtype": "float32"},
        # tuning of a model whose experts are no power of two, odd number of tokens
        {"name": "route, train", "kind": "route", "rows": 32749, "experts": 60, "chosen": 4,
         "groups": 1, "top_groups": 1, "scoring": "softmax", "bias": False, "normalize": False,
         "train": True, "dtype": "float16"},
        # queries of texts with images: positions in time, height and width; tuning
        {"name": "rope, images, train", "kind": "rope", "batch": 4, "heads": 28, "dim": 128,
         "length": 2500, "axes": 3, "dims": 128, "traditional": False, "first": 0, "train": True,
         "dtype": "bfloat16"},
        # neighbouring columns of a part of each head, far into a long text, float32
        {"name": "rope, part of the head", "kind": "rope", "batch": 1, "heads": 16, "dim": 80,
         "length": 1021, "axes": 1, "dims": 32, "traditional": True, "first": 120000,
         "train": False, "dtype": "float32"},
        # chat with one user: the newest token
        {"name": "append, 1 token", "kind": "append", "batch": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "new": 1, "longest": 515, "ragged": False, "page": 16, "axes": 1,
         "dims": 128, "traditional": False, "dtype": "bfloat16"},
        # continuous batching: one token of each of many sequences
        {"name": "append, 48 sequences", "kind": "append", "batch": 48, "heads": 64, "kv_heads": 8,
         "dim": 128, "new": 1, "longest": 8192, "ragged": True, "page": 64, "axes": 1,
         "dims": 128, "traditional": False, "dtype": "float16"},
        # a batch of ragged prompts, padded in front
        {"name": "append, prompts", "kind": "append", "batch": 16, "heads": 28, "kv_heads": 4,
         "dim": 128, "new": 1531, "longest": 1531, "ragged": True, "page": 64, "axes": 1,
         "dims": 128, "traditional": False, "dtype": "bfloat16"},
        # one user with an adapter of their own: latency
        {"name": "adapt, 1 token", "kind": "adapt", "batch": 1, "length": 1, "inputs": 4096,
         "outputs": 4096, "rank": 16, "adapters": 8, "train": False, "dtype": "bfloat16"},
        # many users, hardly two with the same adapter
        {"name": "adapt, 48 requests", "kind": "adapt", "batch": 48, "length": 1, "inputs": 4096,
         "outputs": 14336, "rank": 64, "adapters": 64, "train": False, "dtype": "bfloat16"},
        # prompts of several users
        {"name": "adapt, prompts", "kind": "adapt", "batch": 13, "length": 601, "inputs": 14336,
         "outputs": 4096, "rank": 32, "adapters": 16, "train": False, "dtype": "float16"},
        # tuning of one adapter
        {"name": "adapt, train", "kind": "adapt", "batch": 4, "length": 2048, "inputs": 4096,
         "outputs": 14336, "rank": 16, "adapters": 1, "train": True, "dtype": "bfloat16"},
    ]


def _log_int(rng: random.Random, low: int, high: int) -> int:
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(("route", "rope", "append", "append", "adapt", "adapt"))
    while True:
        case = {"kind": kind}
        if kind == "route":
            experts, chosen, groups, top = rng.choice(EXPERTS)
            case.update(rows=_log_int(rng, 1, 32768), experts=experts, chosen=chosen,
                        groups=groups, top_groups=top,
                        scoring=rng.choice(("softmax", "sigmoid")), bias=rng.random() < 0.4,
                        normalize=rng.random() < 0.6, train=rng.random() < 0.4)
        elif kind == "adapt":
            inputs, outputs = rng.choice(LAYERS)
            long = rng.random() < 0.5
            case.update(batch=_log_int(rng, 1, 16 if long else 64),
                        length=_log_int(rng, 2, 2048) if long else 1, inputs=inputs,
                        outputs=outputs, rank=rng.choice((4, 8, 12, 16, 32, 64, 128)),
                        adapters=_log_int(rng, 1, 64), train=long and rng.random() < 0.5)
        else:
            heads, kv_heads, dim = rng.choice(HEADS)
            case.update(batch=_log_int(rng, 1, 48 if kind == "append" else 16), heads=heads,
                        dim=dim, axes=rng.choice((1, 1, 3)),
                        dims=rng.choice((dim, dim, dim // 2)), traditional=rng.random() < 0.3)
            if kind == "rope":
                case.update(length=_log_int(rng, 1, 4096), train=rng.random() < 0.5)
                case["first"] = _log_int(rng, 1, 131072) - 1 if case["axes"] == 1 else 0
            else:
                case.update(kv_heads=kv_heads, ragged=rng.random() < 0.5,
                            new=rng.choice((1, rng.randrange(2, 10), _log_int(rng, 10, 2048))),
                            page=rng.choice((16, 32, 64, 128, 48)))
                case["longest"] = case["new"] + _log_int(rng, 1, 8192) - 1
        case["dtype"] = rng.choice(("bfloat16", "bfloat16", "float16", "float16", "float32"))
        if _affordable(case):
            return case


def _affordable(case) -> bool:
    """Whether a case costs no more than the largest listed one of its kind."""
    if case["kind"] == "route":
        return case["rows"] * case["experts"] <= 16384 * 256
    if case["kind"] == "rope":
        return case["batch"] * case["heads"] * case["length"] * case["dim"] <= 4 * 28 * 2500 * 128
    if case["kind"] == "append":
        cache = case["batch"] * case["kv_heads"] * case["longest"] * case["dim"]
        tokens = case["batch"] * case["new"] * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        return cache <= 48 * 8 * 8192 * 128 and tokens <= 16 * 1531 * 36 * 128
    slow = 4 if case["dtype"] == "float32" else 1
    tokens = case["batch"] * case["length"]
    return slow * tokens * (case["inputs"] + case["outputs"]) * max(case["rank"], 16) <= \
        8192 * (4096 + 14336) * 16


def _lengths(case):
    """Tokens of each sequence, the newest included: the longest down to an eighth of it."""
    n, longest = case["batch"], case["longest"]
    if not case["ragged"] or n == 1:
        return [longest] * n
    return [max(1, round(longest * (1 + 7 * i / (n - 1)) / 8)) for i in range(n)]


def _sections(case):
    """How many pairs of columns each axis rotates; None for one axis."""
    if case["axes"] == 1:
        return None
    half = case["dims"] // 2
    time = half // 4
    height = (half - time) // 2
    return (time, height, half - time - height)


def _adapter_of(case):
    """The adapter of each request; one request in eight has none, if there are that many."""
    rng = random.Random(case["batch"] * 1009 + case["adapters"])
    return [-1 if i % 8 == 7 else rng.randrange(case["adapters"]) for i in range(case["batch"])]


# ---------------------------------------------------------------- preparation
def _grid_positions(length, first):
    """[3, length]: some text, an image of 24 columns, some text; ``first`` where it begins."""
    text = min(length, max(1, length // 5))
    cells = min(length - text, length * 3 // 5)
    rows = -(-cells // 24)
    i = torch.arange(cells)
    image = torch.stack((torch.zeros_like(i), i // 24, i % 24)) + text
    after = text + max(rows, min(cells, 24)) + torch.arange(length - text - cells)
    return torch.cat((torch.arange(text).expand(3, text), image, after.expand(3, len(after))), 1) + first


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    kind = case["kind"]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    def leaf(t):
        return t.requires_grad_() if case["train"] else t

    if kind == "route":
        rows, experts = case["rows"], case["experts"]
        s = {"k": case["chosen"], "scoring": case["scoring"], "groups": case["groups"],
             "top_groups": case["top_groups"], "normalize": case["normalize"], "bias": None,
             "scale": 2.5 if case["scoring"] == "sigmoid" else 1.0,
             "group_best": 2 if case["bias"] and case["groups"] > 1 else 1,
             "logits": leaf(normal(rows, experts, std=1.7))}
        if case["bias"]:  # moved by steps of a thousandth
            bias = torch.randn((experts,), generator=g, device="cuda") * 50
            s["bias"] = bias.round() * 0.001
        if case["train"]:
            s["grad"] = normal(rows, case["chosen"])
    elif kind == "adapt":
        b, n, inputs, outputs, r = (case[x] for x in ("batch", "length", "inputs", "outputs", "rank"))
        s = {"x": leaf(normal(b, n, inputs)), "y": normal(b, n, outputs),
             "a": leaf(normal(case["adapters"], r, inputs, std=inputs ** -0.5)),
             "b": leaf(normal(case["adapters"], outputs, r, std=0.3 * r ** -0.5)),
             "indices": torch.tensor(_adapter_of(case), dtype=torch.int32, device="cuda"),
             "scale": 2.0}
        if case["train"]:
            s["grad"] = normal(b, n, outputs)
    else:
        # activations as projections leave them: [B, L, H, D] in memory, seen as [B, H, L, D]
        def heads_of(count, length):
            return normal(b, length, count, d).transpose(1, 2)

        b, d, h = case["batch"], case["dim"], case["heads"]
        s = {"dims": case["dims"], "traditional": case["traditional"], "base": 500000.0,
             "sections": _sections(case), "positions": None}
        if kind == "rope":
            n, first = case["length"], case["first"]
            at = first + torch.arange(n) if case["axes"] == 1 else _grid_positions(n, first)
            s["positions"] = at.to(torch.int32).unsqueeze(-2).expand(
                *at.shape[:-1], b, n).contiguous().cuda()
            s["x"] = leaf(heads_of(h, n))
            if case["train"]:
                s["grad"] = heads_of(h, n)
        else:
            kv, n, page = case["kv_heads"], case["new"], case["page"]
            lengths = _lengths(case)
            order = torch.randperm(b, generator=torch.Generator().manual_seed(seed)).tolist()
            lengths = [lengths[i] for i in order]
            if case["axes"] > 1:
                s["positions"] = torch.stack([
                    torch.nn.functional.pad(_grid_positions(x, 0), (max(n - x, 0), 0))[:, -n:]
                    for x in lengths], 1).to(torch.int32).contiguous().cuda()
            per = -(-case["longest"] // page)
            pages = b * per + 8
            table = torch.randperm(pages, generator=g, device="cuda")[:b * per]
            s["table"] = table.reshape(b, per).to(torch.int32)
            s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
            s["k_pages"], s["v_pages"] = (normal(pages, kv, page, d) for _ in range(2))
            s["q"], s["k"], s["v"] = heads_of(h, n), heads_of(kv, n), heads_of(kv, n)
    s["kind"] = kind
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return _run_own(s) if own else _run_plain(s)


_ROUTING = ("scoring", "bias", "groups", "top_groups", "group_best", "normalize", "scale")
_ROTATION = ("dims", "traditional", "base", "sections")


def _run_own(s):
    import mlx_amd

    if s["kind"] == "route":
        indices, weights = mlx_amd.route_experts(s["logits"], s["k"], **{x: s[x] for x in _ROUTING})
        if "grad" not in s:
            return indices, weights
        return (indices, weights.detach(),
                *torch.autograd.grad(weights, (s["logits"],), s["grad"]))
    if s["kind"] == "adapt":
        out = mlx_amd.adapter_matmul(s["x"], s["a"], s["b"], s["indices"], scale=s["scale"], y=s["y"])
        if "grad" not in s:
            return out
        return (out.detach(), *torch.autograd.grad(out, (s["x"], s["a"], s["b"]), s["grad"]))
    rotation = {x: s[x] for x in _ROTATION}
    if s["kind"] == "rope":
        out = mlx_amd.rope(s["x"], s["positions"], **rotation)
        if "grad" not in s:
            return out
        return (out.detach(), *torch.autograd.grad(out, (s["x"],), s["grad"]))
    return mlx_amd.rope_cache_update(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"],
                                     s["lengths"], positions=s["positions"], **rotation)


def _run_plain(s):
    with torch.no_grad():
        return {"route": _plain_route, "adapt": _plain_adapt, "rope": _plain_rope,
                "append": _plain_append}[s["kind"]](s)


def _plain_route(s):
    logits = s["logits"]
    rows, experts = logits.shape
    x = logits.double()
    if s["scoring"] == "sigmoid":
        scores = 1 / (1 + torch.exp(-x))
    else:
        scores = torch.exp(x - x.amax(-1, keepdim=True))
        scores = scores / scores.sum(-1, keepdim=True)
    # without a bias or sums the logits themselves have the scores' order
    choice = scores if s["bias"] is not None or s["group_best"] > 1 else x
    if s["bias"] is not None:
        choice = choice + s["bias"].double()
    if s["top_groups"] < s["groups"]:
        best = choice.reshape(rows, s["groups"], -1).sort(dim=-1, descending=True)[0]
        best = best[..., :s["group_best"]].sum(-1)
        taken = best.sort(dim=-1, descending=True, stable=True)[1][:, :s["top_groups"]]
        open_ = torch.zeros_like(best, dtype=torch.bool).scatter_(1, taken, True)
        open_ = open_.repeat_interleave(experts // s["groups"], 1)
        choice = torch.where(open_, choice, -math.inf)
    indices = choice.sort(dim=-1, descending=True, stable=True)[1][:, :s["k"]]
    scores = scores.float()
    chosen = scores.gather(1, indices)
    total = chosen.sum(-1, keepdim=True) if s["normalize"] else 1.0
    weights = chosen / total
    out = (indices.to(torch.int32), (weights * s["scale"]).to(logits.dtype))
    if "grad" not in s:
        return out
    grad = s["grad"].float() * s["scale"]
    if s["normalize"]:
        grad = (grad - (grad * weights).sum(-1, keepdim=True)) / total
    grad = torch.zeros_like(scores).scatter_(1, indices, grad)
    if s["scoring"] == "sigmoid":
        grad = grad * scores * (1 - scores)
    else:
        grad = scores * (grad - (grad * scores).sum(-1, keepdim=True))
    return (*out, grad.to(logits.dtype))


def _plain_adapt(s):
    x, a, b, y = (s[name].float() for name in ("x", "a", "b", "y"))
    dtype = s["x"].dtype
    at = s["indices"].long()
    scale = torch.where(at >= 0, s["scale"], 0.0)[:, None, None]
    at = at.clamp(min=0)
    a_of, b_of = a[at], b[at]  # one of each request
    h = torch.matmul(x, a_of.transpose(1, 2).contiguous()) * scale
    out = (y + torch.matmul(h, b_of.transpose(1, 2).contiguous())).to(dtype)
    if "grad" not in s:
        return out
    grad = s["grad"].float()
    g = torch.matmul(grad, b_of) * scale
    dx = torch.matmul(g, a_of)
    da = torch.zeros_like(a).index_add_(0, at, torch.matmul(g.transpose(1, 2).contiguous(), x))
    db = torch.zeros_like(b).index_add_(0, at, torch.matmul(grad.transpose(1, 2).contiguous(), h))
    return out, dx.to(dtype), da.to(dtype), db.to(dtype)


def _angles(s, positions):
    """[B, L, dims / 2] in 64 bits; ``positions`` [B, L] or [axes, B, L]"""
    half = s["dims"] // 2
    rate = s["base"] ** (-torch.arange(half, dtype=torch.float64, device=positions.device) / half)
    if s["sections"] is None:
        return positions.double()[..., None] * rate
    axis = torch.repeat_interleave(
        torch.arange(len(s["sections"]), device=positions.device),
        torch.tensor(s["sections"], device=positions.device))
    return positions.double()[axis].permute(1, 2, 0) * rate


def _rotate(s, x, angles):
    dims, half = s["dims"], s["dims"] // 2
    cos, sin = angles.cos().float()[:, None], angles.sin().float()[:, None]
    x = x.float()
    out = x.clone()
    one, two = (slice(0, dims, 2), slice(1, dims, 2)) if s["traditional"] else \
        (slice(0, half), slice(half, dims))
    a, b = x[..., one], x[..., two]
    out[..., one] = a * cos - b * sin
    out[..., two] = b * cos + a * sin
    return out


def _plain_rope(s):
    angles = _angles(s, s["positions"])
    out = _rotate(s, s["x"], angles).to(s["x"].dtype)
    return (out, _rotate(s, s["grad"], -angles).to(out.dtype)) if "grad" in s else out


def _plain_append(s):
    k_pages, v_pages, lengths = s["k_pages"], s["v_pages"], s["lengths"]
    page, new, dtype = k_pages.shape[2], s["q"].shape[2], s["q"].dtype
    slots = lengths[:, None] - new + torch.arange(new, device=lengths.device)
    angles = _angles(s, slots if s["positions"] is None else s["positions"])
    q = _rotate(s, s["q"], angles).to(dtype)
    q = torch.where((slots >= 0)[:, None, :, None], q, 0)  # the others are padding
    k = _rotate(s, s["k"], angles).to(dtype)
    row, i = torch.nonzero(slots >= 0, as_tuple=True)
    slot = slots[row, i]
    to, slot = s["table"][row, slot // page].long(), slot % page
    k_pages[to, :, slot] = k[row, :, i]
    v_pages[to, :, slot] = s["v"][row, :, i]
    return q, k_pages, v_pages


# ---------------------------------------------------------------- accounts
def work(case):
    size = SIZE[case["dtype"]]
    train = case.get("train", False)
    if case["kind"] == "route":
        rows, experts, chosen = case["rows"], case["experts"], case["chosen"]
        out = {"bytes": rows * (experts * size + chosen * (4 + size)), "flops": 0}
        if train:  # the gradient of the weights in, that of the logits out
            out["bytes"] += rows * (chosen + experts) * size
        return out
    if case["kind"] == "rope":
        n = case["batch"] * case["heads"] * case["length"] * case["dim"] * size
        return {"bytes": (4 if train else 2) * n, "flops": 0}
    if case["kind"] == "append":
        tokens = sum(min(n, case["new"]) for n in _lengths(case))
        heads = case["heads"] + 2 * case["kv_heads"]
        return {"bytes": 2 * tokens * heads * case["dim"] * size, "flops": 0}
    inputs, outputs, rank, n = (case[x] for x in ("inputs", "outputs", "rank", "length"))
    of = _adapter_of(case)
    tokens = case["batch"] * n
    adapted = sum(x >= 0 for x in of) * n
    weights = len({x for x in of if x >= 0}) * rank * (inputs + outputs)
    # x and y in, the sum out
    elements = adapted * inputs + 2 * tokens * outputs + weights
    flops = 2 * adapted * rank * (inputs + outputs)
    if train:  # the gradient in, those of x, a and b out
        elements += tokens * (inputs + outputs) + case["adapters"] * rank * (inputs + outputs)
        flops *= 3
    return {"bytes": elements * size, "flops": flops}


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "adapt": _exact_adapt, "rope": _exact_rope,
            "append": _exact_append}[s["kind"]](s)


def _exact_route(s):
    x = s["logits"].detach().double().requires_grad_()
    score = torch.sigmoid(x) if s["scoring"] == "sigmoid" else torch.softmax(x, -1)
    with torch.no_grad():
        if s["bias"] is None and s["group_best"] == 1:
            left = x.detach().clone()
        else:
            left = score + (0 if s["bias"] is None else s["bias"].double())
        number = torch.arange(x.shape[1], device=x.device)
        group = number // (x.shape[1] // s["groups"])

        def largest(values):
            """Column of the largest of each row, the first of equal ones."""
            top = values.amax(1, keepdim=True)
            columns = torch.arange(values.shape[1], device=values.device)
            return torch.where(values == top, columns, values.shape[1]).amin(1, keepdim=True)

        if s["top_groups"] < s["groups"]:
            marks = []
            for n in range(s["groups"]):
                mine = left[:, group == n].clone()
                mark = torch.zeros_like(mine[:, :1])
                for _ in range(s["group_best"]):
                    at = largest(mine)
                    mark += mine.gather(1, at)
                    mine.scatter_(1, at, -math.inf)
                marks.append(mark)
            marks = torch.cat(marks, 1)
            open_ = torch.zeros_like(marks, dtype=torch.bool)
            for _ in range(s["top_groups"]):
                at = largest(marks)
                open_.scatter_(1, at, True)
                marks.scatter_(1, at, -math.inf)
            left[~open_[:, group]] = -math.inf
        chosen = []
        for _ in range(s["k"]):
            chosen.append(largest(left))
            left.scatter_(1, chosen[-1], -math.inf)
        chosen = torch.cat(chosen, 1)
    weights = score.gather(1, chosen)
    if s["normalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    weights = weights * s["scale"]
    out = (chosen.to(torch.int32), weights.detach())
    if "grad" in s:
        out += torch.autograd.grad(weights, (x,), s["grad"].double())
    return out


def _exact_adapt(s):
    grads = [torch.zeros_like(s[name], dtype=torch.float64) for name in ("x", "a", "b")]
    out = s["y"].double()
    for i, n in enumerate(s["indices"].tolist()):
        if n < 0:
            continue
        x, a, b = s["x"][i].detach().double(), s["a"][n].detach().double(), s["b"][n].detach().double()
        out[i] += s["scale"] * ((x @ a.T) @ b.T)
        if "grad" in s:
            back = s["scale"] * s["grad"][i].double()
            grads[0][i] = (back @ b) @ a
            grads[1][n] += (back @ b).T @ x
            grads[2][n] += back.T @ (x @ a.T)
    return (out, *grads) if "grad" in s else out


def _turned(s, x, positions, sign=1):
    """Pairs of columns as complex numbers, times those of their angles.  x [H, L, D],
    positions [axes, L]"""
    dims, half = s["dims"], s["dims"] // 2
    sections = s["sections"] or (half,)
    angles, pair = [], 0
    for axis, count in enumerate(sections):
        for _ in range(count):
            angles.append(positions[axis].double() * math.exp(-math.log(s["base"]) * pair / half))
            pair += 1
    turn = torch.polar(torch.ones_like(angles[0]).expand(half, -1), sign * torch.stack(angles)).T
    x = x.detach().double()
    if s["traditional"]:
        pairs = x[..., :dims].unflatten(-1, (half, 2))
    else:
        pairs = x[..., :dims].unflatten(-1, (2, half)).transpose(-1, -2)
    pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    if not s["traditional"]:
        pairs = pairs.transpose(-1, -2)
    return torch.cat((pairs.flatten(-2), x[..., dims:]), -1)


def _exact_rope(s):
    at = s["positions"].unsqueeze(0) if s["positions"].dim() == 2 else s["positions"]
    batch = range(s["x"].shape[0])
    out = torch.stack([_turned(s, s["x"][b], at[:, b]) for b in batch])
    if "grad" not in s:
        return out
    return out, torch.stack([_turned(s, s["grad"][b], at[:, b], -1) for b in batch])


def _exact_append(s):
    pages = [s["k_pages"].double(), s["v_pages"].double()]
    page, new = pages[0].shape[2], s["k"].shape[2]
    q = torch.zeros_like(s["q"], dtype=torch.float64)
    tables = s["table"].tolist()
    for b, length in enumerate(s["lengths"].tolist()):
        first = max(0, new - length)  # padding in front
        slots = torch.arange(length - new + first, length, device=q.device)
        at = slots[None] if s["positions"] is None else s["positions"][:, b, first:]
        q[b, :, first:] = _turned(s, s["q"][b, :, first:], at)
        k, v = _turned(s, s["k"][b, :, first:], at), s["v"][b, :, first:].double()
        slot = length - new + first
        done = 0
        while slot < length:
            end = min(length, (slot // page + 1) * page)
            for to, x in zip(pages, (k, v)):
                to[tables[b][slot // page], :, slot % page:slot % page + end - slot] = \
                    x[:, done:done + end - slot]
            done += end - slot
            slot = end
    return (q, *pages)
