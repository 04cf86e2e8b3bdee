"""Attention, its key-value cache and speculative decoding, as cases that can be timed.

A case is a dict of plain values.  ``listed()`` gives the ones that are looked at
first, ``draw(rng)`` one more of the same ranges, ``prepare`` what a program holds
before the call, ``run`` one pass -- through the package's operators where ``own``
is true, else in elementary torch operations in 32 bits -- ``work`` the bytes and
operations a pass cannot do without and ``exact`` the same results in 64 bits.

The kinds of case:

* ``append``: ``paged_cache_update``, new keys and values into the pages of a cache.
* ``paged``: ``paged_attention`` of the newest tokens of each sequence over such a
  cache: one token (decode), a few (drafted tokens), a chunk of a prompt.
* ``window``: ``window_attention`` over contiguous keys and values (a prompt).
* ``train``: the same with the gradients of q, k and v.
* ``verify``: ``verify_draft``, drafted tokens against the target's probabilities.

Token ``p`` of a sequence sees the tokens ``j <= p`` with ``p - j < window`` or
``j < keep``.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}

# (query heads, key heads, head size): the attention that goes with the layers (hidden, kv) =
# (4096, 1024), (3584, 512), (2048, 512), (8192, 1024), (4096, 4096), and odd ones
HEADS = ((32, 8, 128), (28, 4, 128), (32, 8, 64), (64, 8, 128), (32, 32, 128), (16, 16, 80),
         (8, 1, 256), (12, 4, 96))
NO_WINDOW = 1 << 30


def listed():
    return [
        # chat with one user: the token just made goes into the cache
        {"name": "append, 1 token", "kind": "append", "batch": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "new": 1, "longest": 515, "ragged": False, "page": 16, "dtype": "bfloat16"},
        # a batch of ragged prompts goes into the cache, padded in front
        {"name": "append, prompts", "kind": "append", "batch": 16, "heads": 28, "kv_heads": 4,
         "dim": 128, "new": 1531, "longest": 1531, "ragged": True, "page": 64, "dtype": "float16"},
        # the smallest decode step in use: one user, a short chat; latency is all
        {"name": "decode, 1 sequence", "kind": "paged", "batch": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "new": 1, "longest": 515, "ragged": False, "window": NO_WINDOW, "keep": 0,
         "page": 16, "dtype": "bfloat16"},
        # one user with a long document
        {"name": "decode, 65000 tokens", "kind": "paged", "batch": 1, "heads": 28, "kv_heads": 4,
         "dim": 128, "new": 1, "longest": 65000, "ragged": False, "window": NO_WINDOW, "keep": 0,
         "page": 64, "dtype": "float16"},
        # continuous batching: sequences of very different lengths
        {"name": "decode, 32 sequences", "kind": "paged", "batch": 32, "heads": 32, "kv_heads": 8,
         "dim": 128, "new": 1, "longest": 8192, "ragged": True, "window": NO_WINDOW, "keep": 0,
         "page": 16, "dtype": "bfloat16"},
        # five tokens at once (four drafted ones) with a window over a long cache
        {"name": "drafts, window", "kind": "paged", "batch": 8, "heads": 32, "kv_heads": 8,
         "dim": 64, "new": 5, "longest": 20011, "ragged": True, "window": 4096, "keep": 4,
         "page": 32, "dtype": "bfloat16"},
        # a chunk of a long prompt over what is in the cache already
        {"name": "prompt chunk", "kind": "paged", "batch": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "new": 2048, "longest": 32768, "ragged": False, "window": NO_WINDOW,
         "keep": 0, "page": 64, "dtype": "bfloat16"},
        # a prompt under a window
        {"name": "window, prompt", "kind": "window", "batch": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "new": 4096, "longest": 4096, "ragged": False, "window": 1024, "keep": 4,
         "dtype": "bfloat16"},
        # a step of tuning on long texts
        {"name": "train, 8192 tokens", "kind": "train", "batch": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "new": 8192, "longest": 8192, "ragged": False, "window": NO_WINDOW,
         "keep": 0, "dtype": "bfloat16"},
        # a step of tuning on a few short texts of odd lengths in the default type, padded in front
        {"name": "train, float32", "kind": "train", "batch": 3, "heads": 16, "kv_heads": 16,
         "dim": 80, "new": 509, "longest": 509, "ragged": True, "window": 128, "keep": 1,
         "dtype": "float32"},
        # a server's step of speculative decoding over the largest vocabulary of the benchmark
        {"name": "verify, 32 sequences", "kind": "verify", "batch": 32, "drafts": 4,
         "vocab": 128256, "dtype": "float32"},
        # one user, drafts without probabilities (looked up in the prompt)
        {"name": "verify, 1 sequence", "kind": "verify", "batch": 1, "drafts": 7,
         "vocab": 32000, "greedy": True, "dtype": "float32"},
    ]


def _log_int(rng: random.Random, low: int, high: int) -> int:
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(("append", "paged", "paged", "paged", "window", "train", "verify"))
    while True:
        dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float16", "float32"))
        if kind == "verify":
            return {"kind": kind, "batch": _log_int(rng, 1, 32), "drafts": rng.randrange(1, 9),
                    "vocab": _log_int(rng, 1000, 128256), "greedy": rng.random() < 0.3,
                    "dtype": rng.choice(("float32", "float32", dtype))}
        heads, kv_heads, dim = rng.choice(HEADS)
        case = {"kind": kind, "batch": _log_int(rng, 1, 32), "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "ragged": rng.random() < 0.5}
        if kind == "append":
            case["new"] = _log_int(rng, 1, 2048)
            case["longest"] = case["new"] + _log_int(rng, 1, 2048) - 1
        elif kind == "paged":
            case["new"] = rng.choice((1, 1, rng.randrange(2, 10), _log_int(rng, 10, 2048)))
            case["longest"] = max(case["new"], _log_int(rng, 100, 65536))
        else:
            case["new"] = _log_int(rng, 16, 8192)
            case["longest"] = case["new"] if rng.random() < 0.7 else \
                case["new"] + rng.randrange(1, 1024)
        if kind != "append":
            narrow = rng.random() < 0.5
            case["window"] = _log_int(rng, 16, 8192) if narrow else NO_WINDOW
            case["keep"] = rng.choice((0, 1, 4, 64)) if narrow else 0
        if kind in ("append", "paged"):
            case["page"] = rng.choice((16, 32, 64, 128, 48))
        case["dtype"] = dtype
        if _affordable(case):
            return case


def _affordable(case) -> bool:
    """Whether a case costs no more than the largest listed ones: the scores of the plain form,
    the cache, and the operations (float32's are slower)."""
    scores = case["batch"] * case["heads"] * case["new"] * case["longest"]
    cache = case["batch"] * case["kv_heads"] * case["longest"] * case["dim"]
    if case["kind"] == "append":
        return cache <= 16 * 4 * 1531 * 128
    slow = 8 if case["dtype"] == "float32" else 1
    wide = max(case["dim"], 128) / 128
    return cache <= 32 * 8 * 8192 * 128 and slow * wide * scores <= 32 * 8192 * 8192


def _lengths(case):
    """Tokens of each sequence, the newest included: the longest down to an eighth of it."""
    n, longest = case["batch"], case["longest"]
    if not case["ragged"] or n == 1:
        return [longest] * n
    return [max(1, round(longest * (1 + 7 * i / (n - 1)) / 8)) for i in range(n)]


# ---------------------------------------------------------------- preparation
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    if case["kind"] == "verify":
        b, k, v = case["batch"], case["drafts"], case["vocab"]
        # logits of a trained model: a few likely tokens, a long tail; the draft is near them
        logits = 3.0 * torch.randn((b, k + 1, v), generator=g, device="cuda")
        target = torch.softmax(logits, -1)
        logits = logits[:, :k] + torch.randn((b, k, v), generator=g, device="cuda")
        probs = torch.softmax(logits, -1)
        draft = torch.multinomial(probs.reshape(b * k, v), 1, generator=g).reshape(b, k)
        return {"kind": "verify", "draft": draft.to(torch.int32), "target": target.to(dtype),
                "probs": None if case.get("greedy") else probs.to(dtype),
                "accept": uniform(b, k), "sample": uniform(b)}

    b, h, kv, d, n = (case[x] for x in ("batch", "heads", "kv_heads", "dim", "new"))
    lengths = _lengths(case)
    order = torch.randperm(b, generator=torch.Generator().manual_seed(seed)).tolist()
    lengths = torch.tensor([lengths[i] for i in order], dtype=torch.int32, device="cuda")
    s = {"kind": case["kind"], "lengths": lengths, "scale": d ** -0.5,
         "window": case.get("window"), "keep": case.get("keep")}

    # activations as projections leave them: [B, L, H, D] in memory, seen as [B, H, L, D]
    def heads_of(count, length):
        return normal(b, length, count, d).transpose(1, 2)

    if case["kind"] in ("append", "paged"):
        page = case["page"]
        per = -(-case["longest"] // page)
        pages = b * per + 8
        table = torch.randperm(pages, generator=g, device="cuda")[:b * per]
        s["table"] = table.reshape(b, per).to(torch.int32)
        s["k_pages"], s["v_pages"] = (normal(pages, kv, page, d) for _ in range(2))
        if case["kind"] == "append":
            s["k"], s["v"] = heads_of(kv, n), heads_of(kv, n)
        else:
            s["q"] = heads_of(h, n)
        return s
    if not case["ragged"]:
        s["lengths"] = None
    s["q"], s["k"], s["v"] = heads_of(h, n), heads_of(kv, case["longest"]), heads_of(kv, case["longest"])
    if case["kind"] == "train":
        s["do"] = heads_of(h, n)
        for x in "qkv":
            s[x].requires_grad_()
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    import mlx_amd

    kind = s["kind"]
    if kind == "append":
        return mlx_amd.paged_cache_update(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"],
                                          s["lengths"])
    if kind == "paged":
        return mlx_amd.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"],
                                       s["lengths"], scale=s["scale"], window=s["window"],
                                       keep=s["keep"])
    if kind == "verify":
        return mlx_amd.verify_draft(s["draft"], s["target"], s["probs"], s["accept"], s["sample"])
    out = mlx_amd.window_attention(s["q"], s["k"], s["v"], scale=s["scale"], window=s["window"],
                                   keep=s["keep"], lengths=s["lengths"])
    if kind == "window":
        return out
    return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["do"]))


def _positions(lengths, new):
    """Of each sequence's newest tokens; negative ones are padding."""
    return lengths[:, None] - new + torch.arange(new, device=lengths.device)


def _visible(pos, keys, window, keep):
    j = torch.arange(keys, device=pos.device)
    p = pos[..., None]
    return (j <= p) & ((p - j < window) | (j < keep))


def _plain_probabilities(q, k, pos, scale, window, keep):
    """softmax of the visible scores, [B, kv heads, heads that share one, new, keys]."""
    b, h, n, d = q.shape
    kv, keys = k.shape[1:3]
    s = torch.matmul(q.reshape(b, kv, h // kv * n, d), k.transpose(-1, -2).contiguous()) * scale
    s = s.reshape(b, kv, h // kv, n, keys)
    hidden = ~_visible(pos, keys, window, keep)[:, None, None]
    s.masked_fill_(hidden, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp_(s.sub_(torch.where(m > -math.inf, m, 0.0)))
    total = p.sum(-1, keepdim=True)
    return p.div_(torch.where(total > 0, total, 1.0))


def _times_values(p, v):
    b, kv, shared, n, keys = p.shape
    return torch.matmul(p.reshape(b, kv, shared * n, keys), v).reshape(b, kv * shared, n, -1)


def _run_plain(s):
    kind = s["kind"]
    if kind == "append":
        return _plain_append(s)
    if kind == "verify":
        return _plain_verify(s)
    with torch.no_grad():
        dtype = s["q"].dtype
        q = s["q"].float()
        if kind == "paged":
            k, v = (x[s["table"].long()].transpose(1, 2).flatten(2, 3).float()
                    for x in (s["k_pages"], s["v_pages"]))
        else:
            k, v = s["k"].float(), s["v"].float()
        lengths = s["lengths"]
        if lengths is None:
            lengths = torch.full((q.shape[0],), k.shape[2], device=q.device)
        pos = _positions(lengths, q.shape[2])
        p = _plain_probabilities(q, k, pos, s["scale"], s["window"], s["keep"])
        out = _times_values(p, v)
        if kind != "train":
            return out.to(dtype)
        do = s["do"].float()
        b, kv, shared, n, keys = p.shape
        rows = (b, kv, shared * n, -1)
        dv = torch.matmul(p.reshape(rows).transpose(-1, -2), do.reshape(rows))
        dp = torch.matmul(do.reshape(rows), v.transpose(-1, -2)).reshape(p.shape)
        delta = (do * out).sum(-1).reshape(b, kv, shared, n, 1)
        ds = dp.sub_(delta).mul_(p).mul_(s["scale"]).reshape(rows)
        dq = torch.matmul(ds, k).reshape(q.shape)
        dk = torch.matmul(ds.transpose(-1, -2), q.reshape(rows))
        return tuple(x.to(dtype) for x in (out, dq, dk, dv))


def _plain_append(s):
    k_pages, v_pages = s["k_pages"], s["v_pages"]
    page = k_pages.shape[2]
    pos = _positions(s["lengths"], s["k"].shape[2])
    row, i = torch.nonzero(pos >= 0, as_tuple=True)
    pos = pos[row, i]
    to, slot = s["table"][row, pos // page].long(), pos % page
    k_pages[to, :, slot] = s["k"][row, :, i]
    v_pages[to, :, slot] = s["v"][row, :, i]
    return k_pages, v_pages


def _plain_verify(s):
    draft, target, probs = s["draft"].long(), s["target"], s["probs"]
    b, k = draft.shape
    vocab = target.shape[-1]
    seq = torch.arange(b, device=draft.device)
    p_at = target[:, :k].gather(-1, draft[..., None])[..., 0].double()
    q_at = 1.0 if probs is None else probs.gather(-1, draft[..., None])[..., 0].double()
    taken = (s["accept"].double() * q_at < p_at).long().cumprod(-1)
    n = taken.sum(-1)
    p = target[seq, n].float()
    at = n.clamp(max=k - 1)
    if probs is None:
        w = torch.where(torch.arange(vocab, device=p.device) == draft[seq, at][:, None], 0.0, p)
    else:
        w = (p - probs[seq, at].float()).clamp(min=0)
    # weights as whole numbers of 2**-40: their sums have no order
    w = (torch.where((n < k)[:, None], w, p).clamp(max=1) * 2.0 ** 40).long()
    p = (p.clamp(max=1) * 2.0 ** 40).long()
    w = torch.where((w.sum(-1) > 0)[:, None], w, p)
    sums = w.cumsum(-1)
    total = sums[:, -1]
    t = torch.minimum((s["sample"].double() * total.double()).floor().long(), total - 1)
    token = (sums <= t[:, None]).sum(-1)
    i = torch.arange(k + 1, device=draft.device)
    tokens = torch.where(i < n[:, None], torch.nn.functional.pad(draft, (0, 1)), -1)
    tokens = torch.where(i == n[:, None], token[:, None], tokens)
    return tokens.to(torch.int32), n.to(torch.int32)


# ---------------------------------------------------------------- accounts
def _sum_min(first, last, most):
    """sum of min(p + 1, most) over positions p = first .. last"""
    first = max(first, 0)
    ramp = min(last, most - 1)  # up to here p + 1 counts
    total = 0
    if ramp >= first:
        total += (first + 1 + ramp + 1) * (ramp - first + 1) // 2
    flat = max(first, most)
    return total + most * max(0, last - flat + 1)


def work(case):
    size = SIZE[case["dtype"]]
    if case["kind"] == "verify":
        rows = 1 if case.get("greedy") else 2
        b, k = case["batch"], case["drafts"]
        return {"bytes": b * (rows * case["vocab"] * size + k * (4 + 4 + rows * size) + 4 * (k + 2)),
                "flops": 0}
    h, kv, d, new = (case[x] for x in ("heads", "kv_heads", "dim", "new"))
    lengths = _lengths(case)
    tokens = sum(min(n, new) for n in lengths)
    if case["kind"] == "append":
        return {"bytes": 2 * 2 * tokens * kv * d * size, "flops": 0}
    most = case["window"] + case["keep"]
    pairs = sum(_sum_min(n - new, n - 1, most) for n in lengths)
    seen = sum(min(n, most + min(n, new) - 1) for n in lengths)
    rows, keys = case["batch"] * new * h * d * size, seen * kv * d * size
    if case["kind"] == "train":
        # q, k, v, do read, out and three gradients written; two products forward, five backward
        return {"bytes": 4 * rows + 4 * keys, "flops": 7 * 2 * d * h * pairs}
    return {"bytes": 2 * rows + 2 * keys, "flops": 2 * 2 * d * h * pairs}


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "verify":
        return _exact_verify(s)
    if s["kind"] == "append":
        return _exact_append(s)
    keys = case["longest"]
    lengths = [keys] * case["batch"] if s["lengths"] is None else s["lengths"].tolist()
    shared = case["heads"] // case["kv_heads"]
    out = []
    for b, length in enumerate(lengths):
        if "table" in s:
            at = s["table"][b].long()
            k, v = (s[x][at].double().movedim(1, 0).flatten(1, 2) for x in ("k_pages", "v_pages"))
        else:
            k, v = s["k"][b].detach().double(), s["v"][b].detach().double()
        k, v = k[:, :length], v[:, :length]
        first = max(0, case["new"] - length)  # padding in front
        q = s["q"][b, :, first:].detach().double()
        p = torch.arange(length - q.shape[1], length, device=q.device)[:, None]
        j = torch.arange(length, device=q.device)[None]
        hidden = (j > p) | ((j <= p - case["window"]) & (j >= case["keep"]))
        parts = [[], [], [], []]
        for h in range(case["heads"]):
            kh, vh = k[h // shared], v[h // shared]
            prob = torch.softmax((q[h] @ kh.T * s["scale"]).masked_fill(hidden, -math.inf), -1)
            o = prob @ vh
            parts[0].append(_padded(o, first, 0))
            if s["kind"] == "train":
                do = s["do"][b, h, first:].double()
                dp = do @ vh.T
                ds = prob * (dp - (prob * dp).sum(-1, keepdim=True)) * s["scale"]
                after = keys - length
                for part, x in zip(parts[1:], (_padded(ds @ kh, first, 0),
                                               _padded(ds.T @ q[h], 0, after),
                                               _padded(prob.T @ do, 0, after))):
                    part.append(x)
        got = [torch.stack(x) for x in parts if x]
        got[2:] = [x.reshape(-1, shared, *x.shape[1:]).sum(1) for x in got[2:]]
        out.append(got)
    out = tuple(torch.stack(x) for x in zip(*out))
    return out if s["kind"] == "train" else out[0]


def _padded(x, before, after):
    return torch.cat([x.new_zeros(before, x.shape[1]), x, x.new_zeros(after, x.shape[1])])


def _exact_append(s):
    pages = [s["k_pages"].double(), s["v_pages"].double()]
    page, new = pages[0].shape[2], s["k"].shape[2]
    tables = s["table"].tolist()
    for b, length in enumerate(s["lengths"].tolist()):
        for to, x in zip(pages, (s["k"], s["v"])):
            at = max(0, length - new)
            while at < length:
                end = min(length, (at // page + 1) * page)
                i = new - length + at
                to[tables[b][at // page], :, at % page:at % page + end - at] = \
                    x[b, :, i:i + end - at].double()
                at = end
    return tuple(pages)


def _exact_verify(s):
    drafts = s["draft"].tolist()
    accept, sample = s["accept"].double().tolist(), s["sample"].double().tolist()
    tokens, counts = [], []
    for b, draft in enumerate(drafts):
        n = 0
        while n < len(draft):
            q = 1.0 if s["probs"] is None else float(s["probs"][b, n, draft[n]])
            if not accept[b][n] * q < float(s["target"][b, n, draft[n]]):
                break
            n += 1
        p = s["target"][b, n].float().cpu().numpy()
        w = p.copy()
        if n < len(draft):
            if s["probs"] is None:
                w[draft[n]] = 0
            else:
                w = np.maximum(p - s["probs"][b, n].float().cpu().numpy(), np.float32(0))
        whole = [np.floor(np.minimum(x, 1).astype(np.float64) * 2.0 ** 40).astype(np.int64)
                 for x in (w, p)]
        c = whole[0] if whole[0].sum() else whole[1]
        total = int(c.sum())
        t = min(math.floor(sample[b] * float(total)), total - 1)
        token = int(np.searchsorted(np.cumsum(c), t, side="right"))
        tokens.append(draft[:n] + [token] + [-1] * (len(draft) - n))
        counts.append(n)
    return (torch.tensor(tokens, dtype=torch.int32), torch.tensor(counts, dtype=torch.int32))
