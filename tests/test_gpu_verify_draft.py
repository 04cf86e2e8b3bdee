"""verify_draft against the same rules in Python integers and 64-bit floats."""
import math

import numpy as np
import pytest
import torch

import mlx_amd

pytestmark = pytest.mark.gpu


def oracle(draft, target, probs, accept, sample, lengths=None):
    B, K = draft.shape
    V = target.shape[2]
    target, probs = (None if x is None else x.float().cpu().numpy() for x in (target, probs))
    draft, accept, sample = (x.cpu().numpy() for x in (draft, accept, sample))
    tokens, counts = [], []
    for b in range(B):
        most = K if lengths is None else min(max(lengths[b], 0), K)
        n = 0
        while n < most:
            x = int(draft[b, n])
            if not 0 <= x < V:
                break
            q = 1.0 if probs is None else float(probs[b, n, x])
            if not float(accept[b, n]) * q < float(target[b, n, x]):
                break
            n += 1
        p = target[b, n]
        w = p.copy()
        if n < most:
            if probs is not None:
                w = p - probs[b, n]
            elif 0 <= draft[b, n] < V:
                w[draft[b, n]] = 0

        def whole(x):
            x = np.where(x > 0, np.minimum(x, np.float32(1)), np.float32(0))
            return (x.astype(np.float64) * 2.0 ** 40).astype(np.int64)

        c = whole(w)
        c = c if c.sum() else whole(p)
        total = int(c.sum())
        token = -1
        if total:
            t = min(math.floor(float(sample[b]) * float(total)), total - 1)
            token = int(np.searchsorted(np.cumsum(c), t, side="right"))
        tokens.append([int(x) for x in draft[b, :n]] + [token] + [-1] * (K - n))
        counts.append(n)
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(counts, dtype=torch.int32)


def case(gpu, B, K, V, dtype, seed, near=0.5):
    g = torch.Generator(device=gpu).manual_seed(seed)
    logits = 2 * torch.randn((B, K + 1, V), generator=g, device=gpu)
    target = torch.softmax(logits, -1).to(dtype)
    probs = torch.softmax(
        logits[:, :K] + near * torch.randn((B, K, V), generator=g, device=gpu), -1)
    draft = torch.multinomial(probs.reshape(B * K, V), 1, generator=g).reshape(B, K).int() \
        if K else torch.zeros((B, 0), dtype=torch.int32, device=gpu)
    accept = torch.rand((B, K), generator=g, device=gpu)
    sample = torch.rand((B,), generator=g, device=gpu)
    return draft, target, probs.to(dtype), accept, sample


def check(args, lengths=None):
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=args[0].device)
    tokens, accepted = mlx_amd.verify_draft(*args, lengths=n)
    want = oracle(*args, lengths)
    assert tokens.dtype == accepted.dtype == torch.int32
    assert torch.equal(accepted.cpu(), want[1])
    assert torch.equal(tokens.cpu(), want[0])
    return want


@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("B, K, V", ((1, 4, 1), (5, 1, 17), (3, 8, 4096), (40, 3, 4097),
                                     (2, 5, 128256), (2, 0, 1000), (2, 100, 65)))
def test_against_the_oracle(gpu, B, K, V, dtype):
    draft, target, probs, accept, sample = case(gpu, B, K, V, dtype, seed=V)
    check((draft, target, probs, accept, sample))
    check((draft, target, None, accept * 0.1, sample))
    check((draft, target, probs, accept, sample), [(i * 3) % (K + 2) for i in range(B)])


def test_edges(gpu):
    draft, target, probs, accept, sample = case(gpu, 8, 3, 300, torch.float32, seed=1)
    # equal distributions: everything is taken; a draw from the last row
    want = check((draft, torch.cat([probs, target[:, 3:]], 1), probs, accept, sample))
    assert (want[1] == 3).all()
    # nothing is left where a draft is refused: the draw is from the target itself
    same = torch.cat([probs, target[:, 3:]], 1)
    assert (check((draft, same, probs, torch.ones_like(accept), sample))[1] == 0).all()
    # the ends of the random numbers, and 1 although it is outside
    for u in (0.0, 1 - 2.0 ** -24, 1.0):
        check((draft, target, probs, accept, torch.full_like(sample, u)))
    # tokens that do not exist, rows without any probability, NaN
    wild = draft.clone()
    wild[::2, 1] = 300
    wild[1::2, 0] = -1
    check((wild, target, probs, accept, sample))
    check((wild, target, None, accept * 0.01, sample))
    none = target.clone()
    none[:4] = 0
    none[4:6, :, ::2] = math.nan
    want = check((draft, none, probs, accept, sample))
    assert (want[0][:4, 0] == -1).all()
    # one token has all of it
    sure = torch.zeros_like(target)
    sure[:, :, 299] = 1
    assert (check((draft, sure, probs, accept, sample))[0].max(1).values == 299).all()


def test_strides(gpu):
    draft, target, probs, accept, sample = case(gpu, 4, 3, 1001, torch.float32, seed=2)
    want = mlx_amd.verify_draft(draft, target, probs, accept, sample)
    wide = torch.zeros((4, 8, 1500), device=gpu)
    wide[:, ::2, 3:1004] = target
    views = (draft.long(), wide[:, ::2, 3:1004],
             probs.transpose(1, 2).contiguous().transpose(1, 2),
             accept.t().contiguous().t(), torch.stack([sample, sample], 1)[:, 0])
    got = mlx_amd.verify_draft(*views)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_result_is_distributed_as_the_target(gpu):
    """One draft of a vocabulary of 8 in many sequences: the first token's frequencies are the
    target's, within 6 standard deviations."""
    B, V = 60000, 8
    g = torch.Generator(device=gpu).manual_seed(3)
    p = torch.tensor([.3, .2, .15, .1, .1, .1, .05, 0.], device=gpu)
    q = torch.tensor([.05, .3, .15, .2, .05, .05, .1, .1], device=gpu)
    draft = torch.multinomial(q.expand(B, V), 1, generator=g).int()
    rand = lambda *s: torch.rand(s, generator=g, device=gpu)  # noqa: E731
    tokens, _ = mlx_amd.verify_draft(draft, p.expand(B, 2, V), q.expand(B, 1, V), rand(B, 1), rand(B))
    found = torch.bincount(tokens[:, 0].long(), minlength=V).double() / B
    sd = (p.double() * (1 - p.double()) / B).sqrt()
    assert ((found - p.double()).abs() <= 6 * sd + 1e-9).all()
