"""Attention and its gradients from the formulas in 64 bits, with bounds on how far an
implementation may be off that keeps sums in float32 and rounds as documented."""
import math

import torch

ROUNDOFF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
NO_WINDOW = 1 << 30


def visible(Lq, Lk, lengths, window, keep, device):
    """[B, 1, Lq, Lk]"""
    n = torch.as_tensor(lengths, device=device).clamp(0, Lk)
    p = (n[:, None] - Lq + torch.arange(Lq, device=device))[:, None, :, None]
    j = torch.arange(Lk, device=device)
    return (j <= p) & ((p - j < (window or NO_WINDOW)) | (j < keep))


def reference(q, k, v, scale, window=None, keep=0, lengths=None, dout=None):
    """({name: value}, {name: bound}): out, and dq, dk, dv where dout is given."""
    dtype = q.dtype
    B, Hq, Lq, D = q.shape
    Hkv, Lk = k.shape[1:3]
    G = Hq // Hkv
    lengths = [Lk] * B if lengths is None else lengths
    seen = visible(Lq, Lk, lengths, window, keep, q.device)
    q, k, v = (x.detach().double() for x in (q, k, v))
    k, v = (x.repeat_interleave(G, 1) for x in (k, v))
    # what no query sees has no part in anything
    some = seen.any(2)[..., None]
    k, v = torch.where(some, k, 0.0), torch.where(some, v, 0.0)
    q = torch.where(seen.any(3)[..., None], q, 0.0)
    s = (q @ k.transpose(-1, -2)) * scale
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > -math.inf, m, 0.0))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    out = p @ v
    # A score is off by at most (D + 4) 2^-24 of the sum of its products' magnitudes, a
    # probability relatively by twice the worst of its row's, and by n 2^-24 for its sum; then
    # it is rounded to the type, as the result is.
    u = ROUNDOFF[dtype]
    f = 2.0 ** -24
    mags = (q.abs() @ k.abs().transpose(-1, -2) * abs(scale)).masked_fill(~seen, 0.0)
    f_p = 2 * (D + 4) * f * mags.amax(-1, keepdim=True) + (Lk + 8) * f
    rounding = u if dtype != torch.float32 else 0.0
    off_p = p * (f_p + rounding)
    values = {"out": out}
    p_v = p @ v.abs()
    bounds = {"out": off_p @ v.abs() + (Lk * f) * p_v + u * out.abs()}
    if dout is not None:
        do = torch.where(seen.any(3)[..., None], dout.double(), 0.0)
        dp = do @ v.transpose(-1, -2)
        delta = (do * out).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        # the sum of dout * out has out's own error in it
        off_delta = (do.abs() * (bounds["out"] + D * f * out.abs())).sum(-1, keepdim=True)
        off_dp = D * f * (do.abs() @ v.abs().transpose(-1, -2))
        off_ds = p * (off_dp + off_delta) + ds.abs() * (f_p + rounding + 4 * f)

        def shared(x):
            return x.reshape(B, Hkv, G, *x.shape[2:]).sum(2)

        n = G * Lq
        values["dq"] = scale * (ds @ k)
        bounds["dq"] = abs(scale) * ((off_ds + Lk * f * ds.abs()) @ k.abs())
        values["dk"] = scale * shared(ds.transpose(-1, -2) @ q)
        bounds["dk"] = abs(scale) * shared((off_ds + n * f * ds.abs()).transpose(-1, -2) @ q.abs())
        values["dv"] = shared(p.transpose(-1, -2) @ do)
        bounds["dv"] = shared((off_p + n * f * p).transpose(-1, -2) @ do.abs())
        for x in ("dq", "dk", "dv"):
            bounds[x] = bounds[x] + u * values[x].abs()
    # (values below the type's normal range are rounded to a fixed step)
    least = 2.0 ** -24 if dtype == torch.float16 else 1e-37
    return values, {x: b * 1.001 + least for x, b in bounds.items()}


def check(got, want, bound, what=""):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    worst = (off / bound).max() if off.numel() else torch.zeros(())
    assert torch.isfinite(got.float()).all(), f"{what}: not finite"
    assert float(worst) <= 1.0, f"{what}: off by {float(worst):.3g} of its bound"


def tensors(B, Hq, Hkv, D, Lq, Lk, dtype, device, seed=0, grad=False):
    g = torch.Generator(device=device).manual_seed(seed)
    shapes = [(B, Lq, Hq, D), (B, Lk, Hkv, D), (B, Lk, Hkv, D)] + [(B, Lq, Hq, D)] * grad
    return [torch.randn(x, generator=g, device=device).to(dtype).transpose(1, 2) for x in shapes]


def pages_of(k, v, page, seed=0, spare=3, fill=0.0):
    """(k_pages, v_pages, table) that hold k and v [B, H, L, D] in a random order of pages."""
    B, H, L, D = k.shape
    per = -(-L // page)
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(B * per + spare, generator=g)[:B * per].reshape(B, per).to(k.device)
    out = []
    for x in (k, v):
        pages = torch.full((B * per + spare, H, page, D), fill, dtype=k.dtype, device=k.device)
        padded = torch.full((B, H, per * page, D), fill, dtype=k.dtype, device=k.device)
        padded[:, :, :L] = x
        pages[table.flatten()] = padded.reshape(B, H, per, page, D).transpose(1, 2).flatten(0, 1)
        out.append(pages)
    return out[0], out[1], table.to(torch.int32)
