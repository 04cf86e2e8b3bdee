"""A small decoder of quantized projections, served and tuned with the framework's attention.

Serving rotates queries and keys on their way into the pages of a cache (``rope_cache_update``) and
attends to them there (``paged_attention``), under a window with a few first tokens that stay
visible.  The first layers of the decoder draft some tokens, the whole decoder reads them all at
once, and ``verify_draft`` keeps those that it would have sampled: what is generated is distributed as
the whole decoder's own samples.  Tuning attends without a cache (``rope``, ``window_attention``) and differentiates through
both and through the quantized products.

    python examples/speculative_decode.py [--batch 4] [--tokens 128] [--drafts 4] [--greedy]

Weights and prompts are random.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import mlx_amd  # noqa: E402
from mlx_amd import nn  # noqa: E402


class PagedCache:
    """Keys and values of a batch of sequences, a pair of page tensors for each layer.  Which
    tokens count is given by the caller's lengths alone: to drop drafted ones, count them no more."""

    def __init__(self, layers, batch, heads, dim, longest, page=64, dtype=torch.bfloat16,
                 device="cuda"):
        each = -(-longest // page)
        shape = (batch * each, heads, page, dim)
        self.k = [torch.empty(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.v = [torch.empty(shape, dtype=dtype, device=device) for _ in range(layers)]
        # any page can be anyone's: here they are dealt out in turn
        self.table = torch.arange(batch * each, dtype=torch.int32, device=device).view(
            each, batch).t().contiguous()


class RMSNorm(torch.nn.Module):
    def __init__(self, dims, device):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.ones(dims, device=device))

    def forward(self, x):
        y = x.float()
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-5)
        return (y * self.weight).to(x.dtype)


class Layer(torch.nn.Module):
    def __init__(self, dims, heads, kv_heads, dim, hidden, window, keep, device, dtype):
        super().__init__()
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.visible = dict(scale=dim ** -0.5, window=window, keep=keep)
        kw = dict(bias=False, device=device, dtype=dtype)
        self.q_proj = nn.QuantizedLinear(dims, heads * dim, **kw)
        self.k_proj = nn.QuantizedLinear(dims, kv_heads * dim, **kw)
        self.v_proj = nn.QuantizedLinear(dims, kv_heads * dim, **kw)
        self.o_proj = nn.QuantizedLinear(heads * dim, dims, **kw)
        self.mlp = nn.SwiGLU(dims, hidden, device=device, dtype=dtype)
        self.attention_norm = RMSNorm(dims, device)
        self.mlp_norm = RMSNorm(dims, device)

    def attention(self, x, lengths, positions, cache, i):
        def heads(y, n):
            return y.view(*y.shape[:2], n, self.dim).transpose(1, 2)

        q = heads(self.q_proj(x), self.heads)
        k = heads(self.k_proj(x), self.kv_heads)
        v = heads(self.v_proj(x), self.kv_heads)
        if cache is None:
            y = mlx_amd.window_attention(mlx_amd.rope(q, positions), mlx_amd.rope(k, positions), v,
                                         **self.visible)
        else:  # (tokens turn by their places in the cache, which are their positions)
            q, *pages = mlx_amd.rope_cache_update(q, k, v, cache.k[i], cache.v[i], cache.table,
                                                  lengths)
            y = mlx_amd.paged_attention(q, *pages, cache.table, lengths, **self.visible)
        return self.o_proj(y.transpose(1, 2).flatten(2))

    def forward(self, x, lengths, positions, cache, i):
        x = x + self.attention(self.attention_norm(x), lengths, positions, cache, i)
        return x + self.mlp(self.mlp_norm(x))


class Decoder(torch.nn.Module):
    def __init__(self, vocab=32000, dims=1024, layers=8, heads=16, kv_heads=4, dim=64,
                 hidden=2816, window=512, keep=4, device="cuda", dtype=torch.bfloat16):
        super().__init__()
        self.kv_heads, self.dim, self.dtype = kv_heads, dim, dtype
        self.embedding = nn.QuantizedEmbedding(vocab, dims, device=device, dtype=dtype)
        self.layers = torch.nn.ModuleList(
            Layer(dims, heads, kv_heads, dim, hidden, window, keep, device, dtype)
            for _ in range(layers))
        self.norm = RMSNorm(dims, device)

    def cache(self, batch, longest):
        return PagedCache(len(self.layers), batch, self.kv_heads, self.dim, longest,
                          dtype=self.dtype, device=self.norm.weight.device)

    def forward(self, tokens, lengths=None, cache=None, layers=None):
        """Logits after each of ``tokens`` [B, L], the newest of ``lengths`` [B] tokens of each
        sequence if there is a cache, all tokens of it if there is none."""
        L = tokens.shape[1]
        first = 0 if lengths is None else (lengths - L)[:, None]
        positions = first + torch.arange(L, device=tokens.device).expand(tokens.shape)
        x = self.embedding(tokens)
        for i, layer in enumerate(self.layers[:layers]):
            x = layer(x, lengths, positions, cache, i)
        return self.embedding.as_linear(self.norm(x))


def probabilities(logits, greedy):
    if greedy:
        return torch.nn.functional.one_hot(logits.argmax(-1), logits.shape[-1]).float()
    return torch.softmax(logits.float(), -1)


@torch.no_grad()
def generate(model, prompts, counts, tokens, drafts=4, draft_layers=2, greedy=False, seed=0):
    """At least ``tokens`` more tokens for each of ``prompts`` [B, L], which are padded in front to a
    common length and have ``counts`` [B] tokens each.  Returns (rows of [B, ...] int32 tokens, -1
    where there is none, and how many drafts were kept of how many).  The drafting layers fill the
    first layers of the one cache with what the whole decoder would put there."""
    device = prompts.device
    g = torch.Generator(device=device).manual_seed(seed)
    B, L = prompts.shape
    cache = model.cache(B, L + tokens + 2 * (drafts + 1))
    lengths = counts.to(torch.int32) - 1  # in the cache; the newest token is not yet
    if L > 1:
        model(prompts[:, :-1], lengths, cache)
    newest = prompts[:, -1:].to(torch.int32)
    made, kept, steps = [], torch.zeros((), dtype=torch.int64, device=device), 0
    count = torch.zeros(B, dtype=torch.int32, device=device)
    while int(count.min()) < tokens:
        row, chosen = newest, []
        asked = []
        for i in range(drafts):
            p = probabilities(model(row, lengths + i + 1, cache, draft_layers)[:, -1], greedy)
            row = p.argmax(-1, keepdim=True) if greedy else torch.multinomial(p, 1, generator=g)
            row = row.to(torch.int32)
            chosen.append(row)
            asked.append(p)
        draft = torch.cat(chosen, 1) if drafts else newest[:, :0]
        target = probabilities(
            model(torch.cat((newest, draft), 1), lengths + drafts + 1, cache), greedy)
        uniform = torch.rand((B, drafts + 1), generator=g, device=device)
        out, accepted = mlx_amd.verify_draft(
            draft, target, None if greedy or not drafts else torch.stack(asked, 1),
            uniform[:, :drafts], uniform[:, drafts])
        # a sequence that has enough stays where it is, so that the cache holds the others
        going = (count < tokens).to(torch.int32)
        made.append(torch.where(going[:, None] > 0, out, -1))
        newest = torch.where(going[:, None] > 0, out.gather(1, accepted[:, None].long()), newest)
        lengths = lengths + going * (accepted + 1)
        count = count + going * (accepted + 1)
        kept += (going * accepted).sum()
        steps += int(going.sum())
    return torch.cat(made, 1), int(kept), steps * drafts


def tune(model, tokens, steps=3, rate=20.0):
    """Steps of gradient descent on the norms' weights; the losses."""
    losses = []
    weights = [p for p in model.parameters() if p.requires_grad]
    for _ in range(steps):
        logits = model(tokens[:, :-1])
        loss = torch.nn.functional.cross_entropy(
            logits.flatten(0, 1).float(), tokens[:, 1:].flatten().long())
        grads = torch.autograd.grad(loss, weights)
        with torch.no_grad():
            for p, g in zip(weights, grads):
                p -= rate * g
        losses.append(float(loss.detach()))
    return losses


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--batch", type=int, default=4)
    parser.add_argument("--prompt", type=int, default=700)
    parser.add_argument("--tokens", type=int, default=128)
    parser.add_argument("--drafts", type=int, default=4)
    parser.add_argument("--greedy", action="store_true")
    args = parser.parse_args()
    torch.manual_seed(0)
    model = Decoder()
    prompts = torch.randint(0, 32000, (args.batch, args.prompt), device="cuda")
    counts = torch.linspace(max(1, args.prompt // 4), args.prompt, args.batch,
                            device="cuda").to(torch.int32)
    print("losses", " ".join(f"{x:.4f}" for x in tune(model, prompts)))
    for drafts in (0, args.drafts):
        for timed in (False, True):
            torch.cuda.synchronize()
            start = time.perf_counter()
            out, kept, of = generate(model, prompts, counts, args.tokens if timed else 8, drafts,
                                     greedy=args.greedy)
            torch.cuda.synchronize()
            seconds = time.perf_counter() - start
        made = int((out >= 0).sum())
        print(f"{drafts} drafts: {made} tokens in {seconds:.3f} s, kept {kept} of {of} drafts")


if __name__ == "__main__":
    main()
