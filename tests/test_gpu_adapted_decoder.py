"""The decoder's operators together: a layer of quantized projections with adapters of several
requests, rotary positions, a paged cache, and experts behind a router, against plain torch in 64 bits,
with all tokens at once and step by step; and the gradients of what is trained."""
import math

import pytest
import torch

import mlx_amd
from mlx_amd import nn

pytestmark = pytest.mark.gpu

DIMS, HEADS, KV, DIM, HIDDEN, EXPERTS, CHOSEN = 128, 4, 2, 32, 192, 8, 2
ADAPTERS, RANK = 3, 8
ROTATION = dict(dims=24, base=5000.0)
# A value goes through some ten sums of up to 256 terms in 32 bits, each off by 256 2**-24 of what it
# sums at most; values are compared to the largest there are
BOUND = 10 * 256 * 2.0 ** -24


class Block(torch.nn.Module):
    def __init__(self):
        super().__init__()
        kw = dict(bias=False, device="cuda", dtype=torch.float32)

        def adapted(inputs, outputs):
            layer = nn.LoRALinear(nn.QuantizedLinear(inputs, outputs, **kw), RANK, ADAPTERS, 2.0)
            with torch.no_grad():
                layer.lora_b.normal_(std=0.1)
            return layer

        self.q_proj, self.k_proj = adapted(DIMS, HEADS * DIM), adapted(DIMS, KV * DIM)
        self.v_proj, self.o_proj = adapted(DIMS, KV * DIM), adapted(HEADS * DIM, DIMS)
        self.gate = torch.nn.Parameter(torch.randn(EXPERTS, DIMS, device="cuda") * 0.3)
        self.register_buffer("balance", torch.randn(EXPERTS, device="cuda") * 0.05)
        self.experts = nn.SwitchGLU(DIMS, HIDDEN, EXPERTS, device="cuda", dtype=torch.float32)

    def forward(self, x, adapters, positions=None, cache=None, lengths=None):
        def heads(y, n):
            return y.view(*y.shape[:2], n, DIM).transpose(1, 2)

        q, k, v = (heads(layer(x, adapters), n) for layer, n in (
            (self.q_proj, HEADS), (self.k_proj, KV), (self.v_proj, KV)))
        if cache is None:
            y = mlx_amd.window_attention(mlx_amd.rope(q, positions, **ROTATION),
                                         mlx_amd.rope(k, positions, **ROTATION), v, scale=DIM ** -0.5)
        else:
            k_pages, v_pages, table = cache
            q, *_ = mlx_amd.rope_cache_update(q, k, v, k_pages, v_pages, table, lengths, **ROTATION)
            y = mlx_amd.paged_attention(q, k_pages, v_pages, table, lengths, scale=DIM ** -0.5)
        x = x + self.o_proj(y.transpose(1, 2).flatten(2), adapters)
        indices, weights = mlx_amd.route_experts(
            torch.nn.functional.linear(x, self.gate), CHOSEN, scoring="sigmoid", bias=self.balance,
            groups=4, top_groups=2, group_best=2, scale=1.5)
        with torch.no_grad():
            y = self.experts(x, indices)
        return x + (y * weights[..., None]).sum(-2)


def plain(block, x, adapters, leaves):
    """The same in 64 bits; ``leaves``: the trained parameters by name."""
    def weights(layer):
        return mlx_amd.dequantize(layer.weight, layer.scales, layer.biases, layer.group_size,
                                  layer.bits).double()

    def adapted(name, x):
        y = x @ weights(getattr(block, name).linear).T
        a, b = leaves[name + ".lora_a"], leaves[name + ".lora_b"]
        rows = []
        for i, row in zip(adapters.tolist(), x):
            rows.append(2.0 * (row @ a[i].T) @ b[i].T if 0 <= i < ADAPTERS else
                        torch.zeros(row.shape[0], b.shape[1], dtype=torch.float64, device=x.device))
        return y + torch.stack(rows)

    B, L, _ = x.shape
    half = ROTATION["dims"] // 2
    angle = torch.arange(L, device=x.device).double()[:, None] * ROTATION["base"] ** (
        -torch.arange(half, device=x.device).double() / half)

    def rotate(t):
        a, b = t[..., :half], t[..., half:2 * half]
        cos, sin = angle.cos(), angle.sin()
        return torch.cat((a * cos - b * sin, b * cos + a * sin, t[..., 2 * half:]), -1)

    q, k, v = (adapted(name, x).view(B, L, n, DIM).transpose(1, 2) for name, n in (
        ("q_proj", HEADS), ("k_proj", KV), ("v_proj", KV)))
    q, k = rotate(q), rotate(k)
    k, v = (t.repeat_interleave(HEADS // KV, 1) for t in (k, v))
    s = (q @ k.transpose(2, 3)) * DIM ** -0.5
    s = s.masked_fill(torch.ones(L, L, device=x.device).triu(1).bool(), -math.inf)
    x = x + adapted("o_proj", (torch.softmax(s, -1) @ v).transpose(1, 2).flatten(2))
    scores = torch.sigmoid(x @ leaves["gate"].T)
    choice = (scores + block.balance.double()).detach()
    marks = choice.view(B, L, 4, 2).sum(-1)
    open_ = torch.zeros_like(marks).scatter_(-1, marks.topk(2)[1], 1).repeat_interleave(2, -1) > 0
    indices = choice.masked_fill(~open_, -math.inf).topk(CHOSEN)[1]
    w = scores.gather(-1, indices)
    w = 1.5 * w / w.sum(-1, keepdim=True)
    with torch.no_grad():
        up, gate, down = (weights(p) for p in (block.experts.up_proj, block.experts.gate_proj,
                                               block.experts.down_proj))
        hidden = torch.nn.functional.silu(torch.einsum("bld,blkhd->blkh", x, gate[indices]))
        hidden = hidden * torch.einsum("bld,blkhd->blkh", x, up[indices])
        y = torch.einsum("blkh,blkdh->blkd", hidden, down[indices])
    return x + (y * w[..., None]).sum(-2)


@pytest.fixture(scope="module")
def block():
    torch.manual_seed(4)
    return Block()


def test_all_at_once_and_step_by_step(gpu, block):
    B, L = 4, 45
    x = torch.randn(B, L, DIMS, device="cuda")
    adapters = torch.tensor([2, -1, 0, 2], dtype=torch.int32, device="cuda")
    leaves = {n: p.detach().double() for n, p in block.named_parameters()}
    want = plain(block, x.double(), adapters, leaves)
    most = float(want.abs().max())
    positions = torch.arange(L, device="cuda").expand(B, L)
    with torch.no_grad():
        out = block(x, adapters, positions)
        assert float((out - want).abs().max()) <= BOUND * most
        pages = [torch.zeros(B * 3, KV, 16, DIM, device="cuda") for _ in range(2)]
        table = torch.randperm(B * 3, device="cuda").view(B, 3).to(torch.int32)
        got, at = [], 0
        for n in (20, 1, 1, 5, 18):
            at += n
            lengths = torch.full((B,), at, dtype=torch.int32, device="cuda")
            got.append(block(x[:, at - n:at], adapters, cache=(*pages, table), lengths=lengths))
    assert float((torch.cat(got, 1) - want).abs().max()) <= BOUND * most


def test_a_captured_step(gpu, block):
    """One token of each request, over and over, beside the eager program."""
    B = 3
    adapters = torch.tensor([1, 1, -1], dtype=torch.int32, device="cuda")
    pages = [[torch.zeros(B * 2, KV, 16, DIM, device="cuda") for _ in range(2)] for _ in range(2)]
    table = torch.arange(B * 2, device="cuda").view(B, 2).to(torch.int32)
    lengths = torch.tensor([1, 7, 3], dtype=torch.int32, device="cuda")
    held, count = torch.randn(B, 1, DIMS, device="cuda"), lengths.clone()
    with torch.no_grad():
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            block(held, adapters, cache=(*pages[0], table), lengths=count)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block(held, adapters, cache=(*pages[0], table), lengths=count)
            count.add_(1)
        for p in pages[0]:
            p.zero_()
        for _ in range(6):
            x = torch.randn(B, 1, DIMS, device="cuda")
            held.copy_(x)
            graph.replay()
            want = block(x, adapters, cache=(*pages[1], table), lengths=lengths)
            lengths = lengths + 1
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_gradients(gpu, block):
    B, L = 3, 33
    x = torch.randn(B, L, DIMS, device="cuda")
    adapters = torch.tensor([0, 2, -1], dtype=torch.int32, device="cuda")
    names = [n for n, p in block.named_parameters() if p.requires_grad]
    assert len(names) == 9
    leaves = {n: p.detach().double().requires_grad_() for n, p in block.named_parameters()}
    up = torch.randn(B, L, DIMS, device="cuda")
    want = torch.autograd.grad((plain(block, x.double(), adapters, leaves) * up.double()).sum(),
                               [leaves[n] for n in names])
    positions = torch.arange(L, device="cuda").expand(B, L)
    got = torch.autograd.grad((block(x, adapters, positions) * up).sum(),
                              [block.get_parameter(n) for n in names])
    for name, g, w in zip(names, got, want):
        # twice as many sums, back and forth
        assert float((g - w).abs().max()) <= 2 * BOUND * float(w.abs().max()), name
