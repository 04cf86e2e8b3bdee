"""The example's decoder: the paged cache, the attention that reads it, the window and the drafts'
verification together against the same decoder without any of them."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

_spec = importlib.util.spec_from_file_location(
    "speculative_decode", Path(__file__).resolve().parents[1] / "examples" / "speculative_decode.py")
example = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(example)


@pytest.fixture(scope="module")
def model():
    torch.manual_seed(3)
    return example.Decoder(vocab=512, dims=128, layers=3, heads=4, kv_heads=2, dim=32, hidden=256,
                           window=24, keep=3, dtype=torch.float32)


def test_cached_logits_are_those_of_all_tokens_at_once(model):
    tokens = torch.randint(0, 512, (2, 75), device="cuda")
    with torch.no_grad():
        want = model(tokens)
        cache = model.cache(2, 80)
        got, at = [], 0
        for n in (1, 40, 1, 5, 28):
            at += n
            lengths = torch.full((2,), at, dtype=torch.int32, device="cuda")
            got.append(model(tokens[:, at - n:at], lengths, cache))
    # float32 sums of up to 256 terms in another order, three layers: 3 * 256 * 2**-24 of the largest
    assert float((torch.cat(got, 1) - want).abs().max()) <= 3 * 256 * 2.0 ** -24 * float(want.abs().max())


def test_greedy_tokens_do_not_depend_on_drafts(model):
    prompts = torch.randint(0, 512, (3, 50), device="cuda")
    counts = torch.tensor([50, 1, 33], device="cuda")
    plain, kept, of = example.generate(model, prompts, counts, 40, drafts=0, greedy=True)
    assert (kept, of) == (0, 0) and plain.shape == (3, 40)
    out, kept, of = example.generate(model, prompts, counts, 40, drafts=3, draft_layers=2, greedy=True)
    assert 0 < kept <= of
    for row, want in zip(out, plain):
        assert row[row >= 0][:40].tolist() == want.tolist()


def test_sampled_tokens_are_tokens_and_repeat(model):
    prompts = torch.randint(0, 512, (2, 30), device="cuda")
    counts = torch.tensor([30, 12], device="cuda")
    runs = [example.generate(model, prompts, counts, 20, drafts=2, seed=5) for _ in range(2)]
    assert torch.equal(runs[0][0], runs[1][0])
    for row in runs[0][0]:
        assert int((row >= 0).sum()) >= 20 and int(row.max()) < 512


def test_tuning_lowers_the_loss(model):
    tokens = torch.randint(0, 512, (2, 60), device="cuda")
    losses = example.tune(model, tokens, steps=4, rate=0.5)
    assert losses[-1] < losses[0] and all(x == x for x in losses)
