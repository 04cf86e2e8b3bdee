"""Infinite values: a row that sees one has it in that column, whatever its probability, a row
that does not see it has what it has with a zero in that place, and every other column too."""
import math

import pytest
import torch

import mlx_amd
from mlx_amd import _lib, ops
from tests.attention_util import pages_of, tensors, visible
from tests.test_gpu_attention import BF16, F16, F32

pytestmark = pytest.mark.gpu


def outputs(q, k, v, lengths, window, scale):
    args = dict(scale=scale, window=window)
    paged = pages_of(k, v, 48, fill=math.nan)
    return (mlx_amd.window_attention(q, k, v, lengths=lengths, **args),
            mlx_amd.paged_attention(q, *paged, lengths, **args))


def check(q, k, v, lengths, window, places, scale=0.1):
    """places: ((key, column, value), ...) of sequence 0."""
    B, Hq, Lq, D = q.shape
    Lk = k.shape[2]
    spoilt, clean = v.clone(), v.clone()
    for key, column, value in places:
        spoilt[0, :, key, column] = value
        clean[0, :, key, column] = 0
    n = torch.tensor(lengths, dtype=torch.int32, device=q.device)
    seen = visible(Lq, Lk, lengths, window, 0, q.device)[0, 0]
    for got, want, form in zip(outputs(q, k, spoilt, n, window, scale),
                               outputs(q, k, clean, n, window, scale), ("contiguous", "paged")):
        want = want.clone()
        assert torch.isfinite(want.float()).all()
        for key, column, value in places:
            want[0, :, seen[:, key], column] += value
        same = (got == want) | (torch.isnan(got) & torch.isnan(want))
        assert same.all(), (form, (~same).nonzero()[:4].tolist(), got[~same][:4].tolist(),
                            want[~same][:4].tolist())


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("Lq", (1, 3))
@pytest.mark.parametrize("Lk, window", ((1, None), (5, None), (64, None), (333, 100), (9000, None)))
@pytest.mark.parametrize("D", (64, 96, 128, 256))
def test_few_rows(gpu, D, Lk, window, Lq, dtype):
    """The last key (its place is taken again by keys past it), the first one of the window, one
    inside; both signs in one column; NaN."""
    q, k, v = tensors(2, 8, 2, D, Lq, Lk, dtype, gpu, seed=D + Lk)
    first, last = Lk - window if window else 0, Lk - 1
    places = [(last, 1, math.inf), (first, 2, -math.inf), (last, D - 1, -math.inf),
              (max(first, last - 40), 33, -math.inf), (last, 40, math.nan)]
    if first < last:
        places.append((first, D - 1, math.inf))
    check(q, k, v, [Lk, max(1, Lk - 7)], window, places)


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("Lq", (1, 3))
def test_a_row_without_a_sum_stays_so(gpu, Lq, dtype):
    """A score that is NaN makes NaN of the whole row, whatever values it sees."""
    q, k, v = tensors(1, 8, 2, 64, Lq, 90, dtype, gpu, seed=3)
    q[0, 1, -1, 5] = math.nan
    v[0, :, 88, 7] = math.inf
    for out in outputs(q, k, v, torch.tensor([90], dtype=torch.int32, device=gpu), None, 0.1):
        assert torch.isnan(out[0, 1, -1]).all()
        assert (out[0, 2:, -1, 7] == math.inf).all()
        assert torch.isfinite(out[0, 2:, -1, :7].float()).all()


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("Lq, Lk, window, D", (
    (200, 500, None, 128), (200, 333, 100, 64), (150, 400, 30, 96), (130, 300, 250, 256)))
def test_many_rows(gpu, Lq, Lk, window, D, dtype):
    """Enough key heads for the kernel of tiles; keys inside tiles that all rows see, at their ends
    and before every window.  The keys before 100 are given scores some 20 to 30 below the others',
    whose probabilities round to zero in float16."""
    heads = next(n for n in (8, 64, 512) if _lib.attention_plan(
        2, n, n, Lq, Lk, D, window or 1 << 30, 0, ops._DTYPE_CODE[dtype])[1].startswith("attention_rows"))
    q, k, v = tensors(2, heads, heads, D, Lq, Lk, dtype, gpu, seed=D + Lk)
    q[..., 0] = 5
    k[..., 0] = 5
    k[:, :, :100, 0] = -45
    first, last = Lk - window if window else 0, Lk - 1
    places = [(last, 1, math.inf), (first, 2, -math.inf), (last, D - 1, -math.inf),
              (first, D - 1, math.inf), (20, 33, -math.inf), (Lk - Lq - 1, 34, math.inf),
              (Lk - Lq // 2, 35, math.inf), (99, 36, -math.inf), (last - 64, 40, math.nan)]
    check(q, k, v, [Lk, Lk - 7], window, places)
