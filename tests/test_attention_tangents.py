"""Forward-mode gradients are refused, not dropped: no GPU."""
import pytest
import torch
from torch.autograd import forward_ad

import mlx_amd


def z(*shape):
    return torch.zeros(shape)


@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("requires_grad", (False, True))
def test_attention(which, requires_grad):
    ints = torch.zeros((2, 2), dtype=torch.int32)
    with forward_ad.dual_level():
        for call, shapes in (
                (lambda *x: mlx_amd.window_attention(*x, scale=1.0),
                 ((2, 4, 3, 64), (2, 2, 5, 64), (2, 2, 5, 64))),
                (lambda *x: mlx_amd.paged_attention(*x, ints, ints[0], scale=1.0),
                 ((2, 4, 3, 64), (5, 2, 16, 64), (5, 2, 16, 64)))):
            args = [z(*s) for s in shapes]
            with pytest.raises(RuntimeError, match="GPU only"):
                call(*args)
            args[which] = forward_ad.make_dual(
                args[which].requires_grad_(requires_grad), torch.ones_like(args[which]))
            with pytest.raises(NotImplementedError, match="no .*gradients"):
                call(*args)


@pytest.mark.parametrize("which", range(4))
def test_update(which):
    ints = torch.zeros((2, 2), dtype=torch.int32)
    args = [z(2, 2, 1, 64), z(2, 2, 1, 64), z(5, 2, 16, 64), z(5, 2, 16, 64)]
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="no gradients"):
            mlx_amd.paged_cache_update(*args, ints, ints[0])
