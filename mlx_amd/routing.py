"""The router in front of ``SwitchGLU`` and ``gather_qmm``: which experts a token goes to, and with
which weights their results count."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib, ops
from ._copy import astype as _astype, contiguous as _contiguous
from .attention import _tangents
from .ops import _DTYPE_CODE, _FLOATING, _finite_scale, _require_gpu, _require_one_device, _rows_of, _stream_ptr

__all__ = ["route_experts"]

_MOST_EXPERTS = 1024
_MOST_CHOSEN = 32
_MOST_GROUPS = 16


def _route(logits, bias, k, sigmoid, groups, top_groups, group_best, normalize, scale):
    shape = (*logits.shape[:-1], k)
    with torch.cuda.device(logits.device):
        rows, stride = _rows_of(logits)
        if bias is not None:
            bias = _contiguous(_astype(bias, torch.float32))
        indices = torch.empty(shape, dtype=torch.int32, device=logits.device)
        weights = torch.empty(shape, dtype=logits.dtype, device=logits.device)
        _lib.check(_lib.load().mlxrocm_route_experts(
            rows.data_ptr(), None if bias is None else bias.data_ptr(), indices.data_ptr(),
            weights.data_ptr(), indices.numel() // k, stride, logits.shape[-1], k, sigmoid, groups,
            top_groups, group_best, normalize, scale, _DTYPE_CODE[logits.dtype], _stream_ptr(logits)))
    return indices, weights


class _RouteVjp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, *args):
        indices, weights = _route(logits, bias, *args)
        ctx.mark_non_differentiable(indices)
        ctx.save_for_backward(logits, indices)
        ctx.args = args
        return indices, weights

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, _, grad):
        logits, indices = ctx.saved_tensors
        k, sigmoid, *_, normalize, scale = ctx.args
        with torch.cuda.device(logits.device):
            rows, stride = _rows_of(logits)
            grad, grad_stride = _rows_of(_astype(grad, logits.dtype))
            out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
            _lib.check(_lib.load().mlxrocm_route_experts_vjp(
                rows.data_ptr(), indices.data_ptr(), grad.data_ptr(), out.data_ptr(),
                indices.numel() // k, stride, grad_stride, logits.shape[-1], k, sigmoid, normalize,
                scale, _DTYPE_CODE[logits.dtype], _stream_ptr(logits)))
        return (out,) + (None,) * (1 + len(ctx.args))


def route_experts(
    logits: torch.Tensor,
    k: int,
    *,
    scoring: str = "softmax",
    bias: Optional[torch.Tensor] = None,
    groups: int = 1,
    top_groups: Optional[int] = None,
    group_best: int = 1,
    normalize: bool = True,
    scale: float = 1.0,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """The ``k`` experts of each token of ``logits`` ``[..., experts]``: ``(indices, weights)``, both
    ``[..., k]``, int32 and of the logits' type, the first choice first.

    Scores are the ``"softmax"`` of a token's logits or the ``"sigmoid"`` of each.  Experts are chosen by
    score plus ``bias`` ``[experts]`` (for balance; the weights do not have it), the lowest index
    first of equal ones.  With ``groups`` the experts come in that many runs of one size, and
    only the ``top_groups`` of them with the largest sum of their ``group_best`` (1 or 2) best choices
    count.  Weights are the chosen scores, divided by their sum with ``normalize``, times ``scale``.

    An expert whose logit is -inf has no weight and is chosen only where no other is left; so is
    one whose choice is NaN.  A token without any score has weights of zero.  A NaN makes NaN of the
    weights that depend on it.  Up to 1024 experts, 16 groups and 32 choices.
    Differentiable with respect to the logits (once, in reverse mode), not to the bias."""
    out = ops._fast.route_experts(logits, k, scoring, bias, groups, top_groups, group_best, normalize,
                                  scale)
    if out is not None:
        return out
    tag = "route_experts"
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= _MOST_EXPERTS:
        raise ValueError(f"[{tag}] logits must have 1 to {_MOST_EXPERTS} experts in the last dimension "
                         f"but have shape {tuple(logits.shape)}.")
    if logits.dtype not in _FLOATING:
        raise ValueError(f"[{tag}] Received unsupported type {logits.dtype}.")
    if scoring not in ("softmax", "sigmoid"):
        raise ValueError(f"[{tag}] scoring must be 'softmax' or 'sigmoid' but is {scoring!r}.")
    experts = logits.shape[-1]
    groups = int(groups)
    top_groups = groups if top_groups is None else int(top_groups)
    if not 1 <= groups <= _MOST_GROUPS or experts % groups != 0 or not 1 <= top_groups <= groups:
        raise ValueError(f"[{tag}] {top_groups} of {groups} groups of {experts} experts.")
    if group_best not in (1, 2) or group_best > experts // groups:
        raise ValueError(f"[{tag}] group_best must be 1 or 2 and at most the {experts // groups} experts of "
                         f"a group but is {group_best}.")
    k = int(k)
    if not 1 <= k <= min(_MOST_CHOSEN, top_groups * (experts // groups)):
        raise ValueError(f"[{tag}] k must be positive and at most "
                         f"{min(_MOST_CHOSEN, top_groups * (experts // groups))} but is {k}.")
    if bias is not None and (bias.dtype not in _FLOATING or tuple(bias.shape) != (experts,)):
        raise ValueError(f"[{tag}] bias must hold {experts} floating-point numbers but has shape "
                         f"{tuple(bias.shape)} and type {bias.dtype}.")
    scale = _finite_scale(tag, scale)
    if _tangents(logits):
        raise NotImplementedError(f"[{tag}] no forward-mode gradients.")
    operands = [logits] if bias is None else [logits, bias]
    _require_gpu(tag, *operands)
    _require_one_device(tag, *operands)
    if bias is not None:
        bias = bias.detach()
    args = (k, int(scoring == "sigmoid"), groups, top_groups, int(group_best), int(bool(normalize)),
            scale)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _RouteVjp.apply(logits, bias, *args)
    return _route(logits, bias, *args)
