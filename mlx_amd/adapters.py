"""Low-rank adapters of many requests beside a projection that they share."""
from __future__ import annotations

import functools
from typing import Optional, Union

import torch

from . import _lib, ops
from ._copy import astype as _astype, contiguous as _contiguous
from .attention import _int32, _tangents
from .ops import _DTYPE_CODE, _FLOATING, _finite_scale, _require_gpu, _require_one_device, _rows_of, _stream_ptr

__all__ = ["adapter_matmul"]

_MOST_ADAPTERS = 1024
_MOST_RANK = 256


def _sizes(x, a, b, indices):
    adapters, rank, K = a.shape
    rows = x.numel() // K
    return (rows, 1 if indices is None else indices.numel(), adapters, rank, K, b.shape[1])


def _pointer(t):
    return None if t is None else t.data_ptr()


def _forward(x, a, b, y, indices, scales, scale, wants_h):
    """(out, h)"""
    lib = _lib.load()
    with torch.cuda.device(x.device):
        sizes = _sizes(x, a, b, indices)
        code = _DTYPE_CODE[x.dtype]
        a, b = _contiguous(a), _contiguous(b)
        x_rows, x_stride = _rows_of(x)
        y_rows, y_stride = (None, 0) if y is None else _rows_of(y)
        out = torch.empty((*x.shape[:-1], sizes[-1]), dtype=x.dtype, device=x.device)
        h = None
        if wants_h:
            h = torch.empty(lib.mlxrocm_adapter_matmul_h_size(*sizes, code), dtype=torch.uint8,
                            device=x.device)
        size = lib.mlxrocm_adapter_matmul_workspace_size(*sizes, code)
        workspace = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
        _lib.check(lib.mlxrocm_adapter_matmul(
            x_rows.data_ptr(), a.data_ptr(), b.data_ptr(), _pointer(indices), _pointer(scales),
            _pointer(y_rows), out.data_ptr(), _pointer(h), *sizes, x_stride, y_stride, scale, code,
            _pointer(workspace), size, _stream_ptr(x)))
    return out, h


class _AdapterVjp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a, b, y, indices, scales, scale):
        out, h = _forward(x, a, b, y, indices, scales, scale, True)
        ctx.save_for_backward(x, a, b, h, indices, scales)
        ctx.scale = scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        x, a, b, h, indices, scales = ctx.saved_tensors
        lib = _lib.load()
        with torch.cuda.device(x.device):
            sizes = _sizes(x, a, b, indices)
            code = _DTYPE_CODE[x.dtype]
            dout = _astype(dout, x.dtype)
            a, b = _contiguous(a), _contiguous(b)
            new = torch.empty if sizes[0] else torch.zeros
            dx, da, db = (new(t.shape, dtype=t.dtype, device=t.device) if wanted else None
                          for t, wanted in zip((x, a, b), ctx.needs_input_grad))
            if sizes[0] and any(ctx.needs_input_grad[:3]):
                x_rows, x_stride = _rows_of(x)
                dout_rows, dout_stride = _rows_of(dout)
                size = lib.mlxrocm_adapter_matmul_vjp_workspace_size(*sizes, code)
                workspace = torch.empty(max(size, 16), dtype=torch.uint8, device=x.device)
                _lib.check(lib.mlxrocm_adapter_matmul_vjp(
                    x_rows.data_ptr(), a.data_ptr(), b.data_ptr(), _pointer(indices),
                    _pointer(scales), h.data_ptr(), dout_rows.data_ptr(), _pointer(dx),
                    _pointer(da), _pointer(db), *sizes, x_stride, dout_stride, ctx.scale, code,
                    workspace.data_ptr(), size, _stream_ptr(x)))
        return dx, da, db, dout if ctx.needs_input_grad[3] else None, None, None, None


def adapter_matmul(
    x: torch.Tensor,
    a: torch.Tensor,
    b: torch.Tensor,
    indices: Optional[torch.Tensor] = None,
    *,
    scale: Union[float, torch.Tensor] = 1.0,
    y: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``y + scale * (x @ a[i].T) @ b[i].T`` with the adapter ``i`` of each request: what low-rank
    adapters add to the product ``y`` (``quantized_matmul(x, ...)``, say; zeros without it) that all
    requests share.  ``x`` ``[..., K]``, ``a`` ``[adapters, rank, K]``, ``b`` ``[adapters, N, rank]``, ``y``
    ``[..., N]``.  ``indices``: integers whose shape is the first dimensions of ``x``'s: one of each
    request ``[B]`` for ``x`` ``[B, L, K]``, or one of each token ``[B, L]``.  A request whose index is no
    adapter's (-1, say) has none: ``y`` as it is.  Without ``indices`` there is one adapter for all, and
    ``a`` and ``b`` may be matrices.  ``scale``: a number, or one of each adapter ``[adapters]``.

    Sums are formed in 32 bits, ``x @ a.T`` is kept in them (float16: in 23 bits of a token's largest), and
    the result is rounded once.  A request's values do not reach another's, whatever they are; where
    adapters or gradients are not finite a request's own may be NaN where infinity is meant.  Up to 1024
    adapters of rank up to 256; adapters of a lower rank than others are filled up with zeros.
    Differentiable with respect to x, a, b and y (once, in reverse mode)."""
    out = ops._fast.adapter_matmul(x, a, b, indices, scale, y)
    if out is not None:
        return out
    tag = "adapter_matmul"
    if a.dim() == 2 and b.dim() == 2 and indices is None:
        a, b = a.unsqueeze(0), b.unsqueeze(0)
    if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
        raise ValueError(f"[{tag}] a and b must have shapes (adapters, rank, K) and (adapters, N, rank) but "
                         f"have {tuple(a.shape)} and {tuple(b.shape)}.")
    adapters, rank, K = a.shape
    N = b.shape[1]
    if not 1 <= adapters <= _MOST_ADAPTERS or not 1 <= rank <= _MOST_RANK or K == 0 or N == 0:
        raise ValueError(f"[{tag}] 1 to {_MOST_ADAPTERS} adapters of rank 1 to {_MOST_RANK} are possible but "
                         f"a and b have shapes {tuple(a.shape)} and {tuple(b.shape)}.")
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"[{tag}] x must have {K} elements in the last dimension but has shape "
                         f"{tuple(x.shape)}.")
    if y is not None and tuple(y.shape) != (*x.shape[:-1], N):
        raise ValueError(f"[{tag}] y must have shape {(*x.shape[:-1], N)} but has {tuple(y.shape)}.")
    if indices is None:
        if adapters != 1:
            raise ValueError(f"[{tag}] indices are needed for {adapters} adapters.")
    else:
        if indices.dtype not in ops._INTEGER:
            raise ValueError(f"[{tag}] indices must hold integers but has type {indices.dtype}.")
        if tuple(indices.shape) != tuple(x.shape[:-1])[:indices.dim()]:
            raise ValueError(f"[{tag}] indices must have the first dimensions of x, {tuple(x.shape[:-1])}, "
                             f"but have shape {tuple(indices.shape)}.")
    operands = [x, a, b] if y is None else [x, a, b, y]
    dtype = functools.reduce(torch.promote_types, (t.dtype for t in operands))
    if dtype not in _FLOATING:
        raise ValueError(f"[{tag}] Received unsupported type {dtype}.")
    scales = None
    if isinstance(scale, torch.Tensor) and scale.dim() > 0:
        if scale.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError(f"[{tag}] no gradients with respect to scale.")
        scales, scale = scale, 1.0
        if tuple(scales.shape) != (adapters,) or scales.dtype not in _FLOATING:
            raise ValueError(f"[{tag}] scale must be a number or {adapters} floating-point numbers but has "
                             f"shape {tuple(scales.shape)} and type {scales.dtype}.")
    scale = _finite_scale(tag, scale)
    if _tangents(*operands) or (scales is not None and _tangents(scales)):
        raise NotImplementedError(f"[{tag}] no forward-mode gradients.")
    others = [t for t in (indices, scales) if t is not None]
    _require_gpu(tag, *operands, *others)
    _require_one_device(tag, *operands, *others)
    with torch.cuda.device(x.device):
        if indices is not None:
            if indices.dtype in (torch.int64, torch.uint64):  # (2 ** 32 is not 0)
                indices = indices.view(torch.int64).clamp(-1, adapters)
            indices = _int32(indices)
        if scales is not None:
            scales = _contiguous(_astype(scales.detach(), torch.float32))
    if torch.is_grad_enabled() and any(t.requires_grad for t in operands):
        # (torch's own conversion: autograd converts the gradients back)
        operands = [t.to(dtype) for t in operands] + [None] * (4 - len(operands))
        return _AdapterVjp.apply(*operands, indices, scales, scale)
    with torch.cuda.device(x.device):
        operands = [_astype(t, dtype) for t in operands] + [None] * (4 - len(operands))
    return _forward(*operands, indices, scales, scale, False)[0]
