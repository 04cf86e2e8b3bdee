"""Rotary positions: ``rope`` (``mx.fast.rope`` with positions of each token in place of an offset, along
one or several axes), and ``rope_cache_update``, which rotates queries and keys on their way to
``paged_attention``.

Pair ``i`` of the first ``dims`` columns of a head turns by ``scale * position / freqs[i]``, where
``freqs[i]`` is ``base ** (2 * i / dims)`` unless ``freqs`` is given.  The pair is the columns ``i``
and ``i + dims / 2``, with ``traditional`` ``2 * i`` and ``2 * i + 1``; further columns stay as
they are.  With ``sections`` positions have several axes (time, height and width of an image, say): the
first ``sections[0]`` pairs turn by the position along the first, and so on.

Angles are formed in 64 bits, so that far positions lose nothing, rotations in 32, rounded once.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence, Tuple

import torch

from . import _lib, ops
from ._copy import astype as _astype, contiguous as _contiguous, copy as _copy
from .attention import (
    _array, _check_pages, _check_table, _empty_like, _int32, _strides, _table, _tangents)
from .ops import _DTYPE_CODE, _FLOATING, _number, _require_gpu, _require_one_device, _stream_ptr

__all__ = ["rope", "rope_cache_update"]

_MOST_AXES = 4
_MOST_DIMS = 256


def _dense_columns(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 or t.numel() == 0 else _copy(t)


class _Rotation:
    """The options of a call, checked, as the library takes them."""

    def __init__(self, tag, D, batch, length, positions, dims, traditional, base, scale, freqs,
                 sections):
        if D % 2 != 0:
            raise ValueError(f"[{tag}] The head dimension must be even but is {D}.")
        dims = D if dims is None else int(dims)
        if dims <= 0 or dims % 2 != 0 or dims > min(D, _MOST_DIMS):
            raise ValueError(f"[{tag}] dims must be even and at most {min(D, _MOST_DIMS)} but is {dims}.")
        if base is not None and freqs is not None:
            raise ValueError(f"[{tag}] Only one of base or freqs can have a value.")
        base = 10000.0 if base is None else _number(tag, "base", base)
        scale = _number(tag, "scale", scale)
        if not (math.isfinite(base) and base > 0 and math.isfinite(scale)):
            raise ValueError(f"[{tag}] base must be positive and scale finite but got {base}, {scale}.")
        shape = (batch, length)
        if sections is not None:
            sections = tuple(int(n) for n in sections)
            if not 1 <= len(sections) <= _MOST_AXES or min(sections) < 0 or sum(sections) * 2 != dims:
                raise ValueError(f"[{tag}] sections must be the pairs of 1 to {_MOST_AXES} axes that add "
                                 f"up to {dims // 2} but are {sections}.")
            shape = (len(sections), *shape)
        if positions is not None:
            if positions.dtype not in (torch.int32, torch.int64, torch.uint32):
                raise ValueError(f"[{tag}] positions must hold integers but has type {positions.dtype}.")
            if tuple(positions.shape) != shape:
                raise ValueError(f"[{tag}] positions must have shape {shape} but has "
                                 f"{tuple(positions.shape)}.")
        elif sections is not None:
            raise ValueError(f"[{tag}] sections need positions.")
        if freqs is not None and (freqs.dtype not in _FLOATING or tuple(freqs.shape) != (dims // 2,)):
            raise ValueError(f"[{tag}] freqs must hold {dims // 2} floating-point numbers but has shape "
                             f"{tuple(freqs.shape)} and type {freqs.dtype}.")
        self.positions, self.freqs, self.sections = positions, freqs, sections
        self.options = (dims, int(bool(traditional)), base, scale)

    def tensors(self):
        return [t for t in (self.positions, self.freqs) if t is not None]

    def load(self) -> None:
        """Conversions on the device, where the call needs any."""
        if self.positions is not None and self.positions.dtype == torch.uint32:
            self.positions = _astype(self.positions, torch.int64)
        if self.freqs is not None:
            self.freqs = _contiguous(_astype(self.freqs.detach(), torch.float32))

    def arguments(self):
        p = self.positions
        strides = None
        if p is not None:
            strides = _array(([0] if p.dim() == 2 else []) + list(p.stride()))
        axes = 1 if self.sections is None else len(self.sections)
        return (None if p is None else p.data_ptr(), strides,
                int(p is not None and p.dtype == torch.int64), axes,
                (ctypes.c_int * axes)(*(self.sections or (0,))), *self.options,
                None if self.freqs is None else self.freqs.data_ptr())


def _rope(x: torch.Tensor, rotation: _Rotation, inverse: bool) -> torch.Tensor:
    with torch.cuda.device(x.device):
        x = _dense_columns(x)
        rotation.load()
        out = _empty_like(x)
        B, H, L, D = x.shape
        _lib.check(_lib.load().mlxrocm_rope(
            x.data_ptr(), out.data_ptr(), B, H, L, D, _array(_strides(x, out)),
            *rotation.arguments(), int(inverse), _DTYPE_CODE[x.dtype], _stream_ptr(x)))
    return out


class _RopeVjp(torch.autograd.Function):
    """A rotation is linear, and its transpose turns back: so any number of derivatives."""

    @staticmethod
    def forward(ctx, x, positions, freqs, rotation, inverse):
        ctx.save_for_backward(positions, freqs)
        ctx.args = (rotation, inverse)
        return _rope(x, rotation, inverse)

    @staticmethod
    def backward(ctx, dout):
        positions, freqs = ctx.saved_tensors  # (that they are as they were)
        rotation, inverse = ctx.args
        return _RopeVjp.apply(dout, positions, freqs, rotation, not inverse), None, None, None, None


def rope(
    x: torch.Tensor,
    positions: torch.Tensor,
    *,
    dims: Optional[int] = None,
    traditional: bool = False,
    base: Optional[float] = None,
    scale: float = 1.0,
    freqs: Optional[torch.Tensor] = None,
    sections: Optional[Sequence[int]] = None,
) -> torch.Tensor:
    """``x`` ``[B, heads, L, D]`` rotated by ``positions``: integers ``[B, L]``, with ``sections`` ``[axes,
    B, L]``.  ``dims`` (even, at most 256): the columns that turn, all without it; ``base``: 10000
    without it; ``freqs`` ``[dims / 2]`` in its place.  The result has ``x``'s shape and, where that is
    dense, its memory order.  Differentiable with respect to x (in reverse mode)."""
    out = ops._fast.rope(x, positions, dims, traditional, base, scale, freqs, sections)
    if out is not None:
        return out
    tag = "rope"
    if x.dim() != 4:
        raise ValueError(f"[{tag}] x must have 4 dimensions but has shape {tuple(x.shape)}.")
    if x.dtype not in _FLOATING:
        raise ValueError(f"[{tag}] Received unsupported type {x.dtype}.")
    if positions is None:
        raise ValueError(f"[{tag}] positions are needed.")
    rotation = _Rotation(tag, x.shape[3], x.shape[0], x.shape[2], positions, dims, traditional, base,
                         scale, freqs, sections)
    if _tangents(x) or (freqs is not None and _tangents(freqs)):
        raise NotImplementedError(f"[{tag}] no forward-mode gradients.")
    if freqs is not None and freqs.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"[{tag}] no gradients with respect to freqs.")
    _require_gpu(tag, x, *rotation.tensors())
    _require_one_device(tag, x, *rotation.tensors())
    if torch.is_grad_enabled() and x.requires_grad:
        return _RopeVjp.apply(x, positions, freqs, rotation, False)
    return _rope(x, rotation, False)


def rope_cache_update(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    positions: Optional[torch.Tensor] = None,
    dims: Optional[int] = None,
    traditional: bool = False,
    base: Optional[float] = None,
    scale: float = 1.0,
    freqs: Optional[torch.Tensor] = None,
    sections: Optional[Sequence[int]] = None,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """:func:`rope` of new queries ``[B, Hq, L, D]`` and keys ``[B, Hkv, L, D]`` and
    :func:`paged_cache_update` of those keys and values, in one pass: returns the rotated queries, which
    ``paged_attention`` takes, and the pages, which are written to in place.  Tokens turn by
    their places in their sequences, or by ``positions`` where those are given (the tokens go to the
    same places of the cache all the same).  Where ``lengths`` is below ``L`` the queries in front are
    padding and give zeros.  No gradients."""
    out = ops._fast.rope_cache_update(q, k, v, k_pages, v_pages, block_table, lengths, positions, dims,
                                      traditional, base, scale, freqs, sections)
    if out is not None:
        return out, k_pages, v_pages
    tag = "rope_cache_update"
    for name, t in (("q", q), ("k", k), ("v", v), ("k_pages", k_pages), ("v_pages", v_pages)):
        if t.dim() != 4:
            raise ValueError(f"[{tag}] {name} must have 4 dimensions but has shape {tuple(t.shape)}.")
    if k.shape != v.shape or k_pages.shape != v_pages.shape:
        raise ValueError(f"[{tag}] Keys and values must have the same shape but got "
                         f"{tuple(k.shape)} and {tuple(v.shape)}, pages {tuple(k_pages.shape)} and "
                         f"{tuple(v_pages.shape)}.")
    if q.shape[0] != k.shape[0] or q.shape[2:] != k.shape[2:]:
        raise ValueError(f"[{tag}] Queries of shape {tuple(q.shape)} do not go with keys of shape "
                         f"{tuple(k.shape)}.")
    if k.shape[1] != k_pages.shape[1] or k.shape[3] != k_pages.shape[3]:
        raise ValueError(f"[{tag}] Keys of shape {tuple(k.shape)} do not fit pages of shape "
                         f"{tuple(k_pages.shape)}.")
    if len({t.dtype for t in (q, k, v, k_pages, v_pages)}) != 1 or k.dtype not in _FLOATING:
        raise ValueError(f"[{tag}] Queries, keys, values and pages must have one real floating type but "
                         f"have {q.dtype}, {k.dtype}, {v.dtype}, {k_pages.dtype} and {v_pages.dtype}.")
    _check_table(tag, block_table, lengths, k.shape[0])
    _check_pages(tag, k_pages, v_pages)
    if any(n > 1 and s == 0 for t in (k_pages, v_pages) for n, s in zip(t.shape, t.stride())):
        raise ValueError(f"[{tag}] Pages that share memory (expanded ones) cannot be written to.")
    rotation = _Rotation(tag, q.shape[3], q.shape[0], q.shape[2], positions, dims, traditional, base,
                         scale, freqs, sections)
    operands = [q, k, v, k_pages, v_pages]
    if freqs is not None:
        operands.append(freqs)
    if _tangents(*operands) or (torch.is_grad_enabled() and any(t.requires_grad for t in operands)):
        raise NotImplementedError(f"[{tag}] no gradients through a paged cache.")
    operands = [q, k, v, k_pages, v_pages, block_table, lengths, *rotation.tensors()]
    _require_gpu(tag, *operands)
    _require_one_device(tag, *operands)
    with torch.cuda.device(q.device):
        table, lengths = _table(block_table), _int32(lengths)
        q, k, v = (_dense_columns(t) for t in (q, k, v))
        rotation.load()
        out = _empty_like(q)
        B, Hq, L, D = q.shape
        _lib.check(_lib.load().mlxrocm_rope_cache_update(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), k_pages.data_ptr(),
            v_pages.data_ptr(), table.data_ptr(), lengths.data_ptr(), B, Hq, k.shape[1], L, D,
            k_pages.shape[0], k_pages.shape[2], table.shape[1],
            _array(_strides(q, k, v, out, k_pages, v_pages) + [table.stride(0)]),
            *rotation.arguments(), _DTYPE_CODE[q.dtype], _stream_ptr(q)))
    for pages in (k_pages, v_pages):  # written to: a graph that saved them is to know
        if not pages.is_inference():
            torch.autograd.graph.increment_version(pages)
    return out, k_pages, v_pages
