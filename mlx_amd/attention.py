"""Attention, its paged key-value cache and the verification of drafted tokens: what stands
between the quantized projections of a decoder when it is served or tuned.

A sequence's token at position ``p`` sees the tokens ``j <= p`` with ``p - j < window`` or
``j < keep``: the newest ``window`` ones, itself included, and the first ``keep`` beside them
(mlx-lm's rotating cache counts the tokens that it keeps in its size; here ``window + keep`` are
visible); without a window, plain causal attention.  ``q`` holds the newest
tokens of each sequence (``mx.fast.scaled_dot_product_attention(..., mask="causal")`` aligns
them so too); where a sequence has fewer tokens than ``q``, those in front are padding and
give zeros.  Heads are laid out as there: ``[B, heads, L, D]``, with any strides (a transposed
``[B, L, heads, D]`` is read and answered in place), and several query heads may share a key head.

Scores, sums and results are formed in 32 bits.  With 16-bit types probabilities are rounded to the
type where they multiply values, and in the gradients so are theirs: results are up to 1.4 times as far
off as their own rounding.  Where rows are few (decoding, drafted tokens) probabilities keep
twice the bits there, and the results' own rounding is all.

As in ``ops``, tensors are torch tensors on the GPU, and every computation is done by the
HIP kernels behind the C ABI.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _lib, ops
from ._copy import astype as _astype, contiguous as _contiguous, copy as _copy
from .ops import _DTYPE_CODE, _FLOATING, _require_gpu, _stream_ptr

__all__ = ["window_attention", "paged_attention", "paged_cache_update", "verify_draft"]

_MOST = 1 << 30  # a window that is never full


def _aligned(t: torch.Tensor) -> bool:
    """Rows along the last dimension dense, and each of them aligned to 16 bytes."""
    unit = 16 // t.element_size()
    return ((t.stride(-1) == 1 or t.shape[-1] == 1) and t.data_ptr() % 16 == 0
            and all(n == 1 or s % unit == 0 for n, s in zip(t.shape[:-1], t.stride()[:-1])))


def _operand(t: torch.Tensor) -> torch.Tensor:
    return t if t.numel() == 0 or _aligned(t) else _copy(t)


def _strides(*tensors: torch.Tensor):
    """Of the first three dimensions of each; 0 where there is one element (any will do)."""
    return [0 if n == 1 else s for t in tensors for n, s in zip(t.shape[:3], t.stride()[:3])]


def _array(values):
    return (ctypes.c_int64 * len(values))(*values)


def _empty_like(t: torch.Tensor) -> torch.Tensor:
    """A new tensor in t's memory order (dense)."""
    out = torch.empty_like(t)
    return out if out.numel() == 0 or _aligned(out) else torch.empty(
        t.shape, dtype=t.dtype, device=t.device)


def _tangents(*tensors: torch.Tensor) -> bool:
    """Whether forward-mode gradients are wanted of any of them."""
    return any(torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _check_visible(tag: str, scale, window, keep) -> Tuple[float, int, int]:
    scale = float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"[{tag}] scale must be finite but got {scale}.")
    if window is not None and window < 1:
        raise ValueError(f"[{tag}] window must be positive but got {window}.")
    if keep < 0:
        raise ValueError(f"[{tag}] keep must not be negative but got {keep}.")
    return scale, _MOST if window is None else min(int(window), _MOST), min(int(keep), _MOST)


def _check_heads(tag: str, q, k, v, what: str) -> None:
    for name, t in (("q", q), (f"k{what}", k), (f"v{what}", v)):
        if t.dim() != 4:
            raise ValueError(f"[{tag}] {name} must have 4 dimensions but has shape {tuple(t.shape)}.")
    if k.shape != v.shape:
        raise ValueError(f"[{tag}] k{what} and v{what} must have the same shape but got "
                         f"{tuple(k.shape)} and {tuple(v.shape)}.")
    if q.shape[-1] != k.shape[-1]:
        raise ValueError(f"[{tag}] The last dimensions of q and k{what} must match but the shapes "
                         f"are {tuple(q.shape)} and {tuple(k.shape)}.")
    if k.shape[1] == 0 or q.shape[1] % k.shape[1] != 0:
        raise ValueError(f"[{tag}] {q.shape[1]} query heads cannot share {k.shape[1]} key heads.")
    if q.shape[-1] % 8 != 0 or not 0 < q.shape[-1] <= 256:
        raise ValueError(f"[{tag}] The head dimension must be a multiple of 8 up to 256 but is "
                         f"{q.shape[-1]}.")


def _check_ints(tag: str, name: str, t: torch.Tensor, shape) -> None:
    if t.dtype not in (torch.int32, torch.int64, torch.uint32):
        raise ValueError(f"[{tag}] {name} must hold integers but has type {t.dtype}.")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"[{tag}] {name} must have shape {tuple(shape)} but has {tuple(t.shape)}.")


def _int32(t: torch.Tensor) -> torch.Tensor:
    return _contiguous(_astype(t, torch.int32))


# ---------------------------------------------------------------- window_attention
def _window_forward(q, k, v, lengths, scale, window, keep, wants_lse):
    lib = _lib.load()
    q, k, v = _operand(q), _operand(k), _operand(v)
    out = _empty_like(q)
    B, Hq, Lq, D = q.shape
    Hkv, Lk = k.shape[1:3]
    code = _DTYPE_CODE[q.dtype]
    lse = None
    if wants_lse:
        size = lib.mlxrocm_window_attention_lse_size(B, Hq, Hkv, Lq, Lk, D, window, keep, code)
        lse = torch.empty(max(size, 16), dtype=torch.uint8, device=q.device)
    size = lib.mlxrocm_window_attention_workspace_size(B, Hq, Hkv, Lq, Lk, D, window, keep, code)
    workspace = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    _lib.check(lib.mlxrocm_window_attention(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
        None if lse is None else lse.data_ptr(), None if lengths is None else lengths.data_ptr(),
        B, Hq, Hkv, Lq, Lk, D, _array(_strides(q, k, v, out)), scale, window, keep, code,
        None if workspace is None else workspace.data_ptr(), size, _stream_ptr(q)))
    return q, k, v, out, lse


class _WindowAttentionVjp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, scale, window, keep):
        q, k, v, out, lse = _window_forward(q, k, v, lengths, scale, window, keep, True)
        ctx.save_for_backward(q, k, v, out, lse, lengths)
        ctx.args = (scale, window, keep)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, lengths = ctx.saved_tensors
        lib = _lib.load()
        dout = _operand(_astype(dout, q.dtype))
        dq, dk, dv = _empty_like(q), _empty_like(k), _empty_like(v)
        B, Hq, Lq, D = q.shape
        Hkv, Lk = k.shape[1:3]
        code = _DTYPE_CODE[q.dtype]
        size = lib.mlxrocm_window_attention_vjp_workspace_size(
            B, Hq, Hkv, Lq, Lk, D, *ctx.args[1:], code)
        workspace = torch.empty(max(size, 16), dtype=torch.uint8, device=q.device)
        _lib.check(lib.mlxrocm_window_attention_vjp(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
            dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
            None if lengths is None else lengths.data_ptr(), B, Hq, Hkv, Lq, Lk, D,
            _array(_strides(q, k, v, out, dout, dq, dk, dv)), *ctx.args, code,
            workspace.data_ptr(), size, _stream_ptr(q)))
        return dq, dk, dv, None, None, None, None


def window_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    scale: float,
    window: Optional[int] = None,
    keep: int = 0,
    lengths: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``softmax(scale q k^T) v`` over the tokens that each one of ``q`` sees (see the module).
    ``q`` ``[B, Hq, Lq, D]``, ``k`` and ``v`` ``[B, Hkv, Lk, D]``; ``lengths`` ``[B]``: how many of
    the ``Lk`` keys each sequence has, all without it.  The result has ``q``'s shape and, where
    that is dense, its memory order.  Differentiable with respect to q, k and v (once,
    in reverse mode)."""
    out = ops._fast.window_attention(q, k, v, scale, window, keep, lengths)
    if out is None and torch.is_grad_enabled():
        out = ops._fast.window_attention_recorded(q, k, v, scale, window, keep, lengths)
    if out is not None:
        return out
    tag = "window_attention"
    scale, window, keep = _check_visible(tag, scale, window, keep)
    _check_heads(tag, q, k, v, "")
    if k.shape[0] != q.shape[0]:
        raise ValueError(f"[{tag}] q and k must have the same batch size but the shapes are "
                         f"{tuple(q.shape)} and {tuple(k.shape)}.")
    dtype = torch.promote_types(torch.promote_types(q.dtype, k.dtype), v.dtype)
    if dtype not in _FLOATING:
        raise ValueError(f"[{tag}] Received unsupported type {dtype}.")
    if _tangents(q, k, v):
        raise NotImplementedError(f"[{tag}] no forward-mode gradients.")
    if lengths is not None:
        _check_ints(tag, "lengths", lengths, (q.shape[0],))
        _require_gpu(tag, lengths)
        lengths = _int32(lengths)
    _require_gpu(tag, q, k, v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        # (torch's own conversion: autograd converts the gradients back)
        q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
        return _WindowAttentionVjp.apply(q, k, v, lengths, scale, window, keep)
    q, k, v = _astype(q, dtype), _astype(k, dtype), _astype(v, dtype)
    return _window_forward(q, k, v, lengths, scale, window, keep, False)[3]


# ---------------------------------------------------------------- the paged cache
def _check_pages(tag: str, k_pages, v_pages) -> None:
    if k_pages.shape[2] == 0 or k_pages.shape[2] % 16 != 0:
        raise ValueError(f"[{tag}] The page size must be a multiple of 16 but the pages have shape "
                         f"{tuple(k_pages.shape)}.")
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        if t.numel() and not _aligned(t):
            raise ValueError(f"[{tag}] {name} must have dense rows that are aligned to 16 bytes.")


def _check_table(tag: str, block_table, lengths, batch: int) -> None:
    if block_table.dim() != 2 or block_table.shape[0] != batch:
        raise ValueError(f"[{tag}] block_table must have shape ({batch}, pages of a sequence) but "
                         f"has {tuple(block_table.shape)}.")
    _check_ints(tag, "block_table", block_table, block_table.shape)
    _check_ints(tag, "lengths", lengths, (batch,))


def _table(block_table: torch.Tensor) -> torch.Tensor:
    """As int32 with dense rows (a slice of a wider table stays where it is)."""
    table = _astype(block_table, torch.int32)
    return table if table.stride(1) == 1 or table.shape[1] <= 1 else _contiguous(table)


def paged_cache_update(
    k: torch.Tensor,
    v: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Writes new keys and values ``[B, Hkv, L, D]`` into the pages of a cache, in place, and
    returns the pages.  ``k_pages`` and ``v_pages`` are ``[pages, Hkv, page size, D]``, the page
    size a multiple of 16; token ``j`` of sequence ``b`` has row ``j % page size`` of page
    ``block_table[b, j // page size]``.  ``lengths`` ``[B]`` counts the tokens of each sequence with
    the new ones; where it is below ``L``, those in front are padding and not written.  No gradients."""
    if ops._fast.paged_cache_update(k, v, k_pages, v_pages, block_table, lengths):
        return k_pages, v_pages
    tag = "paged_cache_update"
    for name, t in (("k", k), ("v", v), ("k_pages", k_pages), ("v_pages", v_pages)):
        if t.dim() != 4:
            raise ValueError(f"[{tag}] {name} must have 4 dimensions but has shape {tuple(t.shape)}.")
    if k.shape != v.shape or k_pages.shape != v_pages.shape:
        raise ValueError(f"[{tag}] Keys and values must have the same shape but got "
                         f"{tuple(k.shape)} and {tuple(v.shape)}, pages {tuple(k_pages.shape)} and "
                         f"{tuple(v_pages.shape)}.")
    if k.shape[1] != k_pages.shape[1] or k.shape[3] != k_pages.shape[3]:
        raise ValueError(f"[{tag}] Keys of shape {tuple(k.shape)} do not fit pages of shape "
                         f"{tuple(k_pages.shape)}.")
    if len({k.dtype, v.dtype, k_pages.dtype, v_pages.dtype}) != 1 or k.dtype not in _FLOATING:
        raise ValueError(f"[{tag}] Keys, values and pages must have one real floating type but have "
                         f"{k.dtype}, {v.dtype}, {k_pages.dtype} and {v_pages.dtype}.")
    if k.shape[3] * k.element_size() % 16 != 0:
        raise ValueError(f"[{tag}] Rows of {k.shape[3]} elements of {k.dtype} are not a multiple of "
                         "16 bytes.")
    _check_table(tag, block_table, lengths, k.shape[0])
    _check_pages(tag, k_pages, v_pages)
    if any(n > 1 and s == 0 for t in (k_pages, v_pages) for n, s in zip(t.shape, t.stride())):
        raise ValueError(f"[{tag}] Pages that share memory (expanded ones) cannot be written to.")
    if _tangents(k, v, k_pages, v_pages) or (torch.is_grad_enabled() and any(
            t.requires_grad for t in (k, v, k_pages, v_pages))):
        raise NotImplementedError(f"[{tag}] no gradients through a paged cache.")
    _require_gpu(tag, k, v, k_pages, v_pages, block_table, lengths)
    lib = _lib.load()
    table, lengths = _table(block_table), _int32(lengths)
    k, v = _operand(k), _operand(v)
    B, H, L, D = k.shape
    _lib.check(lib.mlxrocm_paged_cache_update(
        k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(),
        lengths.data_ptr(), B, H, L, D, k_pages.shape[0], k_pages.shape[2], table.shape[1],
        _array(_strides(k, v, k_pages, v_pages) + [table.stride(0)]), _DTYPE_CODE[k.dtype],
        _stream_ptr(k)))
    for pages in (k_pages, v_pages):  # written to: a graph that saved them is to know
        if not pages.is_inference():
            torch.autograd.graph.increment_version(pages)
    return k_pages, v_pages


def paged_attention(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    scale: float,
    window: Optional[int] = None,
    keep: int = 0,
) -> torch.Tensor:
    """:func:`window_attention` of the newest tokens ``q`` ``[B, Hq, Lq, D]`` of each sequence over
    a cache of pages that holds them already (:func:`paged_cache_update` has the layout).  ``Lq`` is
    1 for decoding, a few for drafted tokens, any number for a chunk of a prompt.  The work is laid
    out for the keys that ``block_table`` has room for: a table much wider than the
    sequences is better passed as its first columns.  No gradients."""
    out = ops._fast.paged_attention(
        q, k_pages, v_pages, block_table, lengths, scale, window, keep)
    if out is not None:
        return out
    tag = "paged_attention"
    scale, window, keep = _check_visible(tag, scale, window, keep)
    _check_heads(tag, q, k_pages, v_pages, "_pages")
    if not q.dtype == k_pages.dtype == v_pages.dtype or q.dtype not in _FLOATING:
        raise ValueError(f"[{tag}] Queries and pages must have one real floating type but have "
                         f"{q.dtype}, {k_pages.dtype} and {v_pages.dtype}.")
    _check_table(tag, block_table, lengths, q.shape[0])
    _check_pages(tag, k_pages, v_pages)
    if _tangents(q, k_pages, v_pages) or (torch.is_grad_enabled() and any(
            t.requires_grad for t in (q, k_pages, v_pages))):
        raise NotImplementedError(f"[{tag}] no gradients through a paged cache.")
    _require_gpu(tag, q, k_pages, v_pages, block_table, lengths)
    lib = _lib.load()
    table, lengths = _table(block_table), _int32(lengths)
    q = _operand(q)
    out = _empty_like(q)
    B, Hq, Lq, D = q.shape
    pages, Hkv, page = k_pages.shape[:3]
    code = _DTYPE_CODE[q.dtype]
    size = lib.mlxrocm_paged_attention_workspace_size(
        B, Hq, Hkv, Lq, D, table.shape[1] * page, window, keep, code)
    workspace = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    _lib.check(lib.mlxrocm_paged_attention(
        q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(), lengths.data_ptr(),
        out.data_ptr(), B, Hq, Hkv, Lq, D, pages, page, table.shape[1],
        _array(_strides(q, k_pages, v_pages, out) + [table.stride(0)]), scale, window, keep, code,
        None if workspace is None else workspace.data_ptr(), size, _stream_ptr(q)))
    return out


# ---------------------------------------------------------------- drafted tokens
def verify_draft(
    draft: torch.Tensor,
    target_probs: torch.Tensor,
    draft_probs: Optional[torch.Tensor],
    accept_uniform: torch.Tensor,
    sample_uniform: torch.Tensor,
    *,
    lengths: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Which drafted tokens to keep, and the token after them, such that the result is distributed
    as samples of the target model.  ``draft`` ``[B, K]``; ``target_probs`` ``[B, K + 1, V]``: the
    target's probabilities at each draft and after the last; ``draft_probs`` ``[B, K, V]``: those
    the drafts were drawn with, ``None`` for drafts that were not drawn (looked up, or greedy);
    ``accept_uniform`` ``[B, K]`` and ``sample_uniform`` ``[B]``: random numbers in ``[0, 1)``;
    ``lengths`` ``[B]``: how many drafts each sequence has, ``K`` without it.

    Draft ``i`` is kept while ``accept_uniform[i] * draft_probs[i, x] < target_probs[i, x]``; at the
    first that is not, the token is drawn from ``max(target - draft, 0)`` there, after the last
    from the target.  Returns ``(tokens [B, K + 1], accepted [B])`` as int32: the kept drafts, the
    token drawn (-1 if no token has any probability), then -1.  Weights are summed as whole
    multiples of 2**-40, so the same inputs give the same tokens whatever the order of sums."""
    out = ops._fast.verify_draft(
        draft, target_probs, draft_probs, accept_uniform, sample_uniform, lengths)
    if out is not None:
        return out
    tag = "verify_draft"
    if draft.dim() != 2:
        raise ValueError(f"[{tag}] draft must have 2 dimensions but has shape {tuple(draft.shape)}.")
    B, K = draft.shape
    if target_probs.dim() != 3 or tuple(target_probs.shape[:2]) != (B, K + 1):
        raise ValueError(f"[{tag}] target_probs must have shape ({B}, {K + 1}, vocabulary) but has "
                         f"{tuple(target_probs.shape)}.")
    V = target_probs.shape[2]
    if draft_probs is not None and tuple(draft_probs.shape) != (B, K, V):
        raise ValueError(f"[{tag}] draft_probs must have shape ({B}, {K}, {V}) but has "
                         f"{tuple(draft_probs.shape)}.")
    if V == 0:
        raise ValueError(f"[{tag}] The vocabulary is empty.")
    dtype = target_probs.dtype
    if dtype not in _FLOATING or (draft_probs is not None and draft_probs.dtype != dtype):
        raise ValueError(f"[{tag}] Probabilities must have one real floating type but have {dtype}"
                         + ("." if draft_probs is None else f" and {draft_probs.dtype}."))
    for name, t, shape in (("accept_uniform", accept_uniform, (B, K)),
                           ("sample_uniform", sample_uniform, (B,))):
        if t.dtype != torch.float32 or tuple(t.shape) != shape:
            raise ValueError(f"[{tag}] {name} must be float32 of shape {shape} but is {t.dtype} of "
                             f"shape {tuple(t.shape)}.")
    _check_ints(tag, "draft", draft, (B, K))
    if lengths is not None:
        _check_ints(tag, "lengths", lengths, (B,))
    _require_gpu(tag, *(t for t in (draft, target_probs, draft_probs, accept_uniform,
                                    sample_uniform, lengths) if t is not None))
    lib = _lib.load()
    target = target_probs if target_probs.stride(2) == 1 or V == 1 else _contiguous(target_probs)
    probs = draft_probs
    if probs is not None and probs.stride(2) != 1 and V != 1:
        probs = _contiguous(probs)
    accept, sample = _contiguous(accept_uniform), _contiguous(sample_uniform)
    draft, lengths = _int32(draft), None if lengths is None else _int32(lengths)
    tokens = torch.empty((B, K + 1), dtype=torch.int32, device=target.device)
    accepted = torch.empty((B,), dtype=torch.int32, device=target.device)
    size = lib.mlxrocm_verify_draft_workspace_size(B, V)
    workspace = torch.empty(max(size, 16), dtype=torch.uint8, device=target.device)
    strides = [*target.stride()[:2], *((0, 0) if probs is None else probs.stride()[:2])]
    _lib.check(lib.mlxrocm_verify_draft(
        draft.data_ptr(), target.data_ptr(), None if probs is None else probs.data_ptr(),
        accept.data_ptr(), sample.data_ptr(), None if lengths is None else lengths.data_ptr(),
        tokens.data_ptr(), accepted.data_ptr(), B, K, V, _array(strides), _DTYPE_CODE[dtype],
        workspace.data_ptr(), size, _stream_ptr(target)))
    return tokens, accepted
