"""Eviction from a paged cache by accumulated attention weight.

A serving loop passes ``weights`` to ``paged_decode_attention`` (or its 4-bit form) every step;
when a sequence outgrows its budget, ``evict_tokens`` keeps its last ``recent`` tokens and those
that attention has weighted most, per kv head, and moves them to the front of the sequence's
pages in their old order.  ``select_tokens`` and ``compact_tokens`` are its two halves.  Keys
carry their positions (they are rotated or embedded before they are appended), so the moved rows
need no other change; page summaries do: rebuild them afterwards.  No reference counterpart.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._util import as_int32, launch


def select_tokens(weights: torch.Tensor, context_lens: torch.Tensor, *, budget: int,
                  recent: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The tokens that stay: ``(keep [B, Hkv, budget], kept_lens [B])``, int32.

    ``weights`` fp32 ``[B, Hkv, T]``.  A sequence of at most ``budget`` tokens keeps them all;
    a longer one its last ``min(recent, budget)`` and, of the others, those of the largest
    weight (ties to the lower token, NaN below every number).  ``keep`` is ascending, then -1."""
    if not (weights.is_cuda and context_lens.is_cuda):
        raise ValueError("CUDA tensors are required")
    if weights.dim() != 3 or weights.dtype != torch.float32 or weights.numel() == 0 or not weights.is_contiguous():
        raise ValueError("weights must be a contiguous float32 tensor [batch, kv_heads, tokens]")
    if budget <= 0 or recent < 0:
        raise ValueError("budget must be positive and recent >= 0")
    batch, heads, tokens = weights.shape
    dev = weights.get_device()
    lens = as_int32(context_lens).contiguous()
    if lens.dim() != 1 or lens.size(0) != batch or lens.get_device() != dev:
        raise ValueError("context_lens must be [batch] on the weights' device")
    keep = torch.empty((batch, heads, budget), dtype=torch.int32, device=weights.device)
    kept = torch.empty_like(lens)
    rc = launch(_lib.lib.spa_select_tokens, dev, weights.data_ptr(), batch, heads, tokens, lens.data_ptr(), budget,
                recent, keep.data_ptr(), kept.data_ptr())
    _lib.check(rc, "spa_select_tokens")
    return keep, kept


def compact_tokens(pools, page_table: torch.Tensor, keep: torch.Tensor, *,
                   weights: torch.Tensor | None = None) -> None:
    """Moves token ``keep[b, h, j]`` to token j in every pool, in place.

    ``pools``: tensors ``[pages, Hkv, P, ...]`` of one geometry, or 4-bit ``(codes, scales)``
    pairs, e.g. ``(cache.k, cache.v)``.  ``keep`` must be ascending and then -1 (as
    ``select_tokens`` returns it); a list that is not leaves its (sequence, kv head) as it was
    and raises the device error word.  ``weights`` ``[B, Hkv, T]`` move along and become zero
    behind the kept tokens; pool rows behind them stay as they were.  A page may belong to one
    sequence only, and no two pools may share memory (ValueError)."""
    flat = [t for p in pools for t in (p if isinstance(p, (tuple, list)) else (p,))]
    if not flat or len(flat) > 8:
        raise ValueError("pools must hold 1 to 8 tensors")
    dev = keep.get_device()
    shape = flat[0].shape
    ptrs, sizes = (ctypes.c_void_p * len(flat))(), (ctypes.c_int * len(flat))()
    if dev < 0 or page_table.get_device() < 0:
        raise ValueError("CUDA tensors are required")
    for i, t in enumerate(flat):
        if t.get_device() != dev:
            raise ValueError("CUDA tensors are required" if not t.is_cuda else "tensors must be on one device")
        if t.dim() < 4 or t.shape[:3] != shape[:3] or t.numel() == 0:
            raise ValueError("pools must be [pages, Hkv, P, ...] of one geometry")
        if not t.is_contiguous():
            raise ValueError("contiguous CUDA tensors are required")
        # (not stride(2): a contiguous tensor may have any stride there when P is 1)
        ptrs[i], sizes[i] = t.data_ptr(), t.numel() // (shape[0] * shape[1] * shape[2]) * t.element_size()
    if page_table.get_device() != dev:
        raise ValueError("tensors must be on one device")
    if keep.dtype != torch.int32 or keep.dim() != 3 or keep.numel() == 0 or not keep.is_contiguous():
        raise ValueError("keep must be a contiguous int32 tensor [batch, kv_heads, budget]")
    table = as_int32(page_table).contiguous()
    pages, heads, page = shape[:3]
    batch, kept_heads, budget = keep.shape
    if kept_heads != heads or table.dim() != 2 or table.size(0) != batch or table.size(1) == 0:
        raise ValueError("keep must be [batch, kv_heads, budget] and page_table [batch, pages]")
    if weights is not None and (weights.dtype != torch.float32 or weights.dim() != 3
                                or weights.shape[:2] != (batch, heads) or weights.size(2) < budget
                                or not weights.is_contiguous() or weights.get_device() != dev):
        raise ValueError("weights must be a contiguous float32 tensor [batch, kv_heads, tokens >= budget]")
    layout = _lib.KvLayout(None, None, pages * heads * page, 0, heads * page, page, table.data_ptr(), table.size(1),
                           page)
    rc = launch(_lib.lib.spa_compact_tokens, dev, ctypes.byref(layout), len(flat), ptrs, sizes, batch, heads,
                keep.data_ptr(), budget, weights.data_ptr() if weights is not None else None,
                weights.size(2) if weights is not None else 0)
    _lib.check(rc, "spa_compact_tokens")


def evict_tokens(cache, weights: torch.Tensor, *, budget: int, recent: int) -> torch.Tensor:
    """Cuts every sequence of a ``PagedKVCache`` or ``PagedKVCacheInt4`` to ``budget`` tokens:
    ``select_tokens``, ``compact_tokens`` of K, V and ``weights``, and ``context_lens`` in
    place.  ``weights`` must cover the contexts, as decode asks (and reports): tokens past them
    are dropped.  Returns ``keep``.  Nothing synchronises, so the whole can be captured."""
    if budget > weights.size(-1):
        raise ValueError("budget must not exceed the weights' tokens")
    keep, kept = select_tokens(weights, cache.context_lens, budget=budget, recent=recent)
    compact_tokens((cache.k, cache.v), cache.page_table, keep, weights=weights)
    cache.context_lens.copy_(kept)
    return keep
