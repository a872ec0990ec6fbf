"""K/V cache held in 4 bits: the paged pools, append, read-back and the decode that reads them.

A pool is a pair ``(codes, scales)``: ``codes`` uint8 ``[pages, Hkv, P, D/2]`` and ``scales``
fp16 ``[pages, Hkv, P, 2, D/32]``.  A row (one token of one kv head) is cut into groups of 32
values, each with a scale and a zero: 5 bits a value, against 16 of a plain pool.  The format
is described with ``spa_int4_append`` in include/spa_b200.h; ``int4_values`` restates it in
torch.  No reference counterpart: the reference keeps K/V in the model's dtype
(experiments/triton_kvcache_transformer_decode.py:51-55).

``paged_decode_attention_int4`` and ``paged_gather_decode_attention_int4`` take the arguments
of ``paged_decode_attention`` and ``paged_gather_decode_attention`` with such pairs in place of
the pools (page summaries for the router come from the keys before they are appended).
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from ._util import as_int32, as_int64, dtype_code, launch

GROUP = 32


class PagedKVCacheInt4:
    """A ``PagedKVCache`` in 4 bits: ``k`` and ``v`` are ``(codes, scales)`` pairs."""

    def __init__(self, num_pages: int, kv_heads: int, page_size: int, head_dim: int, *, batch: int,
                 max_pages_per_seq: int, device="cuda"):
        if head_dim % GROUP or not 0 < head_dim <= 256:
            raise ValueError("head_dim must be a multiple of 32 up to 256")

        def pool():
            rows = (num_pages, kv_heads, page_size)
            return (torch.zeros(*rows, head_dim // 2, dtype=torch.uint8, device=device),
                    torch.zeros(*rows, 2, head_dim // GROUP, dtype=torch.float16, device=device))

        self.k, self.v = pool(), pool()
        self.page_table = torch.full((batch, max_pages_per_seq), -1, dtype=torch.int32, device=device)
        self.context_lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.page_size = page_size


def int4_values(pool: tuple[torch.Tensor, torch.Tensor]) -> torch.Tensor:
    """The fp32 values ``[pages, Hkv, P, D]`` a pool stands for (any device; for inspection)."""
    codes, scales = pool
    by = codes.unflatten(-1, (8, -1, 2))
    n = torch.stack((by & 15, by >> 4), -1).transpose(-4, -3).flatten(-3).double()
    scale, zero = scales.double().unbind(-2)
    return (n * scale[..., None] + zero[..., None]).flatten(-2).float()


def _same_device(device: int, *tensors) -> None:
    for t in tensors:
        if t.get_device() != device:
            raise ValueError("CUDA tensors are required" if not t.is_cuda else "tensors must be on one device")


def _pools(k_pool, v_pool, page_table):
    """Checks two 4-bit pools and returns (layout, the scales' addresses, kv_heads, head_dim, page
    table kept alive, device index)."""
    for pool in (k_pool, v_pool):
        if not isinstance(pool, (tuple, list)) or len(pool) != 2:
            raise ValueError("a 4-bit pool is a pair (codes, scales)")
    (kc, ks), (vc, vs) = k_pool, v_pool
    dev = kc.get_device()
    if dev < 0:
        raise ValueError("CUDA tensors are required")
    _same_device(dev, ks, vc, vs, page_table)
    if kc.dtype != torch.uint8 or vc.dtype != torch.uint8 or ks.dtype != torch.float16 or vs.dtype != torch.float16:
        raise ValueError("a 4-bit pool holds uint8 codes and float16 scales")
    shape = kc.shape
    n, h, p, half = shape if len(shape) == 4 else (0, 0, 0, 0)
    if half == 0 or half % 16 or half > 128 or vc.shape != shape:
        raise ValueError("codes must be [pages, Hkv, P, D/2] with D a multiple of 32 up to 256")
    if ks.shape != (n, h, p, 2, half // 16) or vs.shape != ks.shape:
        raise ValueError("scales must be [pages, Hkv, P, 2, D/32]")
    if not (kc.is_contiguous() and ks.is_contiguous() and vc.is_contiguous() and vs.is_contiguous()):
        raise ValueError("contiguous CUDA tensors are required")
    kp, vp, ksp, vsp = kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr()
    if (kp | vp | ksp | vsp) % 16:
        raise ValueError("4-bit pools must be 16-byte aligned")
    table = as_int32(page_table).contiguous()
    if table.dim() != 2 or table.size(1) == 0:
        raise ValueError("page_table must be [batch, pages]")
    layout = _lib.KvLayout(kp, vp, n * h * p, 0, h * p, p, table.data_ptr(), table.size(1), p)
    return layout, ksp, vsp, h, 2 * half, table, dev


def _lengths(t, batch: int, dev: int, name: str) -> torch.Tensor:
    out = as_int32(t).contiguous()
    if out.dim() != 1 or out.size(0) != batch or out.get_device() != dev:
        raise ValueError(f"{name} must be [batch] on the pools' device")
    return out


def kv_append_int4(k_pool, v_pool, page_table: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                   positions: torch.Tensor, *, new_lens: torch.Tensor | None = None) -> None:
    """Quantises ``k_new``/``v_new`` ``[B, Hkv, D]`` (one token) or ``[B, Hkv, T, D]`` into the
    tokens from ``positions[b]`` on; with ``new_lens`` only the first ``new_lens[b]`` of the T.
    The new tensors may be views with any strides over B, Hkv and T (both the same).  Tokens
    before 0 are skipped; no two sequences may write one row."""
    layout, k_scales, v_scales, kv_heads, dim, table, dev = _pools(k_pool, v_pool, page_table)
    batch = table.size(0)
    _same_device(dev, k_new, v_new, positions)
    shape, strides = k_new.shape, k_new.stride()
    tokens = 1
    if len(shape) == 4:
        tokens = shape[2]
    if (len(shape) not in (3, 4) or v_new.shape != shape or shape[1] != kv_heads or shape[-1] != dim):
        raise ValueError("k_new/v_new must be [B, Hkv, D] or [B, Hkv, T, D]")
    if shape[0] != batch or v_new.dtype != k_new.dtype:
        raise ValueError("k_new/v_new must match the page table's batch and each other's dtype")
    code = dtype_code(k_new)
    if strides[-1] != 1 or strides != v_new.stride():
        k_new, v_new = k_new.contiguous(), v_new.contiguous()
        strides = k_new.stride()
    pos = _lengths(positions, batch, dev, "positions")
    lens = _lengths(new_lens, batch, dev, "new_lens") if new_lens is not None else None
    rc = launch(_lib.lib.spa_int4_append, dev, ctypes.byref(layout), k_scales, v_scales, code, batch, kv_heads, dim,
                tokens, k_new.data_ptr(), v_new.data_ptr(), strides[0], strides[1],
                strides[2] if len(shape) == 4 else 0, pos.data_ptr(), lens.data_ptr() if lens is not None else None)
    _lib.check(rc, "spa_int4_append")


def kv_read_int4(k_pool, v_pool, page_table: torch.Tensor, positions: torch.Tensor, tokens: int, *,
                 lens: torch.Tensor | None = None,
                 dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """The values of tokens ``positions[b] + [0, tokens)`` as contiguous K and V
    ``[B, Hkv, tokens, D]`` of ``dtype`` (a cached prefix for ``local_causal_prefill``); zeros
    past ``lens[b]`` and for tokens without a page."""
    layout, k_scales, v_scales, kv_heads, dim, table, dev = _pools(k_pool, v_pool, page_table)
    batch = table.size(0)
    if tokens < 0:
        raise ValueError("tokens must be >= 0")
    pos = _lengths(positions, batch, dev, "positions")
    n = _lengths(lens, batch, dev, "lens") if lens is not None else None
    k = torch.empty((batch, kv_heads, tokens, dim), dtype=dtype, device=table.device)
    v = torch.empty_like(k)
    rc = launch(_lib.lib.spa_int4_read, dev, ctypes.byref(layout), k_scales, v_scales, dtype_code(k), batch, kv_heads,
                dim, tokens, pos.data_ptr(), n.data_ptr() if n is not None else None, k.data_ptr(), v.data_ptr())
    _lib.check(rc, "spa_int4_read")
    return k, v


def check_weights(weights, batch: int, kv_heads: int, dev: int) -> None:
    """``weights`` must be fp32 ``[B, Hkv, T]``, written in place."""
    if (not isinstance(weights, torch.Tensor) or weights.dtype != torch.float32 or weights.dim() != 3
            or weights.shape[:2] != (batch, kv_heads) or weights.size(2) == 0 or not weights.is_contiguous()
            or weights.get_device() != dev):
        raise ValueError("weights must be a contiguous float32 tensor [batch, kv_heads, tokens] on the query's device")


@functools.lru_cache(maxsize=256)
def cache_decode_workspace(device: int, *shape) -> int:
    """``spa_cache_decode_workspace_size`` on CUDA device ``device``: a function of the shape and
    of the device's number of SMs."""
    with torch.cuda.device(device):
        return _lib.lib.spa_cache_decode_workspace_size(*shape)


def _decode(query, k_pool, v_pool, page_table, context_lens, local_window, selected, weights, block_size=None):
    layout, k_scales, v_scales, kv_heads, dim, table, dev = _pools(k_pool, v_pool, page_table)
    page = layout.page_size
    _same_device(dev, query)
    if not query.is_contiguous():
        raise ValueError("contiguous CUDA tensors are required")
    if query.dim() != 3 or query.size(2) != dim or query.size(1) % kv_heads or query.size(1) == 0:
        raise ValueError("incompatible Q/K/V shapes")
    batch, q_heads, _ = query.shape
    if block_size not in (None, page):
        raise ValueError("unsupported head dimension or page layout")
    if local_window < 0:
        raise ValueError("local_window must be >= 0")
    if context_lens is None:
        raise ValueError("context_lens is required with page_table")
    code = dtype_code(query)
    lens = as_int32(context_lens).contiguous()
    if table.size(0) != batch or lens.dim() != 1 or lens.size(0) != batch or lens.get_device() != dev:
        raise ValueError("page_table must be [batch, pages] and context_lens [batch]")
    w_ptr, w_tokens = None, 0
    if weights is not None:
        check_weights(weights, batch, kv_heads, dev)
        w_ptr, w_tokens = weights.data_ptr(), weights.size(2)
    tokens = table.size(1) * page
    top_m, s_ptr = 0, None
    most = min(tokens, local_window) if local_window else tokens
    if selected is not None:
        top_m, s_ptr = selected.size(1), selected.data_ptr()
        most = min(tokens, local_window) + top_m * page
    out = torch.empty_like(query)
    if batch == 0:
        return out
    need = cache_decode_workspace(dev, batch, q_heads, kv_heads, dim, most, tokens, w_ptr is not None, -1)
    # from the caching allocator, per call: ordered with the stream, and a captured graph keeps its own
    ws = torch.empty(need, dtype=torch.uint8, device=table.device) if need else None
    rc = launch(_lib.lib.spa_int4_decode, dev, query.data_ptr(), code, batch, q_heads, kv_heads, dim,
                ctypes.byref(layout), k_scales, v_scales, lens.data_ptr(), tokens, local_window, s_ptr, top_m, most,
                dim ** -0.5, out.data_ptr(), w_ptr, w_tokens, ws.data_ptr() if need else None, need)
    _lib.check(rc, "spa_int4_decode")
    return out


def paged_decode_attention_int4(query: torch.Tensor, k_pool, v_pool, *, page_table: torch.Tensor,
                                context_lens: torch.Tensor, local_window: int = 0,
                                weights: torch.Tensor | None = None) -> torch.Tensor:
    """``paged_decode_attention`` over 4-bit pools: query ``[B, Hq, D]`` of any supported dtype,
    the first ``context_lens[b]`` tokens of each sequence (the last ``local_window`` of them
    when it is positive); an empty context gives zeros.  ``weights`` (fp32 ``[B, Hkv, T]``, in
    place): each token's probability, summed over its kv head's query heads, is added to it;
    T covers the contexts (for ``select_tokens``)."""
    return _decode(query, k_pool, v_pool, page_table, context_lens, local_window, None, weights)


def paged_gather_decode_attention_int4(query: torch.Tensor, k_pool, v_pool, selected_blocks: torch.Tensor, *,
                                       local_window: int, block_size: int, page_table: torch.Tensor,
                                       context_lens: torch.Tensor) -> torch.Tensor:
    """``paged_gather_decode_attention`` over 4-bit pools: the last ``local_window`` tokens, then
    the pages ``selected_blocks[b, :]`` (negative: an empty slot) under one softmax."""
    if (selected_blocks.dim() != 2 or selected_blocks.size(0) != query.size(0) or selected_blocks.size(1) == 0
            or not selected_blocks.is_contiguous()):
        raise ValueError("selected_blocks must be contiguous [batch, top_blocks]")
    if not selected_blocks.is_cuda:
        raise ValueError("contiguous CUDA tensors are required")
    _same_device(query.get_device(), selected_blocks)
    return _decode(query, k_pool, v_pool, page_table, context_lens, local_window, as_int64(selected_blocks), None,
                   block_size)
