"""CPU restatement (numpy, 64 bits) of the 4-bit cache, of decode attention with accumulated
token weights, and of eviction by them.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py).  The quantiser's roundings belong to the
format, so its steps are fp32 here as well; everything after it is fp64.
"""

from __future__ import annotations

import numpy as np
import torch

__all__ = ["int4_quantise", "int4_dequantise", "attention_weights", "select_tokens", "compact_rows"]


def int4_quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of rows ``[..., D]``."""
    a = x.detach().float().cpu().numpy()
    g = a.shape[-1] // 32
    a = a.reshape(-1, g, 32)
    codes = np.zeros((a.shape[0], g * 8), np.uint16)
    scales = np.zeros((a.shape[0], 2, g), np.float16)
    with np.errstate(all="ignore"):
        lo, hi = a.min(-1), a.max(-1)
        s = np.minimum((hi - lo) * np.float32(1 / 15), np.float32(65504)).astype(np.float16)
        z = np.clip(lo, np.float32(-65504), np.float32(65504)).astype(np.float16)
        n = np.rint((a - z.astype(np.float32)[..., None]) / s.astype(np.float32)[..., None])
    n = np.where((s > 0)[..., None], np.clip(n, 0, 15), 0)
    bad = ~np.isfinite(a).all(-1)
    n = np.where(bad[..., None], 0, n).astype(np.uint16)
    s[bad] = z[bad] = np.nan
    for d in range(32):
        for j in range(g):
            codes[:, (d // 4) * g + j] |= n[:, j, d] << np.uint16(4 * (d % 4))
    scales[:, 0], scales[:, 1] = s, z
    lead = x.shape[:-1]
    return (torch.from_numpy(codes.view(np.uint8).copy()).view(*lead, g * 16),
            torch.from_numpy(scales).view(*lead, 2, g))


def int4_dequantise(pool: tuple[torch.Tensor, torch.Tensor]) -> torch.Tensor:
    """The fp64 values ``[..., D]`` of (codes, scales)."""
    codes, scales = (t.detach().cpu() for t in pool)
    g = scales.size(-1)
    d = torch.arange(32 * g)
    by = 2 * ((d % 32 // 4) * g + d // 32) + d % 4 // 2
    n = (codes[..., by].long() >> (4 * (d % 2))) & 15
    return scales[..., 0, d // 32].double() * n + scales[..., 1, d // 32].double()


def attention_weights(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                      tokens: list) -> tuple[torch.Tensor, torch.Tensor]:
    """Decode attention of q [B, Hq, D] over the listed tokens of contiguous k, v [B, Hkv, L, D]
    (``tokens[b]``: the candidates of sequence b, repeats counted): the output [B, Hq, D] and
    each token's probability summed over its kv head's query heads [B, Hkv, L], fp64."""
    b, hq, d = q.shape
    hkv = k.size(1)
    out = torch.zeros(b, hq, d, dtype=torch.float64)
    w = torch.zeros(b, hkv, k.size(2), dtype=torch.float64)
    for i in range(b):
        t = torch.as_tensor(tokens[i], dtype=torch.long)
        if not t.numel():
            continue
        qi = q[i].double().cpu().view(hkv, hq // hkv, d)
        ki, vi = k[i, :, t].double(), v[i, :, t].double()
        p = torch.softmax(qi @ ki.transpose(1, 2) / d ** 0.5, -1)
        out[i] = (p @ vi).view(hq, d)
        w[i].index_add_(1, t, p.sum(1))
    return out, w


def select_tokens(weights: torch.Tensor, lens: list, budget: int, recent: int) -> tuple[torch.Tensor, torch.Tensor]:
    b, h, total = weights.shape
    keep = torch.full((b, h, budget), -1, dtype=torch.int32)
    kept = torch.zeros(b, dtype=torch.int32)
    for i in range(b):
        n = min(max(int(lens[i]), 0), total)
        kept[i] = min(n, budget)
        r = min(recent, budget)
        for j in range(h):
            ids = list(range(n))
            if n > budget:
                w = weights[i, j].tolist()
                rank = sorted(range(n - r), key=lambda t: (w[t] != w[t], -w[t] if w[t] == w[t] else 0.0, t))
                ids = sorted(rank[: budget - r]) + list(range(n - r, n))
            keep[i, j, : len(ids)] = torch.tensor(ids, dtype=torch.int32)
    return keep, kept


def compact_rows(pool: torch.Tensor, table: torch.Tensor, keep: torch.Tensor) -> torch.Tensor:
    """A copy of the pool [pages, Hkv, P, ...] with token keep[b, h, j] moved to token j."""
    old, new = pool.cpu(), pool.cpu().clone()
    page = pool.size(2)
    for i in range(keep.size(0)):
        for h in range(keep.size(1)):
            for j, t in enumerate(keep[i, h].tolist()):
                if t >= 0:
                    new[table[i, j // page], h, j % page] = old[table[i, t // page], h, t % page]
    return new
