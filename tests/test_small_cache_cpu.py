"""What of the 4-bit cache and of eviction can be checked without a GPU: the entry points'
refusals, the C entry points' argument checks, and the restatement that the GPU tests use."""

import ctypes

import pytest
import torch

import attention_b200 as spa
import oracle.small_cache as ref
from attention_b200 import _lib


def test_cpu_tensors_are_refused():
    cache = spa.PagedKVCacheInt4(2, 2, 4, 64, batch=1, max_pages_per_seq=2, device="cpu")
    q = torch.zeros(1, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        spa.paged_decode_attention_int4(q, cache.k, cache.v, page_table=cache.page_table,
                                        context_lens=cache.context_lens)
    with pytest.raises(ValueError, match="CUDA"):
        spa.paged_gather_decode_attention_int4(q, cache.k, cache.v, torch.zeros(1, 1, dtype=torch.int64),
                                               local_window=0, block_size=4, page_table=cache.page_table,
                                               context_lens=cache.context_lens)
    with pytest.raises(ValueError, match="CUDA"):
        spa.kv_append_int4(cache.k, cache.v, cache.page_table, q, q, cache.context_lens)
    with pytest.raises(ValueError, match="CUDA"):
        spa.kv_read_int4(cache.k, cache.v, cache.page_table, cache.context_lens, 3)
    with pytest.raises(ValueError, match="CUDA"):
        spa.select_tokens(torch.zeros(1, 2, 8), cache.context_lens, budget=2, recent=1)
    with pytest.raises(ValueError, match="CUDA"):
        spa.compact_tokens((cache.k, cache.v), cache.page_table, torch.zeros(1, 2, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="budget"):
        spa.evict_tokens(cache, torch.zeros(1, 2, 8), budget=9, recent=1)
    for dim in (0, 16, 100, 288):
        with pytest.raises(ValueError, match="head_dim"):
            spa.PagedKVCacheInt4(2, 2, 4, dim, batch=1, max_pages_per_seq=2, device="cpu")


def test_c_entry_points_check_arguments_before_the_device():
    lib, bad = _lib.lib, _lib.SPA_ERR_INVALID
    lay = _lib.KvLayout(16, 16, 64, 0, 16, 8, 16, 4, 8)  # never dereferenced: each call below is refused
    kv = ctypes.byref(lay)
    assert lib.spa_int4_append(None, 16, 16, 2, 1, 1, 64, 1, 16, 16, 1, 1, 1, 16, None, None) == bad
    assert lib.spa_int4_append(kv, 16, 16, 2, 1, 1, 48, 1, 16, 16, 1, 1, 1, 16, None, None) == bad  # head_dim
    assert lib.spa_int4_append(kv, 16, 16, 7, 1, 1, 64, 1, 16, 16, 1, 1, 1, 16, None, None) == bad  # dtype
    assert lib.spa_int4_append(kv, 16, 24, 2, 1, 1, 64, 1, 16, 16, 1, 1, 1, 16, None, None) == bad  # alignment
    assert lib.spa_int4_append(kv, 16, 16, 2, 1, 1, 64, -1, 16, 16, 1, 1, 1, 16, None, None) == bad
    assert lib.spa_int4_append(kv, 16, 16, 2, 1, 1, 64, 0, 16, 16, 1, 1, 1, 16, None, None) == _lib.SPA_OK
    assert lib.spa_int4_read(kv, 16, 16, 2, 1, 1, 64, 1, 16, None, None, 16, None) == bad
    assert lib.spa_int4_read(kv, 16, 16, 2, 1, 1, 64, 0, 16, None, None, None, None) == _lib.SPA_OK

    def decode(**kw):
        a = dict(q=16, dtype=2, b=1, hq=4, hkv=2, d=64, kv=kv, ks=16, vs=16, lens=16, cap=32, win=0, sel=None, m=0,
                 cand=32, out=16, w=None, wt=0, ws=None, wsb=0) | kw
        return lib.spa_int4_decode(a["q"], a["dtype"], a["b"], a["hq"], a["hkv"], a["d"], a["kv"], a["ks"], a["vs"],
                                   a["lens"], a["cap"], a["win"], a["sel"], a["m"], a["cand"], 0.125, a["out"], a["w"],
                                   a["wt"], a["ws"], a["wsb"], None)

    for kw in (dict(q=None), dict(out=None), dict(lens=None), dict(dtype=3), dict(b=0), dict(hq=3), dict(d=72),
               dict(d=288), dict(cap=0), dict(win=-1), dict(cand=-1), dict(sel=16), dict(w=16), dict(ks=None),
               dict(w=16, wt=8, sel=16, m=1), dict(kv=None)):
        assert decode(**kw) == bad, kw
    assert decode(hq=600, hkv=2) == _lib.SPA_ERR_UNSUPPORTED
    assert decode(w=16, wt=32) == _lib.SPA_ERR_WORKSPACE
    assert lib.spa_cache_decode_workspace_size(1, 4, 2, 64, 32, 32, 1, -1) > 0
    assert lib.spa_cache_decode_workspace_size(1, 3, 2, 64, 32, 32, 1, -1) == 0
    assert lib.spa_paged_decode_weights(16, 2, 1, 4, 2, 64, kv, 16, 32, 0, 32, 0.125, 16, None, 0, None, 0, None) == bad
    assert lib.spa_select_tokens(16, 1, 1, 8, 16, 0, 0, 16, 16, None) == bad
    assert lib.spa_select_tokens(16, 1, 1, 8, 16, 4, -1, 16, 16, None) == bad
    assert lib.spa_select_tokens(None, 1, 1, 8, 16, 4, 0, 16, 16, None) == bad
    ptr, size = (ctypes.c_void_p * 1)(16), (ctypes.c_int * 1)(0)
    assert lib.spa_compact_tokens(kv, 1, ptr, size, 1, 1, 16, 4, None, 0, None) == bad  # an empty row
    assert lib.spa_compact_tokens(kv, 9, ptr, size, 1, 1, 16, 4, None, 0, None) == bad
    assert lib.spa_compact_tokens(kv, 0, None, None, 1, 1, 16, 4, None, 0, None) == bad  # nothing to move
    assert lib.spa_compact_tokens(kv, 0, None, None, 1, 1, 16, 4, 16, 0, None) == bad


def test_restatements():
    """The oracle's layout is the documented one and agrees with int4_values; its error stays
    within half a step of the group's scale (and fp16's rounding of the zero)."""
    gen = torch.Generator().manual_seed(0)
    for dim in (32, 96, 256):
        x = torch.randn(3, 2, 5, dim, generator=gen)
        codes, scales = ref.int4_quantise(x)
        assert codes.shape == (3, 2, 5, dim // 2) and scales.shape == (3, 2, 5, 2, dim // 32)
        val = ref.int4_dequantise((codes, scales))
        assert torch.equal(spa.int4_values((codes, scales)), val.float())
        g = dim // 32
        for d in (0, 5, 31, dim - 1):
            j, r = d // 32, d % 32
            word = codes.view(torch.int16)[..., (r // 4) * g + j].int() & 0xffff
            n = (word >> (4 * (r % 4))) & 15
            assert torch.equal(val[..., d], scales[..., 0, j].double() * n + scales[..., 1, j].double())
        s = scales[..., 0, :].double().repeat_interleave(32, -1)
        z = scales[..., 1, :].double().repeat_interleave(32, -1)
        # n is clamped to 15, and 15 s may fall short of the range by 15 half steps of fp16
        assert ((val - x.double()).abs() <= 0.5 * s + 15 * s * 2.0 ** -11 + z.abs() * 2.0 ** -11).all()
