"""Batches of no sequence."""

import pytest
import torch

import attention_b200 as spa

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_decode_of_no_sequence_is_empty():
    cache = spa.PagedKVCacheInt4(2, 2, 4, 64, batch=0, max_pages_per_seq=2)
    pool = torch.zeros(2, 2, 4, 64, device=DEV)
    more = dict(page_table=cache.page_table, context_lens=cache.context_lens)
    q, w = torch.zeros(0, 4, 64, device=DEV), torch.zeros(0, 2, 8, device=DEV)
    for weights in (None, w):
        out = spa.paged_decode_attention_int4(q, cache.k, cache.v, weights=weights, **more)
        assert out.shape == (0, 4, 64) and out.dtype == q.dtype
    assert spa.paged_decode_attention(q, pool, pool, weights=w, **more).shape == (0, 4, 64)
    empty = pool[:0].contiguous()
    assert spa.paged_decode_attention(q, empty, empty, weights=w[..., :4].contiguous()).shape == (0, 4, 64)
