"""Shapes of the 4-bit cache beside those of test_int4_gpu.py: head sizes of 5, 6 and 7 groups, pages of
one token and of thousands, negative lengths.  Append and read-back are exact; decode's tolerance is
that of test_int4_gpu.py."""

import pytest
import torch

import attention_b200 as spa
import oracle.small_cache as ref
from test_int4_gpu import bounds, check_out, make_cache, to_dev

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    assert spa.device_error_flags() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [160, 192, 224])
@pytest.mark.parametrize("t", [1, 5, 33, 131])
def test_append_and_read(dtype, dim, t):
    """Rows a step (32 // groups: 6, 5, 4) do not divide the tokens of a warp."""
    gen = torch.Generator().manual_seed(dim + t)
    batch, heads, page = 2, 3, 9
    pages = -(-(t + 4) // page)
    cache = spa.PagedKVCacheInt4(batch * pages, heads, page, dim, batch=batch, max_pages_per_seq=pages)
    cache.page_table.copy_(torch.randperm(batch * pages, generator=gen).view(batch, pages).to(torch.int32))
    new = [torch.randn(batch, heads, t, dim, generator=gen).to(dtype) for _ in range(2)]
    pos = torch.tensor([0, 4], dtype=torch.int32, device=DEV)
    lens = torch.tensor([t, max(0, t - 2)], dtype=torch.int32, device=DEV)
    spa.kv_append_int4(cache.k, cache.v, cache.page_table, *(x.to(DEV) for x in new), pos, new_lens=lens)
    table = cache.page_table.cpu()
    for pool, x in zip((cache.k, cache.v), new):
        want = [torch.zeros_like(p.cpu()) for p in pool]
        for part, (dst, src) in enumerate(zip(want, ref.int4_quantise(x))):
            for b in range(batch):
                for i in range(int(lens[b])):
                    tok = int(pos[b]) + i
                    dst[table[b, tok // page], :, tok % page] = src[b, :, i]
            assert torch.equal(pool[part].cpu(), dst)
    got = spa.kv_read_int4(cache.k, cache.v, cache.page_table, pos, t, lens=lens, dtype=dtype)
    for g, x in zip(got, new):
        want = ref.int4_dequantise(ref.int4_quantise(x)).float().to(dtype)
        want[1, :, int(lens[1]):] = 0
        assert torch.equal(g.cpu(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("page,n", [(1, 1100), (5, 1100), (31, 700), (4096, 5000)])
@pytest.mark.parametrize("dim", [96, 128])
def test_decode_pages_of_any_size(dtype, page, n, dim):
    gen = torch.Generator().manual_seed(page)
    k, v, table, kval, vval, kc = make_cache(2, 2, page, dim, n, gen, spare=0)
    q = torch.randn(2, 8, dim, generator=gen).to(dtype)
    more = dict(page_table=table.to(DEV), context_lens=torch.tensor([n, n // 2], device=DEV))
    tokens = [torch.arange(n), torch.arange(n // 2)]
    want, ww = ref.attention_weights(q, torch.nan_to_num(kval), torch.nan_to_num(vval), tokens)
    rel, tol = bounds(q, kc, kval, vval, tokens, dtype)
    w = torch.zeros(2, 2, n, device=DEV)
    check_out(spa.paged_decode_attention_int4(q.to(DEV), to_dev(k), to_dev(v), weights=w, **more), want, tol, dtype)
    assert ((w.double().cpu() - ww[..., :n]).abs() <= rel * ww[..., :n]).all()
    sel = torch.tensor([[0, (n - 1) // page], [0, -1]])
    tokens = [torch.cat([torch.arange(n - 40, n)] + [torch.arange(s * page, min((s + 1) * page, n)) for s in (0, (n - 1) // page)]),
              torch.cat([torch.arange(n // 2 - 40, n // 2), torch.arange(min(page, n // 2))])]
    want, _ = ref.attention_weights(q, torch.nan_to_num(kval), torch.nan_to_num(vval), tokens)
    out = spa.paged_gather_decode_attention_int4(q.to(DEV), to_dev(k), to_dev(v), sel.to(DEV), local_window=40,
                                                 block_size=page, **more)
    check_out(out, want, bounds(q, kc, kval, vval, tokens, dtype)[1], dtype)


def test_negative_lengths_are_empty():
    gen = torch.Generator().manual_seed(0)
    k, v, table, _, _, _ = make_cache(2, 2, 16, 64, 50, gen)
    w = torch.zeros(2, 2, 50, device=DEV)
    out = spa.paged_decode_attention_int4(torch.randn(2, 4, 64, device=DEV), to_dev(k), to_dev(v), weights=w,
                                          page_table=table.to(DEV), context_lens=torch.tensor([-3, 50], device=DEV))
    assert (out[0] == 0).all() and (w[0] == 0).all() and (out[1] != 0).any()
    assert ((w[1].sum(1) - 2).abs() <= 2.0 ** -18).all()  # two heads each: 50 additions and exp2
