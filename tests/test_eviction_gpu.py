"""Accumulated attention weight, the choice of the tokens that stay, and their move, on the GPU
against 64-bit restatements.  Selections and moved rows are exact.  The weights' tolerance:
a probability is off by a relative 2 (D + 8) 2^-24 Q + N 2^-24 + 2^-20, with Q = max_t
sum_d |q_d k_d| / sqrt(D) (D + 8 roundings of an fp32 score, in numerator and denominator, the
sum over N tokens, exp2); outputs of 16 bits add their own half step and 2^-16 of max |v| for
probabilities held as two bf16 halves."""

import pytest
import torch

import attention_b200 as spa
import oracle.small_cache as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    assert spa.device_error_flags() == 0


def plain_cache(batch, heads, page, dim, tokens, dtype, gen):
    pages = -(-tokens // page)
    n = batch * pages + 1
    table = torch.randperm(n, generator=gen)[: batch * pages].view(batch, pages).to(torch.int32)
    pools, full = [], []
    for _ in range(2):
        x = torch.randn(batch, heads, pages * page, dim, generator=gen).to(dtype)
        x[:, :, tokens:] = float("nan")  # behind the sequence: must not be read
        pool = torch.full((n, heads, page, dim), float("nan"), dtype=dtype)
        for b in range(batch):
            for g in range(pages):
                pool[table[b, g]] = x[b, :, g * page:(g + 1) * page]
        pools.append(pool)
        full.append(torch.nan_to_num(x))
    return *pools, table, *full


def tolerances(q, k, v, n, dtype):
    q_size = (q.double().abs() @ k.double().abs().flatten(0, 2).amax(0)).max() / q.size(2) ** 0.5
    rel = (2 * (q.size(2) + 8) * 2.0 ** -24 * q_size + n * 2.0 ** -24 + 2.0 ** -20).item()
    return rel, (rel + (0 if dtype == torch.float32 else 2.0 ** -16)) * v.double().abs().max().item()


# ---------------------------------------------------------------- weights of a plain cache
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [(4, 4), (20, 4), (12, 1), (33, 3)])
@pytest.mark.parametrize("dim", [32, 40, 64, 128, 256])
def test_decode_weights_plain(dtype, heads, dim):
    hq, hkv = heads
    gen = torch.Generator().manual_seed(hq + dim)
    page = 16 if hkv > 1 else 27
    lens = [150, 0, 1, 64]
    k, v, table, kf, vf = plain_cache(4, hkv, page, dim, 150, dtype, gen)
    q = torch.randn(4, hq, dim, generator=gen).to(dtype)
    for window in (0, 50):
        w0 = torch.rand(4, hkv, 155, generator=gen)
        w = w0.to(DEV)
        out = spa.paged_decode_attention(q.to(DEV), k.to(DEV), v.to(DEV), page_table=table.to(DEV),
                                         context_lens=torch.tensor(lens, device=DEV), local_window=window, weights=w)
        tokens = [torch.arange(max(0, n - window) if window else 0, n) for n in lens]
        want, ww = ref.attention_weights(q, kf, vf, tokens)
        rel, tol = tolerances(q, kf, vf, 150, dtype)
        o = out.double().cpu()
        assert ((o - want).abs() <= tol + torch.finfo(dtype).eps / 2 * want.abs()).all(), (o - want).abs().max()
        total = torch.nn.functional.pad(ww, (0, 155 - ww.size(2)))[..., :155] + w0.double()
        assert ((w.double().cpu() - total).abs() <= rel * (total - w0) + 2.0 ** -23 * total).all()
        assert torch.equal(w.cpu()[total == w0], w0[total == w0])  # untouched where nothing was added


def test_decode_weights_contiguous_and_long():
    gen = torch.Generator().manual_seed(1)
    for dtype, dim in ((torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)):
        n = 3001
        k, v = (torch.randn(2, 2, n, dim, generator=gen).to(dtype) for _ in range(2))
        q = torch.randn(2, 8, dim, generator=gen).to(dtype)
        w = torch.zeros(2, 2, n, device=DEV)
        out = spa.paged_decode_attention(q.to(DEV), k.to(DEV), v.to(DEV), weights=w)
        want, ww = ref.attention_weights(q, k, v, [torch.arange(n)] * 2)
        rel, tol = tolerances(q, k, v, n, dtype)
        assert ((out.double().cpu() - want).abs() <= tol + torch.finfo(dtype).eps / 2 * want.abs()).all()
        assert ((w.double().cpu() - ww).abs() <= rel * ww).all()
        # what the call without weights returns, within both kernels' tolerances
        plain = spa.paged_decode_attention(q.to(DEV), k.to(DEV), v.to(DEV))
        assert ((plain.double() - out.double()).abs().max() <= 2e-2)


def test_weights_shorter_than_the_context_are_reported():
    gen = torch.Generator().manual_seed(1)
    k = torch.randn(1, 1, 40, 64, generator=gen).to(DEV)
    q = torch.randn(1, 1, 64, generator=gen).to(DEV)
    w, full = torch.zeros(1, 1, 39, device=DEV), torch.zeros(1, 1, 40, device=DEV)
    spa.paged_decode_attention(q, k, k, weights=full)
    assert spa.device_error_flags() == 0
    spa.paged_decode_attention(q, k, k, weights=w)
    assert spa.device_error_flags() == 4
    assert torch.equal(w, full[..., :39])


# ---------------------------------------------------------------- selection
@pytest.mark.parametrize("tokens,budget,recent", [(1, 1, 0), (5, 2, 1), (100, 100, 3), (1000, 37, 0), (1000, 999, 5),
                                                  (2049, 700, 700), (2049, 700, 10000), (5000, 1, 0), (9000, 4000, 64)])
def test_select_tokens(tokens, budget, recent):
    gen = torch.Generator().manual_seed(tokens + budget)
    w = torch.rand(4, 3, tokens, generator=gen)
    w[0] = (w[0] * 4).floor()            # many ties
    w[1, 0] = 0.0                        # one value only
    w[1, 1, ::3] = float("nan")
    w[1, 2, ::5] = float("inf")
    w[2, 0] = -w[2, 0]
    w[2, 1, ::2] = -0.0
    w[2, 1, 1::2] = 0.0
    w[2, 2] *= 1e-42                     # subnormal
    lens = [tokens, tokens, max(1, tokens - 3), tokens // 2]
    keep, kept = spa.select_tokens(w.to(DEV), torch.tensor(lens, device=DEV), budget=budget, recent=recent)
    want, want_kept = ref.select_tokens(w, lens, budget, recent)
    assert torch.equal(keep.cpu(), want) and torch.equal(kept.cpu(), want_kept)


@pytest.mark.parametrize("tokens", [300_000, 400_000])
def test_select_long_rows(tokens):
    """Rows that just stay in shared memory, and rows that do not."""
    gen = torch.Generator(device=DEV).manual_seed(tokens)
    w = torch.rand(1, 2, tokens, generator=gen, device=DEV)
    w[:, 1] = (w[:, 1] * 50).floor()
    budget, recent = 70_000, 1000
    keep, kept = spa.select_tokens(w, torch.tensor([tokens], device=DEV), budget=budget, recent=recent)
    key = w.clone()
    key[..., tokens - recent:] = 1e9
    order = torch.sort(key, dim=2, descending=True, stable=True).indices[..., :budget]
    assert torch.equal(keep, order.sort(2).values.int()) and kept.item() == budget


def test_select_lengths_outside_the_tensor():
    w = torch.rand(3, 2, 50)
    lens = [0, -4, 1000]
    keep, kept = spa.select_tokens(w.to(DEV), torch.tensor(lens, device=DEV), budget=20, recent=4)
    want, want_kept = ref.select_tokens(w, lens, 20, 4)
    assert torch.equal(keep.cpu(), want) and torch.equal(kept.cpu(), want_kept)


# ---------------------------------------------------------------- compaction
@pytest.mark.parametrize("dim", [3, 24, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.uint8])
def test_compact_tokens(dtype, dim):
    gen = torch.Generator().manual_seed(dim)
    batch, heads, page, tokens, budget = 3, 2, 13, 900, 420
    pages = -(-tokens // page)
    table = torch.randperm(batch * pages, generator=gen).view(batch, pages).to(torch.int32)
    pools = [torch.randint(0, 255, (batch * pages, heads, page, dim), generator=gen).to(dtype) for _ in range(2)]
    w = torch.rand(batch, heads, tokens, generator=gen)
    keep, _ = ref.select_tokens(w, [tokens, 500, 100], budget, 50)
    dev = [p.to(DEV) for p in pools]
    wd = w.to(DEV)
    spa.compact_tokens(dev, table.to(DEV), keep.to(DEV), weights=wd)
    for p, d in zip(pools, dev):
        assert torch.equal(d.cpu(), ref.compact_rows(p, table, keep))
    want = torch.where(keep >= 0, w.gather(2, keep.long().clamp(min=0)), 0)
    assert torch.equal(wd.cpu()[..., :budget], want) and (wd[..., budget:] == 0).all()


def test_compact_refuses_lists_out_of_order():
    """Each bad list leaves its own (sequence, kv head) as it was, and the others move."""
    bad = [[3, 2, -1, -1], [1, 1, 2, 3], [0, -1, 2, 3], [0, 1, -2, -1], [0, 1, 2, 99]]
    keep = torch.tensor(bad + [[1, 3, 4, 6]], dtype=torch.int32)[None]  # [1, 6 heads, 4]
    pool = torch.arange(4 * 6 * 4 * 4, dtype=torch.float32).view(4, 6, 4, 4)
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    w = torch.rand(1, 6, 8)
    pd, wd = pool.to(DEV), w.to(DEV)
    spa.compact_tokens((pd,), table.to(DEV), keep.to(DEV), weights=wd)
    assert spa.device_error_flags() & 4
    want, ww = pool.clone(), w.clone()
    for j, t in enumerate((1, 3, 4, 6)):
        want[table[0, j // 4], 5, j % 4] = pool[table[0, t // 4], 5, t % 4]
    ww[0, 5] = 0
    ww[0, 5, :4] = w[0, 5, [1, 3, 4, 6]]
    assert torch.equal(pd.cpu(), want) and torch.equal(wd.cpu(), ww)


def test_compact_without_a_page_leaves_the_row_out():
    pool = torch.arange(3 * 1 * 2 * 4, dtype=torch.float32).view(3, 1, 2, 4)
    table = torch.tensor([[0, -1, 2]], dtype=torch.int32)
    pd = pool.to(DEV)
    spa.compact_tokens((pd,), table.to(DEV), torch.tensor([[[1, 2, 4]]], dtype=torch.int32, device=DEV))
    assert spa.device_error_flags() == 2
    want = pool.clone()
    want[0, 0, 0] = pool[0, 0, 1]  # token 1 moves; token 2 has no page; token 4's destination has none
    assert torch.equal(pd.cpu(), want)


# ---------------------------------------------------------------- the operators together
@pytest.mark.parametrize("kind", ["int4", "bf16"])
def test_serving_loop_with_eviction(kind):
    """Prompt append, steps with accumulated weights, eviction whenever a sequence outgrows its
    room, on a scattered cache; every step's output and weights against a 64-bit model of the
    cache that keeps each head's surviving tokens."""
    gen = torch.Generator().manual_seed(21)
    batch, hq, hkv, dim, page, room, budget, recent = 2, 8, 2, 64, 16, 96, 40, 12
    pages = room // page
    dt = torch.bfloat16
    if kind == "int4":
        cache = spa.PagedKVCacheInt4(batch * pages, hkv, page, dim, batch=batch, max_pages_per_seq=pages)
    else:
        cache = spa.PagedKVCache(batch * pages, hkv, page, dim, batch=batch, max_pages_per_seq=pages)
    cache.page_table.copy_(torch.randperm(batch * pages, generator=gen).view(batch, pages).to(torch.int32))
    stored = (lambda x: ref.int4_dequantise(ref.int4_quantise(x))) if kind == "int4" else (lambda x: x.double())
    weights = torch.zeros(batch, hkv, room, device=DEV)
    lens = [70, 33]
    prompt = [torch.randn(batch, hkv, 70, dim, generator=gen).to(dt) for _ in range(2)]
    zero = torch.zeros(batch, dtype=torch.int32, device=DEV)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    if kind == "int4":
        spa.kv_append_int4(cache.k, cache.v, cache.page_table, *(x.to(DEV) for x in prompt), zero, new_lens=n)
    else:
        for t in range(70):
            at = torch.where(n > t, t, -1)
            spa.kv_append(cache.k, cache.v, cache.page_table, *(x[:, :, t].to(DEV) for x in prompt), at)
    cache.context_lens.copy_(n)
    model = [[[stored(x[b, h, : lens[b]]) for x in prompt] for h in range(hkv)] for b in range(batch)]
    acc = [[torch.zeros(lens[b], dtype=torch.float64) for _ in range(hkv)] for b in range(batch)]
    evictions = 0
    for step in range(75):
        new = [torch.randn(batch, hkv, dim, generator=gen).to(dt) for _ in range(2)]
        q = torch.randn(batch, hq, dim, generator=gen).to(dt)
        append = spa.kv_append_int4 if kind == "int4" else spa.kv_append
        append(cache.k, cache.v, cache.page_table, *(x.to(DEV) for x in new), cache.context_lens)
        cache.context_lens += 1
        decode = spa.paged_decode_attention_int4 if kind == "int4" else spa.paged_decode_attention
        out = decode(q.to(DEV), cache.k, cache.v, page_table=cache.page_table, context_lens=cache.context_lens,
                     weights=weights)
        for b in range(batch):
            for h in range(hkv):
                for i in range(2):
                    model[b][h][i] = torch.cat((model[b][h][i], stored(new[i][b, h])[None]))
                k, v = model[b][h]
                qs = q[b].view(hkv, -1, dim)[h].double()
                p = torch.softmax(qs @ k.T / dim ** 0.5, -1)
                want = p @ v
                got = out[b].view(hkv, -1, dim)[h].double().cpu()
                # scores of these sizes are off by under 2^-12, P by 2^-10, the output by half a bf16 step
                assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -9 * v.abs().max() * 3).all()
                acc[b][h] = torch.cat((acc[b][h], torch.zeros(1, dtype=torch.float64))) + p.sum(0)
                got_w = weights[b, h].double().cpu()
                m = acc[b][h].numel()
                assert ((got_w[:m] - acc[b][h]).abs() <= 2.0 ** -11 * acc[b][h]).all() and (got_w[m:] == 0).all()
        if int(cache.context_lens.max()) >= room - 8:
            evictions += 1
            before = cache.context_lens.tolist()
            chosen, _ = ref.select_tokens(weights.cpu(), before, budget, recent)
            keep = spa.evict_tokens(cache, weights, budget=budget, recent=recent)
            assert torch.equal(keep.cpu(), chosen)
            assert cache.context_lens.tolist() == [min(x, budget) for x in before]
            for b in range(batch):
                for h in range(hkv):
                    ids = chosen[b, h][chosen[b, h] >= 0].long()
                    model[b][h] = [x[ids] for x in model[b][h]]
                    acc[b][h] = acc[b][h][ids]
    assert evictions >= 2


def test_eviction_in_a_graph():
    gen = torch.Generator().manual_seed(9)
    cache = spa.PagedKVCacheInt4(8, 2, 16, 64, batch=2, max_pages_per_seq=4)
    cache.page_table.copy_(torch.randperm(8, generator=gen).view(2, 4).to(torch.int32))
    w = torch.zeros(2, 2, 64, device=DEV)
    x = torch.zeros(2, 2, 64, 64, device=DEV)
    zero = torch.zeros(2, dtype=torch.int32, device=DEV)

    def step():
        spa.kv_append_int4(cache.k, cache.v, cache.page_table, x, x, zero)
        return spa.evict_tokens(cache, w, budget=20, recent=5)

    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        keep = step()
    for lens in ([64, 10], [33, 64]):
        wh, xh = torch.rand(2, 2, 64, generator=gen), torch.randn(2, 2, 64, 64, generator=gen)
        w.copy_(wh)
        x.copy_(xh)
        cache.context_lens.copy_(torch.tensor(lens))
        g.replay()
        want, kept = ref.select_tokens(wh, lens, 20, 5)
        assert torch.equal(keep.cpu(), want) and torch.equal(cache.context_lens.cpu(), kept)
        got, _ = spa.kv_read_int4(cache.k, cache.v, cache.page_table, zero, 20, lens=cache.context_lens,
                                  dtype=torch.float32)
        val = ref.int4_dequantise(ref.int4_quantise(xh)).float()
        for b in range(2):
            for h in range(2):
                ids = want[b, h][want[b, h] >= 0].long()
                assert torch.equal(got[b, h, : ids.numel()].cpu(), val[b, h, ids])


# ---------------------------------------------------------------- refusals
def test_refusals():
    w = torch.zeros(1, 2, 8, device=DEV)
    lens = torch.zeros(1, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="CUDA"):
        spa.select_tokens(w.cpu(), lens, budget=4, recent=1)
    with pytest.raises(ValueError, match="float32"):
        spa.select_tokens(w.half(), lens, budget=4, recent=1)
    with pytest.raises(ValueError, match="budget"):
        spa.select_tokens(w, lens, budget=0, recent=1)
    with pytest.raises(ValueError, match="budget"):
        spa.select_tokens(w, lens, budget=1, recent=-1)
    with pytest.raises(ValueError, match="context_lens"):
        spa.select_tokens(w, torch.zeros(2, dtype=torch.int32, device=DEV), budget=1, recent=0)
    pool = torch.zeros(2, 2, 4, 8, device=DEV)
    table = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    keep = torch.full((1, 2, 4), -1, dtype=torch.int32, device=DEV)
    for bad in (dict(keep=keep.long()), dict(keep=keep[:, :1].contiguous()), dict(pools=()), dict(pools=(pool, pool[:, :1])),
                dict(pools=(pool.transpose(1, 2),)), dict(weights=w[..., :3].contiguous()), dict(weights=w.half()),
                dict(page_table=torch.zeros(2, 2, dtype=torch.int32, device=DEV)), dict(pools=(pool.cpu(),))):
        args = dict(pools=(pool,), page_table=table, keep=keep, weights=None) | bad
        with pytest.raises(ValueError):
            spa.compact_tokens(args["pools"], args["page_table"], args["keep"], weights=args["weights"])
    q = torch.zeros(1, 2, 8, device=DEV)
    with pytest.raises(ValueError, match="weights"):
        spa.paged_decode_attention(q, pool[:1].contiguous(), pool[:1].contiguous(), weights=w[:, :1].contiguous())
    with pytest.raises(ValueError, match="weights"):
        spa.paged_decode_attention(q, pool[:1].contiguous(), pool[:1].contiguous(), weights=w.double())
