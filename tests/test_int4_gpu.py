"""The 4-bit cache on the GPU against its 64-bit restatement.

Codes and scales are compared bit for bit (the format fixes every rounding).  Attention is
compared on the values the cache stands for.  Its tolerance follows from the arithmetic.  With
Q = max_t sum_d |q_d| (|s n_d| + |z|) / sqrt(D), every score is a sum of terms of total size Q,
taken in fp32 (at most D + 8 roundings), so a probability is off by a relative
2 delta, delta = (D + 8) 2^-24 Q (the sum in the denominator has the same error), plus N 2^-24
for the sums over N tokens and 2^-20 for exp2 and for what a pair of fp16 halves drops.  A
16-bit output allows each probability two fp16 roundings, 2^-10, and its own half step."""

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


def make_cache(batch, kv_heads, page, dim, tokens, gen, *, scale=1.0, spare=1):
    """A scattered cache of `tokens` tokens per sequence; pages no sequence owns hold NaN."""
    pages = -(-tokens // page) + spare
    n = batch * pages + 2
    table = torch.randperm(n, generator=gen)[: batch * pages].view(batch, pages).to(torch.int32)
    full = []
    for _ in range(2):
        x = torch.randn(batch, kv_heads, pages * page, dim, generator=gen) * scale
        x = x * (0.5 + 2 * torch.rand(dim, generator=gen) ** 4) + 0.3
        codes, scales = ref.int4_quantise(x)
        scales[:, :, tokens:] = float("nan")  # behind the sequence: must not be read
        pool = (torch.full((n, kv_heads, page, dim // 2), 255, dtype=torch.uint8),
                torch.full((n, kv_heads, page, 2, dim // 32), float("nan"), dtype=torch.float16))
        for b in range(batch):
            for g in range(pages):
                for dst, src in zip(pool, (codes, scales)):
                    dst[table[b, g]] = src[b, :, g * page:(g + 1) * page]
        full.append((pool, (codes, scales)))
    (k, kc), (v, vc) = full
    return k, v, table, ref.int4_dequantise(kc), ref.int4_dequantise(vc), kc


def to_dev(pool):
    return tuple(t.to(DEV) for t in pool)


def bounds(q, kc, kval, vval, tokens, dtype):
    """(relative error of a probability, absolute error of an output) per sequence."""
    d = q.size(2)
    n = torch.cat([t for t in tokens]).numel() if tokens else 0
    zero = kc[1][..., 1, torch.arange(d) // 32].double()
    size = (kval - zero).abs() + zero.abs()
    size = torch.nan_to_num(size).flatten(0, 2).amax(0)
    q_size = (q.double().abs() @ size).max() / d ** 0.5
    rel = 2 * (d + 8) * 2.0 ** -24 * q_size + max(n, 1) * 2.0 ** -24 + 2.0 ** -20
    big = 3 * torch.nan_to_num(vval).abs().max()  # |s n| + |z| <= 3 max |v|
    out = rel if dtype == torch.float32 else rel + 2.0 ** -10
    return rel.item(), (out * big).item()


def check_out(out, want, tol, dtype):
    o = out.double().cpu()
    assert torch.isfinite(o).all()
    err = (o - want).abs()
    assert (err <= tol + torch.finfo(dtype).eps / 2 * want.abs()).all(), (err.max().item(), tol)


# ---------------------------------------------------------------- append and read-back
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 256])
def test_append_is_the_format(dtype, dim):
    gen = torch.Generator().manual_seed(dim)
    batch, heads, page, t = 3, 2, 7, 20
    cache = spa.PagedKVCacheInt4(24, heads, page, dim, batch=batch, max_pages_per_seq=7)
    cache.page_table.copy_(torch.randperm(24, generator=gen)[:21].view(3, 7).to(torch.int32))
    new = [torch.randn(batch, heads, t, dim, generator=gen) * 3 for _ in range(2)]
    new[0][0, 0, 0] = 0.1           # one value only
    new[0][0, 0, 1, :32] = 0.0
    new[0][0, 0, 2, 3] = float("nan")
    new[0][0, 1, 2, 5] = float("inf")
    new[0][1, 0, 0] *= 1e-6         # scales among fp16's smallest
    new[0][1, 0, 1, ::2] = 6e4      # near fp16's largest
    if dtype != torch.float16:
        new[0][1, 0, 2, ::2] = -1e6  # past it: saturates
    new = [x.to(dtype) for x in new]
    pos = torch.tensor([0, 5, 13], dtype=torch.int32)
    lens = torch.tensor([20, 0, 11], dtype=torch.int32)
    k0 = tuple(t.clone() for t in cache.k)
    spa.kv_append_int4(cache.k, cache.v, cache.page_table, new[0].to(DEV), new[1].to(DEV), pos.to(DEV),
                       new_lens=lens.to(DEV))
    table = cache.page_table.cpu()
    for pool, x, before in ((cache.k, new[0], k0), (cache.v, new[1], None)):
        codes, scales = ref.int4_quantise(x)
        want = [torch.zeros_like(t.cpu()) for t in pool]
        for b in range(batch):
            for i in range(int(lens[b])):
                tok = int(pos[b]) + i
                want[0][table[b, tok // page], :, tok % page] = codes[b, :, i]
                want[1][table[b, tok // page], :, tok % page] = scales[b, :, i]
        assert torch.equal(pool[0].cpu(), want[0])
        assert torch.equal(torch.nan_to_num(pool[1].cpu().float(), nan=1e9), torch.nan_to_num(want[1].float(), nan=1e9))
        assert torch.equal(torch.nan_to_num(spa.int4_values(pool).cpu()),
                           torch.nan_to_num(ref.int4_dequantise(pool).float()))
    got = spa.kv_read_int4(cache.k, cache.v, cache.page_table, pos.to(DEV), t, lens=lens.to(DEV), dtype=dtype)
    for g, x in zip(got, new):
        want = ref.int4_dequantise(ref.int4_quantise(x)).float().to(dtype)
        for b in range(batch):
            want[b, :, int(lens[b]):] = 0
        assert torch.equal(torch.nan_to_num(g.cpu().float(), nan=7e7), torch.nan_to_num(want.float(), nan=7e7))


def test_append_takes_strided_views_and_single_tokens():
    gen = torch.Generator().manual_seed(3)
    b, h, t, d = 2, 4, 5, 64
    qkv = torch.randn(b, t, 3, h, d, generator=gen).to(torch.bfloat16).to(DEV)
    k_new, v_new = qkv[:, :, 1].transpose(1, 2), qkv[:, :, 2].transpose(1, 2)
    odd = torch.randn(b, h, t, d + 1, generator=gen).to(torch.bfloat16).to(DEV)[..., 1:]  # 2-byte aligned rows
    pos = torch.zeros(b, dtype=torch.int64, device=DEV)
    for kn, vn in ((k_new, v_new), (odd, odd)):
        a, c = (spa.PagedKVCacheInt4(4, h, 4, d, batch=b, max_pages_per_seq=2) for _ in range(2))
        for cache in (a, c):
            cache.page_table.copy_(torch.tensor([[2, 0], [1, 3]], dtype=torch.int32))
        spa.kv_append_int4(a.k, a.v, a.page_table, kn, vn, pos)
        for i in range(t):
            spa.kv_append_int4(c.k, c.v, c.page_table, kn[:, :, i].contiguous(), vn[:, :, i], pos + i)
        for x, y in zip((*a.k, *a.v), (*c.k, *c.v)):
            assert torch.equal(x, y)
        want = ref.int4_dequantise(ref.int4_quantise(kn.cpu())).float()
        got, _ = spa.kv_read_int4(a.k, a.v, a.page_table, pos, t, dtype=torch.float32)
        assert torch.equal(got.cpu(), want)


def test_append_and_read_outside_the_pages():
    """Negative tokens are skipped; a token without a page is skipped and reported."""
    b, h, d = 2, 1, 32
    cache = spa.PagedKVCacheInt4(2, h, 4, d, batch=b, max_pages_per_seq=1)
    cache.page_table.copy_(torch.tensor([[0], [-1]], dtype=torch.int32))
    x = torch.randn(b, h, 6, d, device=DEV)
    spa.kv_append_int4(cache.k, cache.v, cache.page_table, x, x, torch.tensor([-3, -9], device=DEV))
    assert spa.device_error_flags() == 0
    assert (cache.k[1][0, 0, :3, 0] > 0).all() and (cache.k[1][0, 0, 3:] == 0).all() and (cache.k[1][1] == 0).all()
    got, _ = spa.kv_read_int4(cache.k, cache.v, cache.page_table, torch.tensor([-3, -9], device=DEV), 6,
                              dtype=torch.float32)
    want = ref.int4_dequantise(ref.int4_quantise(x.cpu())).float()
    assert torch.equal(got[0, :, 3:].cpu(), want[0, :, 3:]) and (got[0, :, :3] == 0).all() and (got[1] == 0).all()
    spa.kv_append_int4(cache.k, cache.v, cache.page_table, x, x, torch.tensor([2, 0], device=DEV))
    assert spa.device_error_flags() == 2
    assert (cache.k[1][1] == 0).all()
    spa.kv_read_int4(cache.k, cache.v, cache.page_table, torch.tensor([2 ** 31 - 3, -9], device=DEV), 6)
    assert spa.device_error_flags() == 2


# ---------------------------------------------------------------- dense and windowed decode
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [(4, 4), (8, 2), (20, 4), (12, 1), (33, 3)])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 256])
def test_decode_ragged(dtype, heads, dim):
    hq, hkv = heads
    gen = torch.Generator().manual_seed(dim + hq)
    page = 16 if hq % 2 else 33
    lens = [0, 1, 31, 97, 200]
    k, v, table, kval, vval, kc = make_cache(len(lens), hkv, page, dim, 200, gen)
    q = torch.randn(len(lens), hq, dim, generator=gen).to(dtype)
    for window in (0, 40):
        tokens = [torch.arange(max(0, n - window) if window else 0, n) for n in lens]
        out = spa.paged_decode_attention_int4(q.to(DEV), to_dev(k), to_dev(v), page_table=table.to(DEV),
                                              context_lens=torch.tensor(lens, device=DEV), local_window=window)
        want, _ = ref.attention_weights(q, torch.nan_to_num(kval), torch.nan_to_num(vval), tokens)
        _, tol = bounds(q, kc, kval, vval, tokens, dtype)
        assert out.dtype == dtype
        check_out(out, want, tol, dtype)
        assert (out[0] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_decode_long_is_split(dtype, dim):
    gen = torch.Generator().manual_seed(dim)
    n = 5003
    k, v, table, kval, vval, kc = make_cache(1, 2, 64, dim, n, gen)
    q = torch.randn(1, 8, dim, generator=gen).to(dtype)
    out = spa.paged_decode_attention_int4(q.to(DEV), to_dev(k), to_dev(v), page_table=table.to(DEV),
                                          context_lens=torch.tensor([n], device=DEV))
    want, _ = ref.attention_weights(q, torch.nan_to_num(kval), torch.nan_to_num(vval), [torch.arange(n)])
    check_out(out, want, bounds(q, kc, kval, vval, [torch.arange(n)], dtype)[1], dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [1e-4, 60.0, 3000.0])
def test_decode_small_and_large_values(dtype, scale):
    """V far from 1 (group scales to several hundred), queries sized so that scores stay ordinary."""
    gen = torch.Generator().manual_seed(int(scale))
    k, v, table, kval, vval, kc = make_cache(2, 2, 32, 128, 700, gen, scale=scale)
    q = (torch.randn(2, 8, 128, generator=gen) / scale).to(dtype)
    # the first tokens of V are small, so that the largest scales come late
    out = spa.paged_decode_attention_int4(q.to(DEV), to_dev(k), to_dev(v), page_table=table.to(DEV),
                                          context_lens=torch.tensor([700, 500], device=DEV))
    tokens = [torch.arange(700), torch.arange(500)]
    want, _ = ref.attention_weights(q, torch.nan_to_num(kval), torch.nan_to_num(vval), tokens)
    check_out(out, want, bounds(q, kc, kval, vval, tokens, dtype)[1], dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("late", [False, True])
def test_decode_values_past_fp16(dtype, late):
    """Ranges whose middle (zero + 8 scales) fp16 could not hold: values of 0 to 2e5, in all tokens or
    in the last only.  (16-bit outputs: bf16 alone has the range.)"""
    gen = torch.Generator().manual_seed(17)
    k, v, table, _, _, _ = make_cache(1, 2, 16, 64, 400, gen)
    x = torch.rand(2, 1, 2, 400, 64, generator=gen) * 2e5
    if late:
        x[..., :390, :] /= 1e5
    full = [ref.int4_quantise(y) for y in x]
    for pool, (codes, scales) in zip((k, v), full):
        for g in range(25):
            pool[0][table[0, g]] = codes[0, :, g * 16:(g + 1) * 16]
            pool[1][table[0, g]] = scales[0, :, g * 16:(g + 1) * 16]
    kval, vval = (ref.int4_dequantise(f) for f in full)
    q = (torch.randn(1, 4, 64, generator=gen) / 1e5).to(dtype)
    tokens = [torch.arange(400)]
    out = spa.paged_decode_attention_int4(q.to(DEV), to_dev(k), to_dev(v), page_table=table.to(DEV),
                                          context_lens=torch.tensor([400], device=DEV))
    want, _ = ref.attention_weights(q, kval, vval, tokens)
    check_out(out, want, bounds(q, full[0], kval, vval, tokens, dtype)[1], dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_peaked_and_shifted_scores(dtype):
    """Scores of some hundreds, rising along the sequence, so that every tile moves the maximum."""
    gen = torch.Generator().manual_seed(5)
    k, v, table, _, vval, _ = make_cache(1, 1, 16, 64, 300, gen)
    ramp = torch.linspace(-40, 40, 304)[None, None, :, None] * torch.ones(1, 1, 304, 64)
    codes, scales = ref.int4_quantise(ramp)
    for g in range(table.size(1)):
        if g * 16 < 304:
            k[0][table[0, g]] = codes[0, :, g * 16:(g + 1) * 16]
            k[1][table[0, g]] = scales[0, :, g * 16:(g + 1) * 16]
    kval = ref.int4_dequantise((codes, scales))
    q = torch.full((1, 2, 64), 0.5)
    q[0, 1] = -0.5
    q = q.to(dtype)
    tokens = [torch.arange(300)]
    out = spa.paged_decode_attention_int4(q.to(DEV), to_dev(k), to_dev(v), page_table=table.to(DEV),
                                          context_lens=torch.tensor([300], device=DEV))
    want, _ = ref.attention_weights(q, kval, torch.nan_to_num(vval)[:, :, :304], tokens)
    check_out(out, want, bounds(q, (codes, scales), kval, vval, tokens, dtype)[1], dtype)


def test_nan_group_reaches_the_output_and_only_its_sequence():
    gen = torch.Generator().manual_seed(8)
    k, v, table, _, _, _ = make_cache(2, 1, 16, 64, 64, gen)
    k[1][table[0, 1], 0, 3, :, 1] = float("nan")
    q = torch.randn(2, 4, 64, generator=gen).to(torch.bfloat16)
    out = spa.paged_decode_attention_int4(q.to(DEV), to_dev(k), to_dev(v), page_table=table.to(DEV),
                                          context_lens=torch.tensor([64, 64], device=DEV))
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()


# ---------------------------------------------------------------- selected pages
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page", [16, 24, 64])
@pytest.mark.parametrize("window", [0, 30, 64])
def test_gather_decode(dtype, page, window):
    gen = torch.Generator().manual_seed(page + window)
    lens = [301, 5, 0]
    k, v, table, kval, vval, kc = make_cache(3, 2, page, 64, 301, gen)
    q = torch.randn(3, 6, 64, generator=gen).to(dtype)
    last = 300 // page
    sel = torch.tensor([[2, last, -1, 0], [0, -1, -1, 0], [-1, -1, -1, -1]])  # 0 twice in row 1: counted twice
    tokens = []
    for b, n in enumerate(lens):
        t = [torch.arange(max(0, n - window), n)]
        t += [torch.arange(s * page, min((s + 1) * page, n)) for s in sel[b].tolist() if s >= 0]
        tokens.append(torch.cat(t))
    out = spa.paged_gather_decode_attention_int4(q.to(DEV), to_dev(k), to_dev(v), sel.to(DEV), local_window=window,
                                                 block_size=page, page_table=table.to(DEV),
                                                 context_lens=torch.tensor(lens, device=DEV))
    want, _ = ref.attention_weights(q, torch.nan_to_num(kval), torch.nan_to_num(vval), tokens)
    check_out(out, want, bounds(q, kc, kval, vval, tokens, dtype)[1], dtype)


def test_bad_pages_are_skipped_and_reported():
    gen = torch.Generator().manual_seed(11)
    k, v, table, kval, vval, kc = make_cache(1, 2, 16, 64, 64, gen, spare=0)
    q = torch.randn(1, 4, 64, generator=gen)
    for bad in (-1, 10 ** 6):
        broken = table.clone()
        broken[0, 1] = bad
        tokens = [torch.cat((torch.arange(16), torch.arange(32, 64)))]
        w = torch.zeros(1, 2, 64, device=DEV)
        out = spa.paged_decode_attention_int4(q.to(DEV), to_dev(k), to_dev(v), page_table=broken.to(DEV),
                                              context_lens=torch.tensor([64], device=DEV), weights=w)
        assert spa.device_error_flags() == 2
        want, ww = ref.attention_weights(q, kval, vval, tokens)
        rel, tol = bounds(q, kc, kval, vval, tokens, torch.float32)
        check_out(out, want, tol, torch.float32)
        assert ((w.cpu() - ww).abs() <= rel * ww + 1e-30).all()
    # a selected page past the context, and a context past the table
    sel = torch.tensor([[0, 9]])
    out = spa.paged_gather_decode_attention_int4(q.to(DEV), to_dev(k), to_dev(v), sel.to(DEV), local_window=0,
                                                 block_size=16, page_table=table.to(DEV),
                                                 context_lens=torch.tensor([64], device=DEV))
    assert spa.device_error_flags() == 2
    tokens = [torch.arange(16)]
    check_out(out, ref.attention_weights(q, kval, vval, tokens)[0], bounds(q, kc, kval, vval, tokens, torch.float32)[1],
              torch.float32)
    out = spa.paged_decode_attention_int4(q.to(DEV), to_dev(k), to_dev(v), page_table=table.to(DEV),
                                          context_lens=torch.tensor([65], device=DEV))
    assert spa.device_error_flags() == 2
    tokens = [torch.arange(64)]
    check_out(out, ref.attention_weights(q, kval, vval, tokens)[0], bounds(q, kc, kval, vval, tokens, torch.float32)[1],
              torch.float32)


def test_offsets_past_32_bits():
    """Codes and scales of more than 2^32 bytes, the sequence's pages at both ends."""
    gen = torch.Generator().manual_seed(2)
    page, heads, d = 256, 8, 128
    n = (1 << 32) // (heads * page * 64) + 40
    q = torch.randn(1, 8, d, generator=gen).to(torch.bfloat16)
    table = torch.tensor([[n - 1, 0, n - 2]], dtype=torch.int32, device=DEV)
    k, v = ((torch.empty(n, heads, page, d // 2, dtype=torch.uint8, device=DEV),
             torch.empty(n, heads, page, 2, d // 32, dtype=torch.float16, device=DEV)) for _ in range(2))
    new = [torch.randn(1, heads, 3 * page - 5, d, generator=gen).to(torch.bfloat16) for _ in range(2)]
    spa.kv_append_int4(k, v, table, new[0].to(DEV), new[1].to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV))
    out = spa.paged_decode_attention_int4(q.to(DEV), k, v, page_table=table,
                                          context_lens=torch.tensor([3 * page - 5], device=DEV))
    kq = ref.int4_quantise(new[0])
    kval, vval = ref.int4_dequantise(kq), ref.int4_dequantise(ref.int4_quantise(new[1]))
    tokens = [torch.arange(3 * page - 5)]
    check_out(out, ref.attention_weights(q, kval, vval, tokens)[0], bounds(q, kq, kval, vval, tokens, q.dtype)[1], q.dtype)


def test_side_stream_and_graph_replay():
    gen = torch.Generator().manual_seed(4)
    k, v, table, kval, vval, kc = make_cache(2, 2, 32, 128, 1500, gen)
    kd, vd, td = to_dev(k), to_dev(v), table.to(DEV)
    lens = torch.tensor([1500, 40], dtype=torch.int32, device=DEV)
    q = torch.randn(2, 8, 128, generator=gen).to(torch.bfloat16).to(DEV)
    eager = spa.paged_decode_attention_int4(q, kd, vd, page_table=td, context_lens=lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = spa.paged_decode_attention_int4(q, kd, vd, page_table=td, context_lens=lens)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(eager, other)
    w = torch.zeros(2, 2, 1600, device=DEV)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        spa.kv_append_int4(kd, vd, td, q[:, :2], q[:, 2:4], lens - 1)
        out = spa.paged_decode_attention_int4(q, kd, vd, page_table=td, context_lens=lens, weights=w)
    for step in range(3):
        q.copy_(torch.randn(2, 8, 128, generator=gen))
        lens.copy_(torch.tensor([1400 + step, 41 + step]))
        w.zero_()
        g.replay()
        fresh = torch.zeros_like(w)
        again = spa.paged_decode_attention_int4(q, kd, vd, page_table=td, context_lens=lens, weights=fresh)
        assert torch.equal(out, again) and torch.equal(w, fresh)


def test_two_streams_and_two_graphs_at_once():
    """Calls that run side by side, eagerly and replayed, give what they give alone."""
    gen = torch.Generator().manual_seed(31)
    sets = []
    for i in range(2):
        k, v, table, _, _, _ = make_cache(3, 2, 32, 128, 2000, gen)
        lens = torch.tensor([2000, 700 + i, 31], dtype=torch.int32, device=DEV)
        sets.append((torch.randn(3, 8, 128, generator=gen).to(torch.bfloat16).to(DEV), to_dev(k), to_dev(v),
                     dict(page_table=table.to(DEV), context_lens=lens), torch.zeros(3, 2, 2000, device=DEV)))

    def step(s, w):
        w.zero_()
        return spa.paged_decode_attention_int4(s[0], s[1], s[2], weights=w, **s[3])

    want = [(step(s, s[4]), s[4].clone()) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(s, s[4])
        graphs.append((g, out))
    torch.cuda.synchronize()
    for _ in range(20):
        eager = []
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                w = torch.empty_like(sets[i][4])
                eager.append((step(sets[i], w), w))
        torch.cuda.synchronize()
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                graphs[i][0].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(eager[i][0], want[i][0]) and torch.equal(eager[i][1], want[i][1])
            assert torch.equal(graphs[i][1], want[i][0]) and torch.equal(sets[i][4], want[i][1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_queries_off_16_byte_boundaries(dtype):
    gen = torch.Generator().manual_seed(6)
    k, v, table, _, _, _ = make_cache(2, 2, 32, 64, 300, gen)
    args = (to_dev(k), to_dev(v))
    more = dict(page_table=table.to(DEV), context_lens=torch.tensor([300, 17], device=DEV))
    q = torch.randn(2, 8, 64, generator=gen).to(dtype).to(DEV)
    odd = torch.empty(q.numel() + 1, dtype=dtype, device=DEV)[1:].view(q.shape)
    odd.copy_(q)
    assert torch.equal(spa.paged_decode_attention_int4(odd, *args, **more),
                       spa.paged_decode_attention_int4(q, *args, **more))
    pool = torch.randn(8, 2, 32, 64, generator=gen).to(dtype).to(DEV)
    more["page_table"] = torch.arange(8, dtype=torch.int32, device=DEV).view(2, 4)
    more["context_lens"] = torch.tensor([100, 17], device=DEV)
    w = [torch.zeros(2, 2, 128, device=DEV) for _ in range(2)]
    a, b = (spa.paged_decode_attention(x, pool, pool, weights=y, **more) for x, y in zip((odd, q), w))
    # another kernel may serve the unaligned call: scores of these sizes (Q < 2^6, D + 8 = 72) agree to 2^-10
    assert ((a - b).abs() <= torch.finfo(dtype).eps * b.abs() + 2.0 ** -10).all()
    assert ((w[0] - w[1]).abs() <= 2.0 ** -10 * w[1]).all()


@pytest.mark.parametrize("batch,context", [(40, 900), (1100, 300), (700, 20)])
def test_decode_long_batches(batch, context):
    """Batches whose lengths are summed up by more than a warp, batches too long for that, and
    contexts that one CTA takes whole."""
    gen = torch.Generator().manual_seed(batch)
    page, pages = 64, -(-context // 64)
    cache = spa.PagedKVCacheInt4(batch * pages, 1, page, 32, batch=batch, max_pages_per_seq=pages)
    cache.page_table.copy_(torch.randperm(batch * pages, generator=gen).view(batch, pages).to(torch.int32))
    lens = (torch.rand(batch, generator=gen) * (context + 1)).int()
    lens[::7] = 0
    new = [torch.randn(batch, 1, context, 32, generator=gen).to(DEV) for _ in range(2)]
    zero = torch.zeros(batch, dtype=torch.int32, device=DEV)
    spa.kv_append_int4(cache.k, cache.v, cache.page_table, *new, zero, new_lens=lens.to(DEV))
    q = torch.randn(batch, 2, 32, generator=gen)
    w = torch.zeros(batch, 1, context, device=DEV)
    k, v = (x.double() for x in spa.kv_read_int4(cache.k, cache.v, cache.page_table, zero, context, dtype=torch.float32))
    args = dict(page_table=cache.page_table, context_lens=lens.to(DEV))
    plain = spa.paged_decode_attention_int4(q.to(DEV), cache.k, cache.v, **args)
    out = spa.paged_decode_attention_int4(q.to(DEV), cache.k, cache.v, weights=w, **args)
    there = (torch.arange(context) < lens[:, None]).to(DEV)[:, None]
    score = (q.to(DEV).double() @ k[:, 0].transpose(1, 2)) / 32 ** 0.5
    p = torch.nan_to_num(torch.softmax(torch.where(there, score, -torch.inf), -1))
    want = p @ v[:, 0]
    # |q| <= 5 and |k| <= 5 of 32 values: Q <= 5 * 15 * 32 / 32 ** 0.5 < 2^9 (|s n| + |z| <= 15); D + 8 = 40
    rel = 2 * 40 * 2.0 ** -24 * 2 ** 9 + context * 2.0 ** -24 + 2.0 ** -20
    for o in (plain, out):
        assert ((o.double() - want).abs() <= rel * 15).all() and (o[lens == 0] == 0).all()
    assert ((w[:, 0].double() - p.sum(1)).abs() <= rel * p.sum(1)).all()


# ---------------------------------------------------------------- refusals
def test_refusals():
    cache = spa.PagedKVCacheInt4(2, 2, 4, 64, batch=1, max_pages_per_seq=2)
    k, v, t = cache.k, cache.v, cache.page_table
    lens, q = cache.context_lens, torch.zeros(1, 4, 64, device=DEV)
    ok = dict(page_table=t, context_lens=lens)
    dec = spa.paged_decode_attention_int4
    with pytest.raises(ValueError, match="pair"):
        dec(q, k[0][:, :, :, :0], v, **ok)
    with pytest.raises(ValueError, match="uint8 codes"):
        dec(q, (k[0].float(), k[1]), v, **ok)
    with pytest.raises(ValueError, match="scales must be"):
        dec(q, (k[0], k[1][..., :1].contiguous()), v, **ok)
    with pytest.raises(ValueError, match="contiguous"):
        dec(q, (k[0].transpose(1, 2).contiguous().transpose(1, 2), k[1]), v, **ok)
    with pytest.raises(ValueError, match="incompatible"):
        dec(torch.zeros(1, 3, 64, device=DEV), k, v, **ok)
    with pytest.raises(ValueError, match="incompatible"):
        dec(torch.zeros(1, 4, 32, device=DEV), k, v, **ok)
    with pytest.raises(ValueError, match="dtype"):
        dec(q.double(), k, v, **ok)
    with pytest.raises(ValueError, match="CUDA tensors"):
        dec(q.cpu(), k, v, **ok)
    with pytest.raises(ValueError, match="context_lens"):
        dec(q, k, v, page_table=t, context_lens=torch.zeros(2, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="weights"):
        dec(q, k, v, weights=torch.zeros(1, 4, 8, device=DEV), **ok)
    with pytest.raises(ValueError, match="weights"):
        dec(q, k, v, weights=torch.zeros(1, 2, 8, device=DEV, dtype=torch.float16), **ok)
    with pytest.raises(ValueError, match="page layout"):
        spa.paged_gather_decode_attention_int4(q, k, v, torch.zeros(1, 1, dtype=torch.int64, device=DEV),
                                               local_window=0, block_size=8, **ok)
    x = torch.zeros(1, 2, 64, device=DEV)
    with pytest.raises(ValueError, match="k_new"):
        spa.kv_append_int4(k, v, t, x[:, :1], x[:, :1], lens)
    with pytest.raises(ValueError, match="positions"):
        spa.kv_append_int4(k, v, t, x, x, torch.zeros(2, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="dtype"):
        spa.kv_append_int4(k, v, t, x.double(), x.double(), lens)
    spa.kv_append_int4(k, v, t, x[:, :, None][:, :, :0], x[:, :, None][:, :, :0], lens)  # no tokens: nothing to do
    assert spa.kv_read_int4(k, v, t, lens, 0)[0].shape == (1, 2, 0, 64)
