"""Decode over a page table with much more room than the contexts fill, as a serving loop has it:
the CTAs are planned from the room, the work from the lengths.  Workspaces are handed out full
of NaN, so that a partial result which no CTA wrote shows.

Tolerance: that of tests/test_int4_gpu.py and tests/test_eviction_gpu.py.  With Q = max_t
sum_d |q_d k_d| / sqrt(D) a probability is off by a relative 2 (D + 8) 2^-24 Q + N 2^-24 + 2^-20;
16-bit queries over 4 bits add two fp16 roundings of each probability, 2^-10, and over 16 bits
probabilities in two bf16 halves, 2^-16; the output adds its own half step.  Terms |s n| + |z|
of a 4-bit value are at most 3 times the largest value."""

import pytest
import torch

import attention_b200 as spa
import oracle.small_cache as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
HEADS, GROUP, PAGE = 4, 2, 32


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    assert spa.device_error_flags() == 0


@pytest.fixture
def nan_workspaces(monkeypatch):
    plain = torch.empty

    def empty(*size, **kw):
        t = plain(*size, **kw)
        return t.fill_(255) if t.dtype == torch.uint8 and t.is_cuda else t

    monkeypatch.setattr(torch, "empty", empty)


class Roomy:
    """K and V of `lens` tokens a sequence, in scattered pages of a table of `room` tokens whose
    entries behind the sequence are -1.  kind: "int4" or a plain cache in the queries' dtype."""

    def __init__(self, kind, dtype, dim, lens, room, gen):
        self.dtype, self.lens, self.room, most = dtype, lens, room, max(lens)
        pages = -(-most // PAGE)
        n = len(lens) * pages
        shape = (len(lens), HEADS, pages * PAGE, dim)
        full = [torch.randn(shape, generator=gen) for _ in range(2)]
        table = torch.randperm(n, generator=gen).view(len(lens), pages).to(torch.int32)
        self.table = torch.full((len(lens), -(-room // PAGE)), -1, dtype=torch.int32)
        for b, length in enumerate(lens):
            used = -(-length // PAGE)
            self.table[b, :used] = table[b, :used]

        def pool(x):  # [B, H, tokens, ...] to [pages, H, P, ...]
            out = torch.empty(n, HEADS, PAGE, *x.shape[3:], dtype=x.dtype)
            out[table.flatten().long()] = x.unflatten(2, (pages, PAGE)).transpose(1, 2).flatten(0, 1)
            return out.to(DEV)

        if kind == "int4":
            quant = [ref.int4_quantise(x) for x in full]
            self.pools = [tuple(pool(t) for t in q) for q in quant]
            self.values = [ref.int4_dequantise(q) for q in quant]
        else:
            full = [x.to(dtype) for x in full]
            self.pools = [pool(x) for x in full]
            self.values = [x.double() for x in full]
        self.q = torch.randn(len(lens), HEADS * GROUP, dim, generator=gen).to(dtype)
        self.call = spa.paged_decode_attention_int4 if kind == "int4" else spa.paged_decode_attention
        self.kind = kind

    def check(self, window, weights):
        w0 = torch.rand(len(self.lens), HEADS, self.room, generator=torch.Generator().manual_seed(1))
        w = w0.to(DEV) if weights else None
        more = dict(weights=w) if weights else {}
        out = self.call(self.q.to(DEV), *self.pools, page_table=self.table.to(DEV),
                        context_lens=torch.tensor(self.lens, device=DEV), local_window=window, **more)
        tokens = [torch.arange(max(0, n - window) if window else 0, n) for n in self.lens]
        want, ww = ref.attention_weights(self.q, *self.values, tokens)
        k, v = self.values
        dim = k.size(3)
        q_size = (self.q.double().abs() @ k.abs().flatten(0, 2).amax(0)).max() / dim ** 0.5
        if self.kind == "int4":
            q_size *= 3
        rel = 2 * (dim + 8) * 2.0 ** -24 * q_size + max(self.lens) * 2.0 ** -24 + 2.0 ** -20
        half = 0.0 if self.dtype == torch.float32 else 2.0 ** -10 if self.kind == "int4" else 2.0 ** -16
        tol = (rel + half) * v.abs().max() * (3 if self.kind == "int4" else 1)
        err = (out.double().cpu() - want).abs()
        assert (err <= tol + torch.finfo(self.dtype).eps / 2 * want.abs()).all(), (err.max().item(), tol.item())
        if weights:
            got = w.double().cpu()
            total = torch.nn.functional.pad(ww, (0, max(0, self.room - ww.size(2))))[..., : self.room] + w0.double()
            assert ((got - total).abs() <= rel * (total - w0) + 2.0 ** -23 * total).all()


KERNELS = [("int4", torch.bfloat16, 128), ("int4", torch.float16, 64), ("int4", torch.float32, 128),
           ("int4", torch.bfloat16, 256), ("int4", torch.float16, 160), ("plain", torch.bfloat16, 128),
           ("plain", torch.float16, 64), ("plain", torch.bfloat16, 96), ("plain", torch.float32, 64)]
# rooms that are split over CTAs, with fewer tiles, as many and more than the CTAs of the room
LENGTHS = [[1], [33], [50], [400], [1000], [1700], [50, 1, 0, 700], [0, 40], [1700, 3, 300, 33, 5, 0, 64, 1000]]


@pytest.mark.parametrize("room", [4096, 131072])
@pytest.mark.parametrize("kind,dtype,dim", KERNELS)
def test_short_contexts_in_a_long_table(nan_workspaces, kind, dtype, dim, room):
    gen = torch.Generator().manual_seed(dim + room)
    for lens in LENGTHS:
        cache = Roomy(kind, dtype, dim, lens, room, gen)
        for weights in ((False, True) if kind == "int4" else (True,)):
            for window in (0, 900):
                cache.check(window, weights)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float32, 64), (torch.float16, 160)])
def test_long_window_over_a_short_context(nan_workspaces, dtype, dim):
    """The gather's plan counts the window it may have, not the tokens that are there."""
    gen = torch.Generator().manual_seed(dim)
    for lens in ([40], [700], [33, 400, 0]):
        cache = Roomy("int4", dtype, dim, lens, 65536, gen)
        sel = torch.tensor([[0, -1]] * len(lens))
        sel[torch.tensor(lens) == 0] = -1
        out = spa.paged_gather_decode_attention_int4(cache.q.to(DEV), *cache.pools, sel.to(DEV), local_window=16384,
                                                     block_size=PAGE, page_table=cache.table.to(DEV),
                                                     context_lens=torch.tensor(lens, device=DEV))
        tokens = [torch.cat((torch.arange(n), torch.arange(min(n, PAGE)))) for n in lens]
        want, _ = ref.attention_weights(cache.q, *cache.values, tokens)
        # as in Roomy.check: Q < 2^7 for these sizes, D + 8 <= 168
        tol = (2 * 168 * 2.0 ** -24 * 2 ** 7 + 2.0 ** -10) * 3 * cache.values[1].abs().max()
        assert ((out.double().cpu() - want).abs() <= tol + torch.finfo(dtype).eps / 2 * want.abs()).all()


@pytest.mark.parametrize("kind", ["int4", "bf16"])
def test_serving_loop_grows_into_its_room(nan_workspaces, kind):
    """A prompt of 20 tokens in a table of 2048, prompts appended turn by turn, a step with weights after each,
    and an eviction: every output against a 64-bit model."""
    gen = torch.Generator().manual_seed(3)
    batch, dim, room, budget, recent = 2, 64, 2048, 300, 40
    dt = torch.bfloat16
    pages = room // PAGE
    make = spa.PagedKVCacheInt4 if kind == "int4" else spa.PagedKVCache
    cache = make(batch * pages, HEADS, PAGE, dim, batch=batch, max_pages_per_seq=pages)
    cache.page_table.copy_(torch.randperm(batch * pages, generator=gen).view(batch, pages).to(torch.int32))
    stored = (lambda x: ref.int4_dequantise(ref.int4_quantise(x))) if kind == "int4" else (lambda x: x.double())
    decode = spa.paged_decode_attention_int4 if kind == "int4" else spa.paged_decode_attention
    w = torch.zeros(batch, HEADS, room, device=DEV)
    model = [torch.zeros(batch, HEADS, 0, dim, dtype=torch.float64) for _ in range(2)]
    acc = torch.zeros(batch, HEADS, 0, dtype=torch.float64)
    for turn in (20, 1, 70, 400, 1, 200, 30):
        new = [torch.randn(batch, HEADS, turn, dim, generator=gen).to(dt) for _ in range(2)]
        if kind == "int4":
            spa.kv_append_int4(cache.k, cache.v, cache.page_table, *(x.to(DEV) for x in new), cache.context_lens)
        else:
            for t in range(turn):
                spa.kv_append(cache.k, cache.v, cache.page_table, *(x[:, :, t].to(DEV) for x in new),
                              cache.context_lens + t)
        cache.context_lens += turn
        model = [torch.cat((m, stored(x)), 2) for m, x in zip(model, new)]
        q = torch.randn(batch, HEADS * GROUP, dim, generator=gen).to(dt)
        out = decode(q.to(DEV), cache.k, cache.v, page_table=cache.page_table, context_lens=cache.context_lens, weights=w)
        n = model[0].size(2)
        want, ww = ref.attention_weights(q, *model, [torch.arange(n)] * batch)
        acc = torch.nn.functional.pad(acc, (0, turn)) + ww
        # scores of these sizes are off by under 2^-12, P by 2^-10, the output by half a bf16 step
        assert ((out.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -9 * model[1].abs().max() * 3).all()
        got = w.double().cpu()
        assert ((got[..., :n] - acc).abs() <= 2.0 ** -11 * acc).all() and (got[..., n:] == 0).all()
        if n > 600:
            keep = spa.evict_tokens(cache, w, budget=budget, recent=recent).cpu().long()
            assert torch.equal(keep.int(), ref.select_tokens(got.float(), [n] * batch, budget, recent)[0])
            model = [m.gather(2, keep[..., None].expand(-1, -1, -1, dim)) for m in model]
            acc = acc.gather(2, keep)
