"""In-place compaction where it is tightest: lists whose sources are other CTAs' destinations,
at every number of chunks around which the kernel's row tables turn over.  Results are exact."""

import pytest
import torch

import attention_b200 as spa

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    assert spa.device_error_flags() == 0


def lists(batch, heads, budget, tokens, gen):
    """Keep lists [batch, heads, budget]: the first head moves every row down by one, the second by
    three, the others keep a random choice."""
    keep = torch.empty(batch, heads, budget, dtype=torch.int32, device=DEV)
    for b in range(batch):
        for h in range(heads):
            keep[b, h] = torch.randperm(tokens, generator=gen, device=DEV)[:budget].sort().values.int()
    step = torch.arange(budget, device=DEV, dtype=torch.int32)
    keep[:, 0] = step + 1
    if heads > 1:
        keep[:, 1] = step + 3
    return keep


def moved(pool, table, keep):
    page, out = pool.size(2), pool.clone()
    b, h, j = torch.meshgrid(*(torch.arange(n, device=DEV) for n in keep.shape), indexing="ij")
    t, table = keep.long(), table.long()
    out[table[b, j // page], h, j % page] = pool[table[b, t // page], h, t % page]
    return out


# 128-byte rows: 128 a chunk of a CTA, clusters of 8, so 1024 rows a chunk of a cluster
@pytest.mark.parametrize("chunks", [1, 2, 3, 4, 5, 6, 10])
def test_rows_that_others_overwrite(chunks):
    gen = torch.Generator(device=DEV).manual_seed(chunks)
    batch, heads, page, dim = 1, 3, 64, 64
    budget = 1024 * chunks - 5
    tokens = budget + 300
    pages = -(-tokens // page)
    for _ in range(8):
        table = torch.randperm(batch * pages, generator=gen, device=DEV).view(batch, pages).int()
        pools = [torch.randint(-2 ** 15, 2 ** 15, (batch * pages, heads, page, dim), generator=gen, device=DEV,
                               dtype=torch.int16).view(torch.bfloat16) for _ in range(2)]
        keep = lists(batch, heads, budget, tokens, gen)
        want = [moved(p.view(torch.int16), table, keep) for p in pools]
        spa.compact_tokens(pools, table, keep)
        for p, x in zip(pools, want):
            assert torch.equal(p.view(torch.int16), x)


@pytest.mark.parametrize("row", [1, 6, 20, 64, 256, 400, 2048])
def test_rows_of_every_unit(row):
    """Rows moved in units of 1, 2, 4 and 16 bytes, few and many to a chunk."""
    gen = torch.Generator(device=DEV).manual_seed(row)
    batch, heads, page, budget = 2, 3, 16, 1500
    pages = -(-(budget + 200) // page)
    table = torch.randperm(batch * pages, generator=gen, device=DEV).view(batch, pages).int()
    pool = torch.randint(0, 256, (batch * pages, heads, page, row), generator=gen, device=DEV, dtype=torch.uint8)
    keep = lists(batch, heads, budget, budget + 200, gen)
    want = moved(pool, table, keep)
    spa.compact_tokens((pool,), table, keep)
    assert torch.equal(pool, want)


# of 128 bytes (128 rows a chunk of a CTA) or 256 (64): 2, 6 and 10 chunks end on the table that the
# weights' rows go into first
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("chunks", [1, 2, 4, 6, 10])
def test_weights_follow_the_rows(dim, chunks):
    gen = torch.Generator(device=DEV).manual_seed(chunks)
    batch, heads, page = 2, 4, 32
    budget = 8 * (8192 // dim) * chunks - 3
    tokens = budget + 500
    pages = -(-tokens // page)
    for _ in range(8):
        table = torch.randperm(batch * pages, generator=gen, device=DEV).view(batch, pages).int()
        pools = [torch.randint(-2 ** 15, 2 ** 15, (batch * pages, heads, page, dim), generator=gen, device=DEV,
                               dtype=torch.int16).view(torch.bfloat16) for _ in range(2)]
        w = torch.rand(batch, heads, tokens, generator=gen, device=DEV)
        keep = lists(batch, heads, budget, tokens, gen)
        want = [moved(p.view(torch.int16), table, keep) for p in pools]
        want_w = torch.zeros_like(w)
        want_w[..., :budget] = w.gather(2, keep.long())
        spa.compact_tokens(pools, table, keep, weights=w)
        for p, x in zip(pools, want):
            assert torch.equal(p.view(torch.int16), x)
        assert torch.equal(w, want_w)


def test_lists_of_unlike_lengths():
    """Empty lists among long ones, with weights: their clusters have no chunk at all."""
    gen = torch.Generator(device=DEV).manual_seed(0)
    batch, heads, page, dim, budget, tokens = 3, 4, 16, 64, 2048, 2500
    pages = -(-tokens // page)
    table = torch.randperm(batch * pages, generator=gen, device=DEV).view(batch, pages).int()
    pool = torch.randint(0, 256, (batch * pages, heads, page, dim), generator=gen, device=DEV, dtype=torch.uint8)
    w = torch.rand(batch, heads, tokens, generator=gen, device=DEV)
    keep = lists(batch, heads, budget, tokens, gen)
    for b, h, n in ((0, 0, 0), (0, 1, 1), (1, 0, 1024), (1, 2, 0), (2, 3, 1025)):
        keep[b, h, n:] = -1
    to = torch.arange(budget, device=DEV, dtype=torch.int32)
    want = moved(pool, table, torch.where(keep >= 0, keep, to))
    want_w = torch.zeros_like(w)
    want_w[..., :budget] = torch.where(keep >= 0, w.gather(2, keep.long().clamp(min=0)), 0.0)
    spa.compact_tokens((pool,), table, keep, weights=w)
    assert torch.equal(pool, want) and torch.equal(w, want_w)


def test_pages_of_one_token():
    """A pool [pages, Hkv, 1, D] made by a transposition is contiguous with any stride for its third
    dimension: the rows' size comes from the shape."""
    gen = torch.Generator(device=DEV).manual_seed(1)
    batch, heads, dim, tokens, budget = 2, 3, 24, 90, 40
    table = torch.randperm(batch * tokens, generator=gen, device=DEV).view(batch, tokens).int()
    pool = torch.randn(batch * tokens, 1, heads, dim, generator=gen, device=DEV).transpose(1, 2)
    assert pool.is_contiguous() and pool.stride(2) != dim
    keep = lists(batch, heads, budget, tokens, gen)
    want = moved(pool, table, keep)
    spa.compact_tokens((pool,), table, keep)
    assert torch.equal(pool, want)
