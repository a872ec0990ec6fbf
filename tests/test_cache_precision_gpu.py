"""Decode over a small cache against the limits of cache_precision.py, as root mean squares over all
outputs: tighter by orders of magnitude than the bounds that hold for each output alone."""

import pytest
import torch

import attention_b200 as spa
import oracle.small_cache as ref
from cache_precision import attention, int4_parts, output_limit, rms, terms, weight_limit

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    assert spa.device_error_flags() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,heads", [(32, (8, 2)), (64, (8, 2)), (64, (64, 1)), (96, (20, 2)), (128, (8, 2)),
                                       (128, (24, 2)), (192, (8, 2)), (256, (8, 2))])
@pytest.mark.parametrize("n", [300, 3000])
def test_int4(dtype, dim, heads, n):
    gen = torch.Generator().manual_seed(dim + n)
    page, batch = 16, 2
    pages = -(-n // page)
    q = torch.randn(batch, heads[0], dim, generator=gen).to(dtype)
    quant = [ref.int4_quantise(torch.randn(batch, heads[1], pages * page, dim, generator=gen)) for _ in range(2)]
    table = torch.randperm(batch * pages, generator=gen).view(batch, pages).to(torch.int32)

    def pool(x):
        out = torch.empty(batch * pages, heads[1], page, *x.shape[3:], dtype=x.dtype)
        out[table.flatten().long()] = x.unflatten(2, (pages, page)).transpose(1, 2).flatten(0, 1)
        return out.to(DEV)

    pools = [tuple(pool(t) for t in x) for x in quant]
    quant = [tuple(t[:, :, :n] for t in x) for x in quant]
    k, v = (ref.int4_dequantise(x) for x in quant)
    want, want_w = attention(q, k, v, torch.float64)
    plain, plain_w = attention(q, k, v, torch.float32)
    w = torch.zeros(batch, heads[1], n, device=DEV)
    more = dict(page_table=table.to(DEV), context_lens=torch.full((batch,), n, device=DEV))
    size = terms(q, k, int4_parts(v, quant[1][1])[0])
    for weights in (None, w):
        out = spa.paged_decode_attention_int4(q.to(DEV), *pools, weights=weights, **more)
        err, limit = rms(out.double().cpu() - want), output_limit(dtype, want, plain, size)
        assert err <= limit, (err, limit)
    err = rms(w.double().cpu() / want_w - 1)
    limit = weight_limit(dtype, want_w, plain_w, q, int4_parts(k, quant[0][1])[1])
    assert err <= limit, (err, limit)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,heads", [(32, (8, 2)), (64, (64, 1)), (96, (20, 2)), (128, (8, 2)), (256, (8, 2))])
@pytest.mark.parametrize("n", [300, 3000])
def test_plain_with_weights(dtype, dim, heads, n):
    gen = torch.Generator().manual_seed(dim + n)
    q = torch.randn(2, heads[0], dim, generator=gen).to(dtype)
    k, v = (torch.randn(2, heads[1], n, dim, generator=gen).to(dtype) for _ in range(2))
    want, want_w = attention(q, k, v, torch.float64)
    plain, plain_w = attention(q, k, v, torch.float32)
    w = torch.zeros(2, heads[1], n, device=DEV)
    out = spa.paged_decode_attention(q.to(DEV), k.to(DEV), v.to(DEV), weights=w)
    err, limit = rms(out.double().cpu() - want), output_limit(dtype, want, plain, terms(q, k, v.abs()))
    assert err <= limit, (err, limit)
    err, limit = rms(w.double().cpu() / want_w - 1), weight_limit(dtype, want_w, plain_w, q)
    assert err <= limit, (err, limit)
