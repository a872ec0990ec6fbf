"""The limits of cache_precision.py let a plain fp32 evaluation pass and a planted loss of bits fail."""

import pytest
import torch

import oracle.small_cache as ref
from cache_precision import attention, int4_parts, output_limit, rms, terms, weight_limit


@pytest.mark.parametrize("n,dim", [(300, 64), (3000, 128)])
def test_limits_see_a_loss_of_bits(n, dim):
    gen = torch.Generator().manual_seed(n)
    q = torch.randn(2, 8, dim, generator=gen)
    quant = [ref.int4_quantise(torch.randn(2, 2, n, dim, generator=gen)) for _ in range(2)]
    k, v = (ref.int4_dequantise(x) for x in quant)
    want, want_w = attention(q, k, v, torch.float64)
    plain, plain_w = attention(q, k, v, torch.float32)
    size = terms(q, k, int4_parts(v, quant[1][1])[0])
    limit = output_limit(torch.float32, want, plain, size)
    assert rms(plain.double() - want) < limit / 3
    for bits, seen in ((22, False), (16, True), (11, True)):
        lost, lost_w = attention(q, k, v, torch.float64, p_bits=bits)
        assert (rms(lost - want) > limit) == seen, bits
    limit_w = weight_limit(torch.float32, want_w, plain_w, q)
    assert rms(plain_w.double() / want_w - 1) < limit_w
    assert rms(attention(q, k, v, torch.float64, p_bits=14)[1] / want_w - 1) > limit_w
    for dtype in (torch.float16, torch.bfloat16):
        bits = -torch.finfo(dtype).eps
        assert rms((want * (1 + bits / 4)).to(dtype).double() - want) > output_limit(dtype, want, plain, size)
