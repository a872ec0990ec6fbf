"""4-bit decode where a group's zero, not its scale, is near fp16's largest value: the middle of the
group, zero + 8 scales, lies past it.  Tolerances are those of test_int4_gpu.py."""

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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,heads", [(32, 4), (64, 4), (96, 20), (128, 4), (256, 4)])
@pytest.mark.parametrize("which", ["k", "v", "v late"])
def test_decode_zeros_near_fp16s_largest(dtype, dim, heads, which):
    """Values of 60000 to 80000 in one group of every token, or of the last ten, of K or of V."""
    gen = torch.Generator().manual_seed(dim)
    k, v, table, _, _, _ = make_cache(1, 2, 16, dim, 400, gen)
    x = torch.randn(2, 1, 2, 400, dim, generator=gen)
    large = 6e4 + 2e4 * torch.rand(1, 2, 400, 32, generator=gen)
    if which == "v late":
        x[1, :, :, 390:, -32:] = large[:, :, 390:]
    else:
        x[0 if which == "k" else 1, ..., -32:] = large
    full = [ref.int4_quantise(y) for y in x]
    for pool, (codes, scales) in zip((k, v), full):
        for g in range(25):
            pool[0][table[0, g]] = codes[0, :, g * 16:(g + 1) * 16]
            pool[1][table[0, g]] = scales[0, :, g * 16:(g + 1) * 16]
    kval, vval = (ref.int4_dequantise(f) for f in full)
    q = torch.randn(1, heads, dim, generator=gen)
    if which == "k":
        q[..., -32:] /= 1e5
    q = q.to(dtype)
    tokens = [torch.arange(400)]
    w = torch.zeros(1, 2, 400, device=DEV)
    more = dict(page_table=table.to(DEV), context_lens=torch.tensor([400], device=DEV))
    out = spa.paged_decode_attention_int4(q.to(DEV), to_dev(k), to_dev(v), weights=w, **more)
    want, ww = ref.attention_weights(q, kval, vval, tokens)
    # the bound is that of every term; heads' outputs differ in size by group, so per group
    rel, _ = bounds(q, full[0], kval, vval, tokens, dtype)
    for j in range(dim // 32):
        part = slice(32 * j, 32 * j + 32)
        tol = (rel + (0 if dtype == torch.float32 else 2.0 ** -10)) * 3 * vval[..., part].abs().max().item()
        check_out(out[..., part], want[..., part], tol, dtype)
    assert ((w.double().cpu() - ww).abs() <= rel * ww).all()
