"""Attention with the least scales that are taken, on the device: all weights are alike, whatever the units of the scores, so that outputs are means of the
values, finite where the values are. Means of equal values are those values, up to one rounding and what the weights' rounding leaves (2^-6 is far more)."""
import pytest
import torch

from oracle import attention
from test_attention_gpu import BF, DEV, HF, int32, randn
from test_shared_gpu import reference, setup

pytestmark = pytest.mark.gpu
SCALES = [1.2e-38, 5e-38, 1e-37, 4e-37, 3e-32, 1e-27]


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("dtype,size", [(BF, 3.0e38), (HF, 65504.0)])
@pytest.mark.parametrize("B,Hq,D", [(2, 4, 64), (40, 8, 128)])
def test_shared_of_values_as_large_as_the_type_has(capi, B, Hq, D, dtype, size, scale):
    gen = torch.Generator().manual_seed(9)
    prefix, lengths = 700, [(31 * b) % 100 for b in range(B)]
    cache, rows, table, pages = setup(gen, prefix, lengths, 1, D, 16, dtype, 16)
    values = torch.where(torch.isnan(rows[1]), rows[1], torch.full_like(rows[1], size)).to(dtype).to(DEV)
    q = randn(gen, B, Hq, D, dtype=dtype).to(DEV)
    out = capi.attn_shared(q, [cache[0], values], pages.to(DEV), prefix, table.to(DEV), int32(lengths), max(lengths), scale).cpu().double()
    assert torch.isfinite(out).all() and ((out - size).abs() <= 2.0 ** -6 * size).all()


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_shared_is_the_mean(capi, dtype, bits, scale):
    gen = torch.Generator().manual_seed(bits)
    prefix, lengths = 150, [100, 0, 700]
    cache, rows, table, pages = setup(gen, prefix, lengths, 2, 64, 16, dtype, bits)
    q = randn(gen, 3, 4, 64, dtype=dtype)
    out = capi.attn_shared(q.to(DEV), cache, pages.to(DEV), prefix, table.to(DEV), int32(lengths), 700, scale)
    ref, mag = reference(q, rows, pages, prefix, table, lengths, 16, scale)
    assert ((out.cpu().double() - ref).abs() <= attention.tolerance(ref, mag, dtype, True, prefix + 700)).all()


def test_shared_of_scores_as_large_as_a_float_holds(capi):
    """Scores of 2e38 and their negatives, which such a scale makes +- 2.4: no maximum overflows, and what weighs more does."""
    B, D, prefix = 2, 64, 128
    gen = torch.Generator().manual_seed(3)
    k, v = torch.zeros(10, 1, 16, D), randn(gen, 10, 1, 16, D, dtype=torch.float32)
    k[:8, 0, :, 0] = 2.0e38 * torch.where(torch.arange(128).view(8, 16) % 3 == 0, 1.0, -1.0)
    q = torch.zeros(B, 1, D)
    q[:, :, 0] = 1.0
    cache, q = [k.to(BF), v.to(BF)], q.to(BF)
    rows, pages, table = [c.double() for c in cache], torch.arange(8, dtype=torch.int32), torch.tensor([[8], [9]], dtype=torch.int32)
    out = capi.attn_shared(q.to(DEV), [c.to(DEV) for c in cache], pages.to(DEV), prefix, table.to(DEV), int32([5, 0]), 5, 1.2e-38).cpu().double()
    ref, mag = reference(q, rows, pages, prefix, table, [5, 0], 16, 1.2e-38)
    assert ((out - ref).abs() <= attention.tolerance(ref, mag, BF, True, 133)).all()


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("dtype,size", [(BF, 3.0e38), (HF, 65504.0)])
@pytest.mark.parametrize("n,Hq,D", [(300, 4, 64), (900, 8, 128), (200, 2, 256)])
def test_prompts_of_values_as_large_as_the_type_has(capi, n, Hq, D, dtype, size, scale):
    gen = torch.Generator().manual_seed(n)
    q, k = (randn(gen, n, h, D, dtype=dtype).to(DEV) for h in (Hq, 1))
    out = capi.attn_prompt(q, k, torch.full_like(k, size), int32([0, n]), int32([0, n]), scale).cpu().double()
    assert torch.isfinite(out).all() and ((out - size).abs() <= 2.0 ** -6 * size).all()


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_prompts_are_means(capi, dtype, scale):
    gen = torch.Generator().manual_seed(2)
    cu = [0, 1, 70, 200]
    q, k, v = (randn(gen, 200, h, 64, dtype=dtype) for h in (4, 2, 2))
    out = capi.attn_prompt(q.to(DEV), k.to(DEV), v.to(DEV), int32(cu), int32(cu), scale)
    ref, mag = attention.prompt(q, k, v, cu, cu, scale)
    assert ((out.cpu().double() - ref).abs() <= attention.tolerance(ref, mag, dtype, True, 130)).all()
