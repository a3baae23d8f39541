"""Rows at the end of the range in which fp32 holds the sum of their squares, as the header states it."""
import pytest
import torch

from dlblas_amd.kernels.rms_norm import rms_norm, rms_norm_quant
from oracle import decoder as orc

pytestmark = pytest.mark.gpu
bf16, f32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize('dtype', [bf16, f32])
@pytest.mark.parametrize('H', [128, 1024, 7168])
def test_the_sum_of_squares_is_fp32(dtype, H):
    dev = torch.device('cuda:0')
    unit = 1 + torch.rand(2, H, generator=torch.Generator().manual_seed(H), dtype=torch.float64)
    below = (unit * (2.0**126 / unit.square().sum(1, keepdim=True)).sqrt()).to(dtype)  # a quarter of the range: bf16 rounds by 2^-8
    above = (unit * (2.0**130 / unit.square().sum(1, keepdim=True)).sqrt()).to(dtype)
    x, w = torch.cat([below, above]), torch.ones(H, dtype=dtype)
    y = rms_norm(x.to(dev), w.to(dev)).cpu()
    ref = orc.rms_norm(below, w, 1e-6)
    assert float(((y[:2].double() - ref).abs() - (torch.finfo(dtype).eps / 2 + 40 * 2.0**-24) * ref.abs()).max()) <= 0
    assert bool((y[2:] == 0).all())
    q, s = rms_norm_quant(x.to(dev), w.to(dev))
    ref_s = orc.quant_1x128(ref)[0]
    assert float(((s[:2].cpu().double() - ref_s).abs() / ref_s).max()) <= 42 * 2.0**-24 and bool((q[2:].float() == 0).all())
