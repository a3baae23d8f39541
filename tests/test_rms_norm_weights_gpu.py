"""Norm weights in 32 bits under 16-bit rows: gradients and quantiser, with the tolerances of tests/test_rms_norm_gpu.py (40 and 64 units of
2^-24; dw is held in the weight's own type)."""
import pytest
import torch

from dlblas_amd.kernels.rms_norm import rms_norm, rms_norm_quant
from oracle import decoder as orc

pytestmark = pytest.mark.gpu
bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32
FP32 = 2.0**-24


@pytest.fixture(scope='module')
def dev():
    return torch.device('cuda:0')


def inputs(rows, H, dtype, dev):
    g = torch.Generator().manual_seed(rows + H)
    x, res, dy, dsum = (torch.randn(rows, H, generator=g).to(dtype) for _ in range(4))
    return x, 1 + 0.2 * torch.randn(H, generator=g), res, dy, dsum


@pytest.mark.parametrize('dtype', [bf16, f16])
@pytest.mark.parametrize('rows,H', [(3, 8), (2, 9), (700, 128), (33, 776), (5, 2050), (600, 7168), (2, 20001)])
def test_gradients(dev, rows, H, dtype):
    x, w, res, dy, dsum = inputs(rows, H, dtype, dev)
    leaves = [t.to(dev).requires_grad_() for t in (x, w, res)]
    got = torch.autograd.grad(rms_norm(leaves[0], leaves[1], 1e-5, leaves[2]), leaves, [dy.to(dev), dsum.to(dev)])
    assert got[1].dtype == f32
    dx, dw, mag, dw_mag = orc.rms_norm_grad(dy, dsum, orc.norm_input(x, res), w, 1e-5)
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    for t in (got[0], got[2]):
        assert float(((t.cpu().double() - dx).abs() - (half * dx.abs() + 64 * FP32 * mag + tiny)).max()) <= 0
    # at most rows / 512 terms a share, then at most 128 additions, 60 for the factors: as for weights of the rows' type
    assert float(((got[1].cpu().double() - dw).abs() - (FP32 * dw.abs() + (-(-rows // 512) + 128 + 60) * FP32 * dw_mag)).max()) <= 0


@pytest.mark.parametrize('dtype', [bf16, f16])
@pytest.mark.parametrize('rows,H', [(1, 128), (40, 256), (17, 1152), (64, 7168)])
def test_quantiser(dev, rows, H, dtype):
    x, w, res, _, _ = inputs(rows, H, dtype, dev)
    q, s, h = rms_norm_quant(x.to(dev), w.to(dev), 1e-5, res.to(dev))
    assert torch.equal(h.cpu(), orc.norm_input(x, res))
    ref_s, v = orc.quant_1x128(orc.rms_norm(h.cpu(), w, 1e-5))
    assert float(((s.cpu().double() - ref_s).abs() / ref_s).max()) <= 42 * FP32
    half = (v.abs() * 2.0**-4).clamp_min(2.0**-10)
    assert float(((q.cpu().double() - v).abs() - half - 90 * FP32 * v.abs()).max()) <= 0
    # 448 h w carries two roundings of fp32 here (h w, and times 448), the largest one: beside a quotient within 2^-21 of the middle of two
    # codes nothing may differ
    hw = (h.cpu().double() * w.double()).reshape(rows, -1, 128)
    u = hw * 448.0 / hw.abs().amax(-1, keepdim=True)
    low, high = ((u * (1 + k * 2.0**-21)).float().to(torch.float8_e4m3fn).reshape(rows, H).float() for k in (-1, 1))
    exact = u.float().to(torch.float8_e4m3fn).reshape(rows, H).float()
    assert bool(((q.cpu().float() == exact) | (low != high)).all())
