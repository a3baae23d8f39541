"""Rows at the end of the range of fp32: finite rows have a finite mean, and those whose sum of squares passes what fp32 holds give the bias, as the header states it."""
import pytest
import torch

from dlblas_amd.kernels.layer_norm import layer_norm
from oracle import layer_norm as orc

pytestmark = pytest.mark.gpu
bf16, f32 = torch.bfloat16, torch.float32


@pytest.fixture(scope='module')
def dev():
    return torch.device('cuda:0')


def inside(got, want, bound, what):
    step = torch.finfo(got.dtype).eps / 2
    off = (got.detach().cpu().double() - want).abs() - (bound * (1 + step) + step * want.abs() + torch.finfo(got.dtype).smallest_normal * step)
    assert float(off.max()) <= 0, f'{what}: {float(off.max()):.3e} beyond the bound'


@pytest.mark.parametrize('dtype', [bf16, f32])
@pytest.mark.parametrize('H', [5, 64, 1000, 1024, 7168, 20001])
def test_large_rows(dev, H, dtype):
    """Rows of numbers of both signs and of one sign: the squares' sum is 2^126 in two, far beyond fp32 in the others, where the bias is what is left.  What they add to the gradient of the
    weight is nothing, whatever their dy."""
    g = torch.Generator().manual_seed(H)
    unit = torch.randn(2, H, generator=g, dtype=torch.float64)
    spread = (unit - unit.mean(1, keepdim=True)).square().sum(1, keepdim=True).sqrt()
    below = unit * (2.0**63 / spread)
    one_sign = torch.rand(1, H, generator=g, dtype=torch.float64) + 1
    signs = torch.where(torch.arange(H) % 2 == 0, 1.0, -1.0)
    above = [one_sign * 1e30, one_sign * 1e36, one_sign * signs * 1e36, one_sign * 1.6e38, one_sign * signs * 1.6e38, torch.where(torch.arange(H) == 0, 3e38, -3e38)[None]]
    x = torch.cat([below] + above).to(dtype)
    w, b = (1 + 0.2 * torch.randn(H, generator=g)).to(dtype), torch.randn(H, generator=g).to(dtype)
    leaves = [t.to(dev).requires_grad_() for t in (x, w, b)]
    y = layer_norm(*leaves)
    assert torch.equal(layer_norm(*(t.detach() for t in leaves)), y)
    inside(y[:2], *orc.layer_norm(x[:2], w, b, 1e-5), 'below')
    assert torch.equal(y[2:].detach().cpu(), b.expand(len(x) - 2, H))
    dy = torch.randn(x.shape, generator=g).to(dtype)
    dx, dw, db = torch.autograd.grad([y], leaves, [dy.to(dev)])
    # of the rows above nothing: r is 0
    (_, want_w, _), (_, (n_off, dw_mag), _) = orc.layer_norm_grad(dy[:2], None, x[:2], w, 1e-5)
    inside(dw, want_w, n_off + 200 * orc.FP32 * dw_mag, 'dw')
    assert bool(dx.isfinite().all()) and float(dx[2:].abs().max()) == 0.0
    inside(db, dy.double().sum(0), 200 * orc.FP32 * dy.double().abs().sum(0), 'db')


def test_infinities_still_show(dev):
    x = torch.zeros(3, 1024)
    x[0, 5], x[1, 7], x[2] = float('inf'), float('-inf'), 3e38
    x[2, 9] = float('nan')
    w, b = torch.ones(1024), torch.zeros(1024)
    assert bool(layer_norm(*(t.to(dev) for t in (x, w, b))).isnan().all())
