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


@pytest.mark.parametrize('dtype', [bf16, torch.float16, f32])
@pytest.mark.parametrize('residual', [False, True])
@pytest.mark.parametrize('H', [5, 64, 264, 1000, 2050, 7168, 20001, 32768])
def test_constant_rows(dev, H, residual, dtype):
    """The mean of a constant row is its value, whatever 1 / H rounds to: y = b, and nothing for the weight's gradient."""
    g = torch.Generator().manual_seed(H)
    values = torch.tensor([0.1, 3.0, -1000.1, 60000.0] + ([] if dtype == torch.float16 else [1e5, -1.2345e9, 7e25]))
    x = values[:, None].expand(-1, H).to(dtype).contiguous()
    res = (torch.zeros_like(x) if residual else None)
    w, b = (1 + 0.2 * torch.randn(H, generator=g)).to(dtype), torch.randn(H, generator=g).to(dtype)
    leaves = [t.to(dev).requires_grad_() for t in (x, w, b)]
    y = layer_norm(*leaves, 1e-5, None if res is None else res.to(dev))
    y = y[0] if residual else y
    assert torch.equal(y.detach().cpu(), b.expand_as(x))
    _, dw, _ = torch.autograd.grad([y], leaves, [torch.randn(x.shape, generator=g).to(dtype).to(dev)])
    assert float(dw.abs().max()) == 0.0


@pytest.mark.parametrize('H', [264, 1000, 7168])
@pytest.mark.parametrize('far', [100.0, 1e4, 1e6])
def test_rows_far_from_zero(dev, H, far):
    """The mean is corrected by that of h - mean, so what it is off by is its own rounding, 2^-24 of it, and 60 2^-24 of the mean |h - m|; the squares' mean is off by the square of that and 64 roundings
    (56 of the sum and the correction's), the root by half."""
    g = torch.Generator().manual_seed(H)
    x = far + torch.randn(9, H, generator=g)
    w, b = torch.ones(H), torch.zeros(H)
    h = x.double()
    d = h - h.mean(1, keepdim=True)
    r = 1 / (d.square().mean(1, keepdim=True) + 1e-5).sqrt()
    off = 2.0**-24 * h.mean(1, keepdim=True).abs() + 60 * 2.0**-24 * d.abs().mean(1, keepdim=True)
    bound = r * (off + 2.0**-24 * d.abs()) + (d * r).abs() * ((off * r)**2 / 2 + 40 * 2.0**-24)
    inside(layer_norm(*(t.to(dev) for t in (x, w, b))), d * r, bound, f'{far}')
