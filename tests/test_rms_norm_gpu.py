"""RMS norm, its quantising form and its gradients against the definitions in 64 bits.

Tolerances, u = half a step of the stored type.  The sum of squares is added in fp32: at most 32 terms a lane, 6 steps over the wave, 16
waves, each rounding 2^-24 of a partial sum, and the root halves what the sum is off; with the division, the root and two
products of the result that is below 40 * 2^-24 of the value.  Gradients: 64 * 2^-24 of the magnitudes that go into them (their sums over
a row have the same number of additions); dw: a workgroup adds rows / 512 terms, a lane of the second kernel a quarter of 512 shares."""
import pytest
import torch

import dlblas_amd
from dlblas_amd.kernels import rms_norm as mod
from dlblas_amd.kernels.fp8 import per_token_group_quant_fp8
from dlblas_amd.kernels.rms_norm import rms_norm, rms_norm_quant
from oracle import decoder as orc

pytestmark = pytest.mark.gpu
bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32
FP32 = 2.0**-24


@pytest.fixture(scope='module')
def dev():
    return torch.device('cuda:0')


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """Half a step of the subnormal numbers of a type."""
    return torch.finfo(t).smallest_normal * half_step(t)


def inputs(rows, H, dtype, residual, w_dtype=None, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(1000 * rows + H + seed)
    x = (torch.randn(rows, H, generator=g) * scale).to(dtype)
    x[:, ::7] *= 8
    res = (torch.randn(rows, H, generator=g) * scale).to(dtype) if residual else None
    w = (1 + 0.2 * torch.randn(H, generator=g)).to(w_dtype or dtype)
    return x, w, res


def on(dev, *tensors):
    return [None if t is None else t.to(dev) for t in tensors]


def check_y(y, h, w, eps, what):
    ref = orc.rms_norm(h, w, eps)
    off = (y.cpu().double() - ref).abs() - ((half_step(y.dtype) + 40 * FP32) * ref.abs() + tiny(y.dtype))
    assert float(off.max()) <= 0, f'{what}: {float(off.max()):.3e} beyond the bound'


SHAPES = [(1, 1), (1, 7), (3, 8), (2, 9), (5, 64), (4, 127), (3, 513), (2, 1000), (300, 264), (7, 2050), (2, 4096), (1, 7168), (33, 7168), (2, 8199), (3, 16384), (2, 20001),
          (1, 32768)]


@pytest.mark.parametrize('dtype', [bf16, f16, f32])
@pytest.mark.parametrize('residual', [False, True])
@pytest.mark.parametrize('rows,H', SHAPES)
def test_norm(dev, rows, H, residual, dtype):
    x, w, res = inputs(rows, H, dtype, residual)
    xd, wd, rd = on(dev, x, w, res)
    out = rms_norm(xd, wd, 1e-5, rd)
    h = orc.norm_input(x, res)
    if residual:
        out, hd = out
        assert torch.equal(hd.cpu(), h)
    check_y(out, h, w, 1e-5, f'{rows}x{H} {dtype}')


@pytest.mark.parametrize('rows,H', [(1, 128), (3, 256), (17, 1152), (4, 7168), (2, 16384), (1, 32768)])
@pytest.mark.parametrize('residual', [False, True])
@pytest.mark.parametrize('dtype', [bf16, f16, f32])
@pytest.mark.parametrize('column_major', [False, True])
def test_norm_quant(dev, rows, H, residual, dtype, column_major):
    x, w, res = inputs(rows, H, dtype, residual)
    xd, wd, rd = on(dev, x, w, res)
    out = rms_norm_quant(xd, wd, 1e-5, rd, column_major_scales=column_major)
    q, s = out[:2]
    h = orc.norm_input(x, res)
    if residual:
        assert torch.equal(out[2].cpu(), h)
    assert q.dtype == torch.float8_e4m3fn and s.dtype == f32 and tuple(s.shape) == (rows, H // 128)
    assert s.stride() == ((1, rows) if column_major else (H // 128, 1)) or rows == 1 or H == 128
    y = orc.rms_norm(h, w, 1e-5)
    ref_s, v = orc.quant_1x128(y)
    assert float(((s.cpu().double() - ref_s).abs() / ref_s).max()) <= 42 * FP32
    # e4m3: half a step is 2^-4 of the value, 2^-10 below 2^-6; both operands of the quotient are off by the bounds above
    half = (v.abs() * 2.0**-4).clamp_min(2.0**-10)
    off = (q.cpu().double() - v).abs() - half - 90 * FP32 * v.abs()
    assert float(off.max()) <= 0


@pytest.mark.parametrize('dtype', [bf16, f16])
@pytest.mark.parametrize('rows,H', [(64, 7168), (5, 384)])
def test_codes_half_way_between_two_stay_there(dev, rows, H, dtype):
    """y / s = 448 h w / max |h w| does not depend on r.  bf16: both operands are exact in fp32 (8 + 8 + 3 bits), so the codes are those of
    the fp32 quotient, ties to even among them.  fp16: 448 h w takes up to 25 bits, a rounding of 2^-24, so beside a quotient that is
    within 2^-22 of the middle of two codes nothing may differ."""
    x, w, res = inputs(rows, H, dtype, True)
    q = rms_norm_quant(*on(dev, x, w), 1e-5, res.to(dev))[0].cpu()
    hw = (orc.norm_input(x, res).double() * w.double()).reshape(rows, -1, 128)
    v = hw * 448.0 / hw.abs().amax(-1, keepdim=True)
    low, high = ((v * (1 + k * 2.0**-22)).float().to(torch.float8_e4m3fn).reshape(rows, H).float() for k in (-1, 1))
    exact = v.float().to(torch.float8_e4m3fn).reshape(rows, H).float()
    assert torch.equal(q.float(), exact) if dtype == bf16 else bool(((q.float() == exact) | (low != high)).all())


@pytest.mark.parametrize('rows,H', [(1, 128), (9, 2048), (3, 7168)])
def test_fp32_rows_quantise_to_the_bits_of_the_two_steps(dev, rows, H):
    """y of fp32 rows is not rounded on its way to memory, so norm and quantiser apart are the same arithmetic."""
    x, w, res = on(dev, *inputs(rows, H, f32, True))
    y, h = rms_norm(x, w, 1e-6, res)
    q, s = per_token_group_quant_fp8(y, 128)
    q1, s1, h1 = rms_norm_quant(x, w, 1e-6, res)
    assert torch.equal(s, s1) and torch.equal(h, h1) and torch.equal(q.view(torch.uint8), q1.view(torch.uint8))


def test_weight_in_32_bits(dev):
    for dtype in (bf16, f16):
        x, w, res = inputs(6, 776, dtype, True, w_dtype=f32)
        y, h = rms_norm(*on(dev, x, w), 1e-6, *on(dev, res))
        check_y(y, h.cpu(), w, 1e-6, 'fp32 weight')


@pytest.mark.parametrize('dtype', [bf16, f32])
def test_rows_where_they_lie(dev, dtype):
    """Rows of a wider tensor, at any element offset, broadcast rows, transposed and three-dimensional inputs."""
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(6, 300, generator=g).to(dtype)
    w = torch.randn(130, generator=g).to(dtype)
    wd = wide.to(dev)
    for off in (0, 1, 2, 3, 5, 8):
        x, r = wide[:, off:off + 130], wide[:, off + 140:off + 270]
        y, h = rms_norm(wd[:, off:off + 130], w.to(dev), 1e-6, wd[:, off + 140:off + 270])
        assert torch.equal(h.cpu(), orc.norm_input(x, r))
        check_y(y, h.cpu(), w, 1e-6, f'offset {off}')
    row = wide[:1, :130]
    check_y(rms_norm(row.to(dev).expand(9, 130), w.to(dev)), row.expand(9, 130), w, 1e-6, 'broadcast')
    t = torch.randn(130, 4, generator=g).to(dtype)
    check_y(rms_norm(t.to(dev).t(), w.to(dev)), t.t(), w, 1e-6, 'transposed')
    cube = torch.randn(2, 3, 130, generator=g).to(dtype)
    y = rms_norm(cube.to(dev), w.to(dev))
    assert y.shape == cube.shape
    check_y(y, cube, w, 1e-6, 'three dimensions')
    vec = rms_norm(cube[0, 0].to(dev), w.to(dev))
    assert vec.shape == (130, ) and torch.equal(vec, y[0, 0])
    q, s = rms_norm_quant(cube[:, :, :128].to(dev), w[:128].to(dev), column_major_scales=True)
    assert tuple(s.shape) == (2, 3, 1) and q.shape == (2, 3, 128)
    q2, s2 = rms_norm_quant(cube[:, :, :128].to(dev), w[:128].to(dev))
    assert torch.equal(s, s2) and torch.equal(q.view(torch.uint8), q2.view(torch.uint8))


def test_no_rows(dev):
    w = torch.ones(256, device=dev, dtype=bf16, requires_grad=True)
    x = torch.empty(0, 256, device=dev, dtype=bf16)
    assert rms_norm(x, w.detach()).shape == (0, 256)
    q, s = rms_norm_quant(x, w.detach())
    assert q.shape == (0, 256) and s.shape == (0, 2)
    rms_norm(x, w).sum().backward()
    assert float(w.grad.float().abs().max()) == 0.0


def test_rows_of_zeros_and_values_that_are_no_numbers(dev):
    x = torch.zeros(4, 256, dtype=bf16)
    x[1, 3] = float('nan')
    x[2, 200] = float('inf')
    x[3] = 1.0
    w = torch.ones(256, dtype=bf16)
    y = rms_norm(x.to(dev), w.to(dev)).cpu()
    assert bool((y[0] == 0).all()) and bool(y[1].isnan().all()) and bool(y[2, 200].isnan())
    assert float((y[3].double() - (1 + 1e-6)**-0.5).abs().max()) <= 2.0**-8
    q, s = rms_norm_quant(x.to(dev), w.to(dev))
    back = (q.float().view(4, 2, 128) * s.view(4, 2, 1)).cpu()
    assert bool((back[0] == 0).all()) and bool(back[1].isnan().all()) and bool(back[2, 1, 72].isnan()) and bool((back[3] - 1).abs().max() < 0.04)
    assert float(s[0, 0]) == pytest.approx(1e-10 / 448, rel=1e-6)


@pytest.mark.parametrize('dtype', [bf16, f16, f32])
@pytest.mark.parametrize('residual', [False, True])
@pytest.mark.parametrize('rows,H', [(1, 1), (2, 9), (5, 64), (4, 127), (1100, 136), (600, 513), (7, 2050), (33, 7168), (2, 9000), (3, 20001),
                                    (17, 128), (9001, 64), (5003, 256), (8301, 520), (2, 8), (33, 248)])
def test_gradients(dev, rows, H, residual, dtype):
    x, w, res = inputs(rows, H, dtype, residual, seed=1)
    g = torch.Generator().manual_seed(rows + H)
    dy, dsum = (torch.randn(rows, H, generator=g).to(dtype) for _ in range(2))
    leaves = [t.to(dev).requires_grad_() for t in (x, w) + ((res, ) if residual else ())]
    out = rms_norm(leaves[0], leaves[1], 1e-5, leaves[2] if residual else None)
    if residual:
        got = torch.autograd.grad(out, leaves, on(dev, dy, dsum))
        check_y(out[0].detach(), out[1].detach().cpu(), w, 1e-5, 'with gradient')
    else:
        got = torch.autograd.grad([out], leaves, on(dev, dy))
    dx, dw, mag, dw_mag = orc.rms_norm_grad(dy, dsum if residual else None, orc.norm_input(x, res), w, 1e-5)
    for t in (got[0], ) + tuple(got[2:]):
        off = (t.cpu().double() - dx).abs() - (half_step(dtype) * dx.abs() + 64 * FP32 * mag + tiny(dtype))
        assert float(off.max()) <= 0, f'dx {float(off.max()):.3e}'
    adds = -(-rows // 512) + 128 + 60
    off = (got[1].cpu().double() - dw).abs() - (half_step(dtype) * dw.abs() + adds * FP32 * dw_mag + tiny(dtype))
    assert float(off.max()) <= 0, f'dw {float(off.max()):.3e}'


def test_gradients_by_differences(dev):
    """Along a random direction d: (L(+) - L(-)) / 2 step of the kernel's own fp32 norm.  L sums 1280 terms of size one whose roundings are
    2^-24 each and independent of the step: with a step of 2^-6 the quotient is off by 1280 * 40 * 2^-24 / 2^-5 = 0.1 at the very most plus
    the third derivative, step^2 times a few times |d|^3; against gradients of size sqrt(1280) = 36."""
    x, w, res = (t.to(dev) for t in inputs(5, 256, f32, True, seed=2, scale=2.0))
    g = torch.Generator().manual_seed(0)
    dy, dsum, ex, ew, er = (torch.randn(*s, generator=g).to(dev) for s in ((5, 256), (5, 256), (5, 256), (256, ), (5, 256)))
    ex, er = ex / 4, er / 4
    leaves = [t.clone().requires_grad_() for t in (x, w, res)]
    grads = torch.autograd.grad(rms_norm(leaves[0], leaves[1], 1e-5, leaves[2]), leaves, [dy, dsum])
    loss = lambda a, b, c: float(sum((o.double() * d.double()).sum() for o, d in zip(rms_norm(a, b, 1e-5, c), (dy, dsum))))
    step = 2.0**-6
    for grad, direction in zip(grads, ((ex, 0, 0), (0, ew, 0), (0, 0, er))):
        d = next(t for t in direction if torch.is_tensor(t))
        up = loss(*(v + step * e for v, e in zip((x, w, res), direction)))
        down = loss(*(v - step * e for v, e in zip((x, w, res), direction)))
        assert abs((up - down) / (2 * step) - float((grad.double() * d.double()).sum())) < 0.15


def test_gradients_that_are_not_asked_for_and_shared_ones(dev):
    x, w, res = (t.to(dev) for t in inputs(6, 512, bf16, True))
    dy = torch.randn(6, 512, device=dev, dtype=bf16)
    # weights alone, input alone, one tensor as input and residual, only the sum used, broadcast gradients
    wl = w.clone().requires_grad_()
    dw, = torch.autograd.grad(rms_norm(x, wl, 1e-6, res)[0], [wl], [dy])
    xl, rl = x.clone().requires_grad_(), res.clone().requires_grad_()
    dx, = torch.autograd.grad(rms_norm(xl, w, 1e-6, res)[0], [xl], [dy])
    full = [t.clone().requires_grad_() for t in (x, w, res)]
    both = torch.autograd.grad(rms_norm(full[0], full[1], 1e-6, full[2])[0], full, [dy])
    assert torch.equal(dw, both[1]) and torch.equal(dx, both[0]) and torch.equal(dx, both[2])
    y, h = rms_norm(xl, w, 1e-6, xl)
    twice, = torch.autograd.grad(y, [xl], [dy])
    single = torch.autograd.grad(rms_norm(full[0], w, 1e-6, full[0].detach())[0], [full[0]], [dy])[0]
    assert float((twice.float() - 2 * single.float()).abs().max()) <= 2 * 2.0**-8 * float(single.float().abs().max())
    only = torch.autograd.grad(rms_norm(xl, wl, 1e-6, rl)[1], [xl, rl], [dy])
    assert torch.equal(only[0], dy) and torch.equal(only[1], dy)
    xl2 = x.clone().requires_grad_()
    rms_norm(xl2, w).sum().backward()  # a gradient with stride 0
    ref = torch.autograd.grad(rms_norm(xl, w), [xl], [torch.ones_like(x)])[0]
    assert torch.equal(xl2.grad, ref)
    d, = torch.autograd.grad(rms_norm(xl, w), [xl], [dy.requires_grad_()], create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


def test_both_paths_give_the_same_bits(dev, monkeypatch):
    x, w, res = (t.to(dev) for t in inputs(9, 1280, bf16, True))
    fast = rms_norm(x, w, 1e-6, res), rms_norm(x, w), rms_norm_quant(x, w, 1e-6, res), rms_norm_quant(x, w, 1e-6, column_major_scales=True)
    monkeypatch.setattr(mod._fast, 'rms_norm', lambda *a: None)
    monkeypatch.setattr(mod._fast, 'rms_norm_quant', lambda *a: None)
    slow = rms_norm(x, w, 1e-6, res), rms_norm(x, w), rms_norm_quant(x, w, 1e-6, res), rms_norm_quant(x, w, 1e-6, column_major_scales=True)
    for a, b in zip(fast, slow):
        for u, v in zip(a if isinstance(a, tuple) else (a, ), b if isinstance(b, tuple) else (b, )):
            assert u.dtype == v.dtype and u.stride() == v.stride() and torch.equal(u.contiguous().view(torch.uint8), v.contiguous().view(torch.uint8))


def test_native_path_takes_plain_calls(dev):
    x, w, res = (t.to(dev) for t in inputs(4, 256, bf16, True))
    assert mod._fast.rms_norm(x, w, 1e-6, res) is not None and mod._fast.rms_norm(x, w, 1e-6, None) is not None
    assert mod._fast.rms_norm_quant(x, w, 1e-6, res, 128, 1e-10, False) is not None
    assert mod._fast.rms_norm(x.requires_grad_(), w, 1e-6, res)[0].grad_fn is not None
    assert mod._fast.rms_norm_quant(x, w, 1e-6, res, 128, 1e-10, False) is None


@pytest.mark.parametrize('residual', [False, True])
def test_gradients_are_those_of_the_python_path(dev, monkeypatch, residual):
    x, w, res = (None if t is None else t.to(dev) for t in inputs(40, 520, bf16, residual))
    dy, dsum = (torch.randn(40, 520, device=dev, dtype=bf16) for _ in range(2))

    def passes():
        leaves = [t.clone().requires_grad_() for t in (x, w, res) if t is not None]
        out = rms_norm(leaves[0], leaves[1], 1e-6, leaves[2] if residual else None)
        out = out if residual else (out, )
        return tuple(out) + torch.autograd.grad(out, leaves, [dy, dsum][:len(out)])

    fast = passes()
    monkeypatch.setattr(mod._fast, 'rms_norm', lambda *a: None)
    for a, b in zip(fast, passes()):
        assert torch.equal(a, b)


def test_registry(dev):
    x, w, _ = (None if t is None else t.to(dev) for t in inputs(4, 256, bf16, False))
    assert torch.equal(dlblas_amd.get_op('rms_norm', (x, w))(x, w), rms_norm(x, w))
    q, s = dlblas_amd.get_op('rms_norm_quant', (x, w))(x, w)
    assert torch.equal(s, rms_norm_quant(x, w)[1])


@pytest.mark.parametrize('up', [2.0**-60, 2.0**55, 2.0**110])
def test_quantiser_near_the_ends_of_fp32(dev, up):
    """Groups whose h w leaves the range in which r cancels: y itself is ordinary."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 256, generator=g).to(bf16)
    w = (torch.rand(256, generator=g) + 0.5).to(bf16)
    h = (x.double() * 2.0**-55).to(bf16) if up != 2.0**-60 else x
    wide = (w.double() * up).to(bf16)
    q, s = rms_norm_quant(*on(dev, h, wide), 1e-38)
    ref_s, v = orc.quant_1x128(orc.rms_norm(h, wide, 1e-38))
    assert float(((s.cpu().double() - ref_s).abs() / ref_s).max()) <= 42 * FP32
    half = (v.abs() * 2.0**-4).clamp_min(2.0**-10)
    assert float(((q.cpu().double() - v).abs() - half - 90 * FP32 * v.abs()).max()) <= 0
