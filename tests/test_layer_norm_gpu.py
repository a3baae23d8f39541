"""Layer norm and its gradients against the definitions in 64 bits; the bounds are those of oracle/layer_norm.py plus half a step of the stored
type.  dw, db: a workgroup adds at most rows / 256 + 1 terms, a lane of the second kernel an eighth of a sixteenth of up to 4096 shares, and their sums
are added in 3 + 4 steps: below rows / 256 + 128 + 60 roundings of the sum of magnitudes, as for the RMS norm."""
import pytest
import torch

import dlblas_amd
from dlblas_amd.kernels import layer_norm as mod
from dlblas_amd.kernels.layer_norm import layer_norm
from oracle import layer_norm as orc

pytestmark = pytest.mark.gpu
bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope='module')
def dev():
    return torch.device('cuda:0')


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """Half a step of the subnormal numbers of a type."""
    return torch.finfo(t).smallest_normal * half_step(t)


def inputs(rows, H, dtype, residual, bias=True, w_dtype=None, seed=0):
    g = torch.Generator().manual_seed(1000 * rows + H + seed)
    x = torch.randn(rows, H, generator=g) + 0.5 * torch.randn(rows, 1, generator=g)
    x[:, ::7] *= 8
    res = torch.randn(rows, H, generator=g).to(dtype) if residual else None
    w = (1 + 0.2 * torch.randn(H, generator=g)).to(w_dtype or dtype)
    b = (0.5 * torch.randn(H, generator=g)).to(w_dtype or dtype) if bias else None
    return x.to(dtype), w, b, res


def on(dev, *tensors):
    return [None if t is None else t.to(dev) for t in tensors]


def inside(got, want, bound, what):
    step = half_step(got.dtype)
    off = (got.detach().cpu().double() - want).abs() - (bound * (1 + step) + step * want.abs() + tiny(got.dtype))
    assert float(off.max()) <= 0, f'{what}: {float(off.max()):.3e} beyond the bound'


def check_y(y, h, w, b, eps, what):
    inside(y, *orc.layer_norm(h, w, b, eps), what)


SHAPES = [(1, 1), (1, 7), (3, 8), (2, 9), (5, 64), (33, 128), (4, 127), (9, 248), (3, 513), (2, 1000), (300, 264), (7, 2050), (2, 4096), (1, 7168), (33, 7168), (2, 8199),
          (3, 16384), (2, 20001), (1, 32768)]


@pytest.mark.parametrize('dtype', [bf16, f16, f32])
@pytest.mark.parametrize('residual,bias', [(False, True), (True, False), (True, True)])
@pytest.mark.parametrize('rows,H', SHAPES)
def test_norm(dev, rows, H, residual, bias, dtype):
    x, w, b, res = inputs(rows, H, dtype, residual, bias)
    xd, wd, bd, rd = on(dev, x, w, b, res)
    out = layer_norm(xd, wd, bd, 1e-5, rd)
    h = orc.norm_input(x, res)
    if residual:
        out, hd = out
        assert torch.equal(hd.cpu(), h)
    check_y(out, h, w, b, 1e-5, f'{rows}x{H} {dtype}')


def test_weights_in_32_bits(dev):
    for dtype in (bf16, f16):
        x, w, b, res = inputs(6, 776, dtype, True, w_dtype=f32)
        y, h = layer_norm(*on(dev, x, w, b), 1e-6, *on(dev, res))
        check_y(y, h.cpu(), w, b, 1e-6, 'fp32 weights')


@pytest.mark.parametrize('dtype', [bf16, f32])
def test_rows_where_they_lie(dev, dtype):
    """Rows of a wider tensor, at any element offset, broadcast rows, transposed and three-dimensional inputs."""
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(6, 300, generator=g).to(dtype)
    w, b = (torch.randn(130, generator=g).to(dtype) for _ in range(2))
    wd, w_, b_ = on(dev, wide, w, b)
    for off in (0, 1, 2, 3, 5, 8):
        x, r = wide[:, off:off + 130], wide[:, off + 140:off + 270]
        y, h = layer_norm(wd[:, off:off + 130], w_, b_, 1e-6, wd[:, off + 140:off + 270])
        assert torch.equal(h.cpu(), orc.norm_input(x, r))
        check_y(y, h.cpu(), w, b, 1e-6, f'offset {off}')
    row = wide[:1, :130]
    check_y(layer_norm(row.to(dev).expand(9, 130), w_, b_), row.expand(9, 130), w, b, 1e-5, 'broadcast')
    t = torch.randn(130, 4, generator=g).to(dtype)
    check_y(layer_norm(t.to(dev).t(), w_, b_), t.t(), w, b, 1e-5, 'transposed')
    strided = torch.randn(260, generator=g).to(dtype)
    check_y(layer_norm(row.to(dev), strided.to(dev)[::2], b_), row, strided[::2], b, 1e-5, 'weights that do not lie together')
    cube = torch.randn(2, 3, 130, generator=g).to(dtype)
    y = layer_norm(cube.to(dev), w_, b_)
    assert y.shape == cube.shape
    check_y(y, cube, w, b, 1e-5, 'three dimensions')
    vec = layer_norm(cube[0, 0].to(dev), w_, b_)
    assert vec.shape == (130, ) and torch.equal(vec, y[0, 0])


def test_no_rows(dev):
    w = torch.ones(256, device=dev, dtype=bf16, requires_grad=True)
    b = torch.ones(256, device=dev, dtype=bf16, requires_grad=True)
    x = torch.empty(0, 256, device=dev, dtype=bf16)
    assert layer_norm(x, w.detach()).shape == (0, 256)
    layer_norm(x, w, b).sum().backward()
    assert float(w.grad.float().abs().max()) == 0.0 and float(b.grad.float().abs().max()) == 0.0


def test_constant_rows_and_values_that_are_no_numbers(dev):
    x = torch.zeros(4, 256, dtype=bf16)
    x[1, 3] = float('nan')
    x[2, 200] = float('inf')
    x[3] = 3.0
    w, b = torch.full((256, ), 2.0, dtype=bf16), torch.full((256, ), 0.25, dtype=bf16)
    y = layer_norm(*on(dev, x, w, b)).cpu()
    assert bool((y[0] == 0.25).all()) and bool(y[1:3].isnan().all()) and bool((y[3] == 0.25).all())


def test_a_row_far_from_zero(dev):
    """mean(h^2) - mean(h)^2 in fp32 would be noise: the spread is 2^-12 of the mean."""
    g = torch.Generator().manual_seed(9)
    x = 1000.0 + 0.25 * torch.randn(3, 4096, generator=g)
    w, b = torch.ones(4096), torch.zeros(4096)
    y = layer_norm(*on(dev, x, w, b))
    ref, bound = orc.layer_norm(x, w, b, 1e-5)
    inside(y, ref, bound, 'far from zero')
    assert float((y.cpu().double() - ref).abs().max()) < 0.01


GRAD_SHAPES = [(1, 1), (2, 9), (5, 64), (4, 127), (1100, 136), (600, 513), (7, 2050), (33, 7168), (2, 9000), (3, 20001), (17, 128), (9001, 64), (5003, 256), (8301, 520), (2, 8), (33, 248),
               (1, 32768)]


@pytest.mark.parametrize('dtype', [bf16, f16, f32])
@pytest.mark.parametrize('residual,bias', [(False, True), (True, False), (True, True)])
@pytest.mark.parametrize('rows,H', GRAD_SHAPES)
def test_gradients(dev, rows, H, residual, bias, dtype):
    x, w, b, res = inputs(rows, H, dtype, residual, bias, seed=1)
    g = torch.Generator().manual_seed(rows + H)
    dy, dsum = (torch.randn(rows, H, generator=g).to(dtype) for _ in range(2))
    leaves = {name: t.to(dev).requires_grad_() for name, t in (('x', x), ('w', w), ('b', b), ('res', res)) if t is not None}
    out = layer_norm(leaves['x'], leaves['w'], leaves.get('b'), 1e-5, leaves.get('res'))
    if residual:
        grads = torch.autograd.grad(out, list(leaves.values()), on(dev, dy, dsum))
        check_y(out[0], out[1].detach().cpu(), w, b, 1e-5, 'with gradient')
    else:
        grads = torch.autograd.grad([out], list(leaves.values()), on(dev, dy))
    got = dict(zip(leaves, grads))
    (dx, dw, db), (dx_off, (n_off, dw_mag), db_mag) = orc.layer_norm_grad(dy, dsum if residual else None, orc.norm_input(x, res), w, 1e-5)
    inside(got['x'], dx, dx_off, 'dx')
    if residual:
        assert torch.equal(got['res'], got['x'])
    adds = -(-rows // 256) + 128 + 60
    inside(got['w'], dw, n_off + adds * orc.FP32 * dw_mag, 'dw')
    if bias:
        inside(got['b'], db, adds * orc.FP32 * db_mag, 'db')


def test_gradients_by_differences(dev):
    """Along a direction, from the kernel's own fp32 norm: L sums 1280 terms whose roundings are about 2^-22 each and independent of the step
    2^-6, so the quotient is off by 1280 * 50 * 2^-24 / 2^-5 = 0.12 at the very most, plus the third derivative times the step's square."""
    x, w, b, res = on(dev, *inputs(5, 256, f32, True, seed=2))
    g = torch.Generator().manual_seed(0)
    dy, dsum, ex, ew, eb, er = (torch.randn(*s, generator=g).to(dev) for s in ((5, 256), (5, 256), (5, 256), (256, ), (256, ), (5, 256)))
    ex, er = ex / 4, er / 4
    leaves = [t.clone().requires_grad_() for t in (x, w, b, res)]
    grads = torch.autograd.grad(layer_norm(leaves[0], leaves[1], leaves[2], 1e-5, leaves[3]), leaves, [dy, dsum])
    loss = lambda x, w, b, r: float(sum((o.double() * d.double()).sum() for o, d in zip(layer_norm(x, w, b, 1e-5, r), (dy, dsum))))
    step = 2.0**-6
    for i, d in enumerate((ex, ew, eb, er)):
        up, down = ([t + sign * step * d if j == i else t for j, t in enumerate((x, w, b, res))] for sign in (1, -1))
        assert abs((loss(*up) - loss(*down)) / (2 * step) - float((grads[i].double() * d.double()).sum())) < 0.16


def test_gradients_that_are_not_asked_for_and_shared_ones(dev):
    x, w, b, res = on(dev, *inputs(6, 512, bf16, True))
    dy = torch.randn(6, 512, device=dev, dtype=bf16)
    full = [t.clone().requires_grad_() for t in (x, w, b, res)]
    want = torch.autograd.grad(layer_norm(full[0], full[1], full[2], 1e-5, full[3])[0], full, [dy])
    for i in range(4):  # one alone
        alone = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b, res))]
        got, = torch.autograd.grad(layer_norm(alone[0], alone[1], alone[2], 1e-5, alone[3])[0], [alone[i]], [dy])
        assert torch.equal(got, want[i]), i
    # without a bias, the residual alone
    rl = res.clone().requires_grad_()
    got, = torch.autograd.grad(layer_norm(x, w, None, 1e-5, rl)[0], [rl], [dy])
    assert torch.equal(got, want[3])
    # the same tensor twice, the sum alone, a broadcast gradient, a second derivative
    xl = x.clone().requires_grad_()
    twice, = torch.autograd.grad(layer_norm(xl, w, b, 1e-5, xl)[0], [xl], [dy])
    single, = torch.autograd.grad(layer_norm(full[0], w, b, 1e-5, full[0].detach())[0], [full[0]], [dy])
    assert torch.equal(twice, single + single)
    only = torch.autograd.grad(layer_norm(full[0], full[1], full[2], 1e-5, full[3])[1], [full[0], full[3]], [dy])
    assert torch.equal(only[0], dy) and torch.equal(only[1], dy)
    layer_norm(xl, w, b).sum().backward()
    assert torch.equal(xl.grad, torch.autograd.grad(layer_norm(full[0], w, b), [full[0]], [torch.ones_like(x)])[0])
    d, = torch.autograd.grad(layer_norm(xl, w, b), [xl], [dy.requires_grad_()], create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


@pytest.mark.parametrize('residual,bias', [(False, True), (True, True), (True, False)])
def test_both_paths_give_the_same_bits(dev, monkeypatch, residual, bias):
    x, w, b, res = on(dev, *inputs(40, 520, bf16, residual, bias))
    dy, dsum = (torch.randn(40, 520, device=dev, dtype=bf16) for _ in range(2))

    def passes():
        plain = layer_norm(x, w, b, 1e-5, res)
        leaves = [None if t is None else t.clone().requires_grad_() for t in (x, w, b, res)]
        out = layer_norm(leaves[0], leaves[1], leaves[2], 1e-5, leaves[3])
        out, plain = (out, plain) if residual else ((out, ), (plain, ))
        return tuple(plain) + tuple(out) + torch.autograd.grad(out, [t for t in leaves if t is not None], [dy, dsum][:len(out)])

    assert mod._fast.layer_norm(x, w, b, 1e-5, res) is not None
    fast = passes()
    monkeypatch.setattr(mod._fast, 'layer_norm', lambda *a: None)
    for a, c in zip(fast, passes()):
        assert torch.equal(a, c)


def test_registry(dev):
    x, w, b, _ = on(dev, *inputs(4, 256, bf16, False))
    assert torch.equal(dlblas_amd.get_op('layer_norm', (x, w, b))(x, w, b), layer_norm(x, w, b))
