"""4-bit floating point: quantiser and products against the definitions in 64 bits.

The quantiser is exact arithmetic (powers of two, one rounding): codes and scales are equal bit for bit.  Products: the sum of a group is exact; the
sums over K / 32 groups take at most K / 32 + 8 additions in fp32, each off by at most 2^-23 of the sum of magnitudes (the unit cuts off where it does not
round), then half a step of the stored type."""
import pytest
import torch

import dlblas_amd
from dlblas_amd.kernels import mxfp4_gemm as mod
from dlblas_amd.kernels.mxfp4_gemm import mxfp4_gemm, per_group_quant_mxfp4
from oracle import mxfp4 as orc

pytestmark = pytest.mark.gpu
bf16, f16, f32, u8 = torch.bfloat16, torch.float16, torch.float32, torch.uint8


@pytest.fixture(scope='module')
def dev():
    return torch.device('cuda:0')


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * half_step(t)


def operand(rows, K, g, spread=3):
    q = torch.randint(0, 256, (rows, K // 2), generator=g, dtype=u8)
    s = torch.randint(124 - spread, 124 + spread, (rows, K // 32), generator=g, dtype=u8)
    return q, s


def inside(got, want, mag, adds, what):
    step = half_step(got.dtype)
    off = (got.cpu().double() - want).abs() - (step * want.abs() + adds * 2 * orc.FP32 * mag * (1 + step) + tiny(got.dtype))
    assert float(off.max()) <= 0, f'{what}: {float(off.max()):.3e} beyond the bound'


# ---- quantiser ----


@pytest.mark.parametrize('dtype', [bf16, f16, f32])
@pytest.mark.parametrize('rows,K', [(1, 32), (3, 64), (7, 96), (33, 7168), (1000, 1056), (2, 18432)])
def test_codes(dev, rows, K, dtype):
    g = torch.Generator().manual_seed(rows + K)
    x = (torch.randn(rows, K, generator=g) * torch.exp2(torch.randint(-8, 8, (rows, 1), generator=g).float())).to(dtype)
    q, s = per_group_quant_mxfp4(x.to(dev))
    want_q, want_s = orc.quant(x)
    assert q.dtype == s.dtype == u8 and torch.equal(s.cpu(), want_s) and torch.equal(q.cpu(), want_q)


@pytest.mark.parametrize('dtype', [bf16, f16, f32])
def test_every_border_between_two_codes(dev, dtype):
    """Halves of all codes, their neighbours on both sides, at every scale that the type has room for, both signs."""
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.5], dtype=torch.float64)
    eps = torch.finfo(dtype).eps
    near = torch.cat([borders, borders * (1 - 2 * eps), borders * (1 + 2 * eps), torch.tensor([4.0])])
    rows = []
    for e in range(-100, 100, 7) if dtype != f16 else range(-9, 12):
        rows.append(torch.cat([near, torch.zeros(1, dtype=torch.float64)])[:32] * 2.0**e)
    x = torch.stack(rows).to(dtype)
    assert x.shape[1] == 32
    x = torch.cat([x, -x], 1)
    q, s = per_group_quant_mxfp4(x.to(dev))
    want_q, want_s = orc.quant(x)
    assert torch.equal(s.cpu(), want_s) and torch.equal(q.cpu(), want_q)


def test_groups_of_zeros_tiny_huge_and_no_numbers(dev):
    x = torch.zeros(8, 64)
    x[1, 3] = float('nan')
    x[2, 5], x[2, 40] = float('inf'), 1.0
    x[3] = -0.0
    x[4, :4] = torch.tensor([2.0**-149, 2.0**-127, -(2.0**-128), 3 * 2.0**-130])
    x[5, :2] = torch.tensor([3.4e38, -1e38])
    x[6, :3] = torch.tensor([2.0**-126, 2.0**-125, 2.0**-127])
    x[7, 0] = 2.0**-149
    for dtype in (f32, bf16):
        y = x.to(dtype)
        q, s = per_group_quant_mxfp4(y.to(dev))
        want_q, want_s = orc.quant(y)
        assert torch.equal(s.cpu(), want_s), dtype
        assert torch.equal(q.cpu(), want_q), dtype
        assert s[1, 0] == 255 and s[1, 1] == 0 and s[2, 0] == 255 and s[2, 1] == 125


def test_rows_where_they_lie(dev):
    g = torch.Generator().manual_seed(1)
    wide = torch.randn(6, 300, generator=g).to(bf16)
    for off in (0, 1, 3, 8):
        q, s = per_group_quant_mxfp4(wide.to(dev)[:, off:off + 96])
        want_q, want_s = orc.quant(wide[:, off:off + 96])
        assert torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s)
    cube = torch.randn(2, 3, 64, generator=g)
    q, s = per_group_quant_mxfp4(cube.to(dev).transpose(0, 1))
    want_q, want_s = orc.quant(cube.transpose(0, 1))
    assert q.shape == (3, 2, 32) and s.shape == (3, 2, 2) and torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s)
    q, s = per_group_quant_mxfp4(cube[0, 0].to(dev))
    assert q.shape == (32, ) and s.shape == (2, )
    q, s = per_group_quant_mxfp4(torch.empty(0, 64, device=dev))
    assert q.shape == (0, 32) and s.shape == (0, 2)


# ---- product ----

SHAPES = [(1, 1, 32), (1, 16, 512), (3, 17, 96), (16, 100, 544), (5, 2112, 7168), (17, 33, 1056), (32, 64, 4096), (40, 50, 160), (64, 200, 2080), (65, 70, 32), (100, 130, 96), (129, 127, 128),
          (200, 300, 1056), (128, 128, 640), (300, 1000, 544), (513, 257, 4096)]


@pytest.mark.parametrize('out', [bf16, f16, f32])
@pytest.mark.parametrize('M,N,K', SHAPES)
def test_product(dev, M, N, K, out):
    print(f'case product {M}x{N}x{K} {out}', flush=True)
    g = torch.Generator().manual_seed(M + N + K)
    (a, a_s), (b, b_s) = operand(M, K, g), operand(N, K, g)
    c = mxfp4_gemm(*(t.to(dev) for t in (a, b, a_s, b_s)), out)
    assert c.dtype == out and c.shape == (M, N)
    inside(c, *orc.gemm(a, a_s, b, b_s), K // 32 + 8, f'{M}x{N}x{K}')


@pytest.mark.parametrize('M,N,K', [(2100, 4100, 288), (4096, 2304, 1024), (2050, 4097, 1056)])
def test_product_of_many_tiles(dev, M, N, K):
    """The large tiles: checked on the device, in 64 bits."""
    print(f'case large product {M}x{N}x{K}', flush=True)
    g = torch.Generator().manual_seed(M)
    (a, a_s), (b, b_s) = operand(M, K, g), operand(N, K, g)
    c = mxfp4_gemm(*(t.to(dev) for t in (a, b, a_s, b_s)), f32)
    x, w = orc.values(a, a_s).to(dev), orc.values(b, b_s).to(dev)
    off = (c.double() - x @ w.t()).abs() - 2 * orc.FP32 * (K // 32 + 9) * (x.abs() @ w.abs().t())
    assert float(off.max()) <= 0


@pytest.mark.parametrize('M', [4, 70])
def test_scales_over_the_whole_range(dev, M):
    """Products of scales between 2^-100 and 2^100, and the sums of groups that differ by much: every lane's scale at its own place."""
    g = torch.Generator().manual_seed(M)
    K, N = 1056, 40
    (a, _), (b, _) = operand(M, K, g), operand(N, K, g)
    a_s, b_s = (torch.randint(77, 177, (r, K // 32), generator=g, dtype=u8) for r in (M, N))
    c = mxfp4_gemm(*(t.to(dev) for t in (a, b, a_s, b_s)), f32)
    inside(c, *orc.gemm(a, a_s, b, b_s), K // 32 + 8, 'wide scales')
    # one group alone, at every place of K
    for k in range(K // 32):
        one = torch.zeros_like(a)
        one[:, 16 * k:16 * k + 16] = a[:, 16 * k:16 * k + 16]
        c = mxfp4_gemm(*(t.to(dev) for t in (one, b, a_s, b_s)), f32)
        inside(c, *orc.gemm(one, a_s, b, b_s), 9, f'group {k}')


@pytest.mark.parametrize('M', [3, 80])
def test_a_scale_that_is_no_number(dev, M):
    g = torch.Generator().manual_seed(M)
    (a, a_s), (b, b_s) = operand(M, 160, g), operand(50, 160, g)
    a_s[1, 4] = 255
    b_s[7, 0] = 255
    b[7] = 0  # zeros do not hide it
    c = mxfp4_gemm(*(t.to(dev) for t in (a, b, a_s, b_s)), f32).cpu()
    nan = torch.zeros(M, 50, dtype=torch.bool)
    nan[1], nan[:, 7] = True, True
    assert torch.equal(c.isnan(), nan)


def test_extents_and_places(dev):
    """Three dimensions, no rows, operands that start off 16 bytes, the default type."""
    g = torch.Generator().manual_seed(7)
    (a, a_s), (b, b_s) = operand(6, 192, g), operand(33, 192, g)
    want = mxfp4_gemm(*(t.to(dev) for t in (a, b, a_s, b_s)), bf16)
    cube = mxfp4_gemm(a.to(dev).view(2, 3, 96), b.to(dev), a_s.to(dev).view(2, 3, 6), b_s.to(dev), bf16)
    assert cube.shape == (2, 3, 33) and torch.equal(cube.view(6, 33), want)
    row = mxfp4_gemm(a.to(dev)[0], b.to(dev), a_s.to(dev)[0], b_s.to(dev), bf16)
    assert row.shape == (33, ) and torch.equal(row, want[0])

    def moved(t, n):
        flat = torch.zeros(t.numel() + n, dtype=u8, device=dev)
        flat[n:] = t.flatten().to(dev)
        return flat[n:].view(t.shape)

    assert torch.equal(mxfp4_gemm(moved(a, 3), moved(b, 5), moved(a_s, 1), moved(b_s, 2), bf16), want)
    assert mxfp4_gemm(a.to(dev)[:0], b.to(dev), a_s.to(dev)[:0], b_s.to(dev)).shape == (0, 33)
    assert mxfp4_gemm(a.to(dev), b.to(dev)[:0], a_s.to(dev), b_s.to(dev)[:0]).shape == (6, 0)
    assert mxfp4_gemm(*(t.to(dev) for t in (a, b, a_s, b_s))).dtype == torch.get_default_dtype()


def test_registry(dev):
    g = torch.Generator().manual_seed(8)
    (a, a_s), (b, b_s) = operand(6, 192, g), operand(33, 192, g)
    args = tuple(t.to(dev) for t in (a, b, a_s, b_s))
    assert torch.equal(dlblas_amd.get_op('mxfp4_gemm', args)(*args), mxfp4_gemm(*args))
    x = torch.randn(4, 64, device=dev)
    assert torch.equal(dlblas_amd.get_op('per_group_quant_mxfp4', (x, ))(x)[0], per_group_quant_mxfp4(x)[0])
