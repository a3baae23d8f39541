"""Products with 4-bit weights at the values where they can go wrong: zero points at and past the end of their range, rows that are nearly
constant, rows close to the end of fp32.

The sizes of MATRICES are served by both kernels: few weights by the one whose waves split K, many by the one whose tiles share x."""
import pytest
import torch

from dlblas_amd.kernels.w4_gemm import w4_gemm, w4_gemm_grouped
from oracle import decoder as orc

pytestmark = pytest.mark.gpu
bf16, f16 = torch.bfloat16, torch.float16
MATRICES = [  # M, N, K, group
    (1, 40, 256, 128), (2, 33, 320, 64), (5, 48, 160, 32), (3, 16401, 544, 32), (16, 8195, 2112, 64), (2, 8193, 2176, 128), (20, 96, 512, 128), (33, 40, 704, 64),
    (40, 129, 96, 32), (3, 203, 18464, 32), (2, 193, 9344, 128),
]


@pytest.fixture(scope='module')
def dev():
    return torch.device('cuda:0')


def half_step(t):
    return torch.finfo(t).eps / 2


def weights(N, K, group, dtype, seed=0):
    g = torch.Generator().manual_seed(N + K + seed)
    q = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, generator=g)
    s = ((0.5 + torch.rand(N, K // group, generator=g)) * 0.01).to(dtype)
    return q, s, torch.randint(0, 17, (N, K // group), dtype=torch.uint8, generator=g)


def on(dev, *tensors):
    return [None if t is None else t.to(dev) for t in tensors]


def check(y, x, q, s, z, what):
    ref, bound = orc.w4_gemm(x, q, s, z)
    off = (y.cpu().double() - ref).abs() - (half_step(y.dtype) * (ref.abs() + bound) + bound + torch.finfo(y.dtype).smallest_normal * half_step(y.dtype))
    assert float(off.max()) <= 0, f'{what}: {float(off.max()):.3e} beyond the bound'


# ---- zero points --------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize('dtype', [bf16, f16])
@pytest.mark.parametrize('M,N,K,group', MATRICES)
def test_zero_points_up_to_16(dev, M, N, K, group, dtype):
    """16 is what a checkpoint that keeps z - 1 comes to: exact like the others, in both kernels."""
    q, s, z = weights(N, K, group, dtype)
    z[::3] = 16
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(dtype)
    check(w4_gemm(*on(dev, x, q, s, z)), x, q, s, z, f'{M}x{N}x{K}/{group}')


@pytest.mark.parametrize('dtype', [bf16, f16])
@pytest.mark.parametrize('M,N,K,group', MATRICES)
def test_zero_points_past_their_range_show(dev, M, N, K, group, dtype):
    """A byte above 16 is no zero point: its column is NaN whichever kernel runs, the others are untouched."""
    q, s, z = weights(N, K, group, dtype)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(dtype)
    good = w4_gemm(*on(dev, x, q, s, z)).cpu()
    g = torch.Generator().manual_seed(5)
    values = torch.tensor([17, 18, 31, 32, 127, 128, 129, 143, 144, 240, 255], dtype=torch.uint8)
    rows = torch.arange(0, N, 5)
    places = torch.randint(0, K // group, (len(rows), ), generator=g)
    places[0], places[-1] = 0, K // group - 1
    z[rows, places] = values[torch.arange(len(rows)) % len(values)]
    y = w4_gemm(*on(dev, x, q, s, z)).cpu()
    bad = torch.zeros(N, dtype=torch.bool)
    bad[rows] = True
    assert bool(y[:, bad].isnan().all()) and torch.equal(y[:, ~bad], good[:, ~bad])


@pytest.mark.parametrize('N,K,group', [(40, 256, 64), (4105, 544, 32), (1056, 2176, 128)])
def test_zero_points_by_expert(dev, N, K, group):
    parts = [weights(N, K, group, f16, seed=e) for e in range(4)]
    q, s, z = (torch.stack(t) for t in zip(*parts))
    z[2, 7] = 17
    x = torch.randn(9, K, generator=torch.Generator().manual_seed(1)).to(f16)
    start, end = torch.tensor([0, 1, 4, 4], dtype=torch.int32), torch.tensor([1, 4, 4, 9], dtype=torch.int32)
    y = w4_gemm_grouped(*on(dev, x, q, s, start, end, z))
    for e in (0, 1, 3):
        a, b = int(start[e]), int(end[e])
        check(y[a:b], x[a:b], q[e], s[e], z[e], f'expert {e}')  # the third expert's byte is nobody's
    end[2], start[3] = 6, 6
    y = w4_gemm_grouped(*on(dev, x, q, s, start, end, z)).cpu()
    assert bool(y[4:6, 7].isnan().all()) and int(y.isnan().sum()) == 2


# ---- rows ---------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize('dtype', [bf16, f16])
@pytest.mark.parametrize('M,N,K,group', MATRICES)
def test_rows_that_are_nearly_constant(dev, M, N, K, group, dtype):
    """sum x (16 + q) and (16 + z) sum x are both large then and their difference is not: the case the bound is made for."""
    q, s, z = weights(N, K, group, dtype)
    g = torch.Generator().manual_seed(M)
    x = (3 * (1 + 2.0**-6 * torch.randn(M, K, generator=g))).to(dtype)
    codes = orc.w4_codes(q).reshape(N, -1, group)
    z = codes.float().mean(-1).round().to(torch.uint8)
    check(w4_gemm(*on(dev, x, q, s, z)), x, q, s, z, f'{M}x{N}x{K}/{group}')
    check(w4_gemm(*on(dev, x, q, s)), x, q, s, None, f'{M}x{N}x{K}/{group}, no zero points')


@pytest.mark.parametrize('M,N,K,group', MATRICES)
def test_rows_close_to_the_end_of_fp32(dev, M, N, K, group):
    """What the bound covers: 32 sum |x| of a group below 2^128.  Rows just inside are products like any other; an infinity gives NaN,
    whatever its weight, since both sums hold it."""
    q, s, z = weights(N, K, group, bf16)
    s = (s.double() * 2.0**-20).to(bf16)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M))
    x = (x * (2.0**122 / x.abs().reshape(M, -1, group).sum(-1).max())).to(bf16)  # 2^127 with the factor 32, and bf16's rounding
    check(w4_gemm(*on(dev, x, q, s, z)), x, q, s, z, f'{M}x{N}x{K}/{group}')
    x[0, K // 2] = float('inf')
    y = w4_gemm(*on(dev, x, q, s, z)).cpu()
    assert bool(y[0].isnan().all()) and bool(y[1:].isfinite().all())
