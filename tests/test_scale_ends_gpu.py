"""4-bit weights whose scales are at the ends of the format, 2^-127 and 2^127, beside rows and between products that make their parts ordinary numbers: bf16 holds neither 2^128
nor, but as subnormal numbers, what is below 2^-126.  Bounds as in the tests of the same calls at ordinary scales."""
import pytest
import torch

from dlblas_amd.kernels.few_token_experts import few_token_experts
from dlblas_amd.kernels.mxfp4_gemm import mxfp4_weight_gemm
from oracle import mxfp4 as orc

pytestmark = pytest.mark.gpu
bf16, f16, u8 = torch.bfloat16, torch.float16, torch.uint8


@pytest.fixture(scope='module')
def dev():
    return torch.device('cuda:0')


def inside(got, want, bound, what):
    step = torch.finfo(got.dtype).eps / 2
    off = (got.cpu().double() - want).abs() - (step * want.abs() + bound * (1 + step) + torch.finfo(got.dtype).smallest_normal * step)
    assert float(off.max()) <= 0, f'{what}: {float((off / want.abs().max()).max()):.3e} of the largest beyond the bound'


def codes(size, K, g, lowest, count):
    return torch.randint(0, 256, size + (K // 2, ), generator=g, dtype=u8), torch.randint(lowest, lowest + count, size + (K // 32, ), generator=g, dtype=u8)


def on(dev, *things):
    return [tuple(t.to(dev) for t in v) if isinstance(v, tuple) else v.to(dev) for v in things]


@pytest.mark.parametrize('M', [1, 7, 16, 40])
@pytest.mark.parametrize('lowest,count,up', [(0, 1, 2.0**100), (1, 1, 2.0**100), (0, 6, 2.0**100), (0, 3, 2.0**125), (249, 6, 2.0**-60), (253, 1, 2.0**-60), (254, 1, 2.0**-100)])
def test_product(dev, M, lowest, count, up):
    """Rows of which one is zeros: a weight that is an infinity would make it NaN.  Up to 2^125: the sums before a scale of 2^-127 must not pass 2^128."""
    g = torch.Generator().manual_seed(M + lowest)
    for N, K in ((70, 1056), (33, 32), (20, 2048)):
        x = (torch.randn(M, K, generator=g).clamp(-2, 2) * up).to(bf16)
        x[M // 2] = 0
        q, s = codes((N, ), K, g, lowest, count)
        y = mxfp4_weight_gemm(*on(dev, x, q, s))
        w = orc.values(q, s)
        inside(y, x.double() @ w.t(), (K + 16) * 2 * orc.FP32 * (x.double().abs() @ w.abs().t()), f'{M}x{N}x{K}')


def test_one_such_group_among_others(dev):
    """At every place of K, of every row of a tile."""
    g = torch.Generator().manual_seed(3)
    K, N = 544, 40
    x = torch.randn(5, K, generator=g).to(bf16)
    q, s = codes((N, ), K, g, 120, 4)
    for k in range(K // 32):
        for s_at, up in ((254, 2.0**-100), (0, 2.0**100)):
            t, y = s.clone(), x.clone()
            t[k % N::16, k] = s_at
            y[:, 32 * k:32 * k + 32] *= up
            w = orc.values(q, t)
            inside(mxfp4_weight_gemm(*on(dev, y, q, t)), y.double() @ w.t(), (K + 16) * 2 * orc.FP32 * (y.double().abs() @ w.abs().t()), f'group {k}, scale {s_at}')


def test_no_numbers_beside_them(dev):
    g = torch.Generator().manual_seed(5)
    x = (torch.randn(3, 320, generator=g) * 2.0**-60).to(bf16)
    q, s = codes((20, ), 320, g, 252, 3)
    s[4, 9], q[4] = 255, 0
    x[1, 5] = float('nan')
    y = mxfp4_weight_gemm(*on(dev, x, q, s)).cpu()
    nan = torch.zeros(3, 20, dtype=torch.bool)
    nan[1], nan[:, 4] = True, True
    assert torch.equal(y.isnan(), nan)


@pytest.mark.parametrize('T,E,topk', [(2, 2, 1), (4, 3, 2), (13, 4, 2), (40, 3, 2)])
@pytest.mark.parametrize('gates,ups,downs,up,dtype', [((252, 3), (227, 1), (0, 3), -100, bf16), ((223, 1), (130, 3), (251, 4), -100, bf16), ((122, 3), (122, 3), (0, 256), 0, bf16),
                                                      ((122, 3), (122, 3), (0, 256), 0, f16)])
def test_experts(dev, T, E, topk, gates, ups, downs, up, dtype):
    """Rows of 2^-100 against scales of 2^127: g up to 2^27, u of about 1, their sums times 2^-127.  g of about 1, u of 2^-97, times 2^127.  The second matrix's scales from one end to the other."""
    print(f'case T={T} E={E} gates {gates} ups {ups} downs {downs} {dtype}', flush=True)
    g = torch.Generator().manual_seed(T + downs[0])
    H, I = 160, 544
    x = (torch.randn(T, H, generator=g) * 2.0**up).to(dtype)
    gate, other = codes((E, I), H, g, *gates), codes((E, I), H, g, *ups)
    w13 = tuple(torch.cat(t, 1) for t in zip(gate, other))
    w2 = codes((E, H), I, g, *downs)
    if downs[1] == 256:  # any scale but NaN, of few columns: one group alone
        w2 = w2[0], torch.full_like(w2[1], 0)
        w2[1][:, :, 3] = torch.randint(0, 255, (E, H), generator=g, dtype=u8)
    ids = torch.stack([torch.randperm(E, generator=g)[:topk] for _ in range(T)])
    weights = torch.rand(T, topk, generator=g)
    want, bound = orc.experts(x, ids, weights, orc.values(*w13), orc.values(*w2))
    out = few_token_experts(*on(dev, x, ids, weights, w13, w2))
    # where the terms' magnitudes add up to less than the output's type holds: a sum whose parts pass 2^128 is an infinity in fp32 though the whole does not.  (I + 40) 2 2^-24 of them is in
    # the bound.
    here = bound < torch.finfo(dtype).max * (I + 40) * 2 * orc.FP32
    assert bool(here.any()) and bool(out.cpu()[here].isfinite().all())
    inside(torch.where(here.to(dev), out, torch.zeros_like(out)), torch.where(here, want, torch.zeros_like(want)), bound, f'{T} tokens')
