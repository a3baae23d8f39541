"""Products of a few 16-bit rows with 4-bit floating-point weights, and the layer of experts for a few tokens, against the definitions in 64 bits;
bounds as derived in oracle/mxfp4.py, and half a step of the stored type."""
import pytest
import torch

import dlblas_amd
from dlblas_amd.kernels import few_token_experts as experts_mod
from dlblas_amd.kernels import mxfp4_gemm as mod
from dlblas_amd.kernels.few_token_experts import few_token_experts
from dlblas_amd.kernels.mxfp4_gemm import mxfp4_weight_gemm, per_group_quant_mxfp4
from oracle import mxfp4 as orc

pytestmark = pytest.mark.gpu
bf16, f16, f32, u8, f8 = torch.bfloat16, torch.float16, torch.float32, torch.uint8, torch.float8_e4m3fn


@pytest.fixture(scope='module')
def dev():
    return torch.device('cuda:0')


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * half_step(t)


def inside(got, want, bound, what):
    step = half_step(got.dtype)
    off = (got.cpu().double() - want).abs() - (step * want.abs() + bound * (1 + step) + tiny(got.dtype))
    assert float(off.max()) <= 0, f'{what}: {float(off.max()):.3e} beyond the bound'


def codes(size, K, g, middle=122, spread=2):
    q = torch.randint(0, 256, size + (K // 2, ), generator=g, dtype=u8)
    return q, torch.randint(middle - spread, middle + spread, size + (K // 32, ), generator=g, dtype=u8)


# ---- one matrix ----

SHAPES = [(1, 1, 32), (1, 16, 256), (2, 17, 96), (16, 100, 544), (5, 2112, 7168), (17, 33, 1056), (31, 6400, 288), (32, 64, 4096), (33, 50, 160), (64, 6411, 2080), (100, 30, 64)]


def weight_reference(x, q, s):
    w = orc.values(q, s)
    x = x.double()
    K = x.shape[1]
    return x @ w.t(), (K + 16) * 2 * orc.FP32 * (x.abs() @ w.abs().t())


@pytest.mark.parametrize('dtype', [bf16, f16])
@pytest.mark.parametrize('M,N,K', SHAPES)
def test_product(dev, M, N, K, dtype):
    print(f'case {M}x{N}x{K} {dtype}', flush=True)
    g = torch.Generator().manual_seed(M + N + K)
    x = torch.randn(M, K, generator=g).to(dtype)
    q, s = codes((N, ), K, g)
    y = mxfp4_weight_gemm(*(t.to(dev) for t in (x, q, s)))
    assert y.dtype == dtype and y.shape == (M, N)
    inside(y, *weight_reference(x, q, s), f'{M}x{N}x{K}')


@pytest.mark.parametrize('dtype', [bf16, f16])
def test_every_place_has_its_own_scale(dev, dtype):
    """One group of x alone, weights whose scales differ by up to 2^30 (fp16 rows: sums are scaled in fp32, the result is what its type holds)."""
    g = torch.Generator().manual_seed(3)
    M, N, K = 3, 40, 1056
    x = torch.randn(M, K, generator=g).to(dtype)
    q, s = codes((N, ), K, g, 112, 15)
    for k in range(K // 32):
        one = torch.zeros_like(x)
        one[:, 32 * k:32 * k + 32] = x[:, 32 * k:32 * k + 32]
        y = mxfp4_weight_gemm(*(t.to(dev) for t in (one, q, s)))
        want, bound = weight_reference(one, q, s)
        inside(y, want, bound, f'group {k}')


def test_scales_over_the_whole_range(dev):
    """bf16 rows of size 2^60 and 2^-60 against scales of both ends."""
    g = torch.Generator().manual_seed(4)
    for middle, up in ((20, 2.0**60), (235, 2.0**-60)):
        x = (torch.randn(4, 320, generator=g) * up).to(bf16)
        q, s = codes((24, ), 320, g, middle, 16)
        y = mxfp4_weight_gemm(*(t.to(dev) for t in (x, q, s)))
        inside(y, *weight_reference(x, q, s), f'scales around {middle}')


@pytest.mark.parametrize('dtype', [bf16, f16])
def test_scales_and_rows_that_are_no_numbers(dev, dtype):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(3, 320, generator=g).to(dtype)
    q, s = codes((20, ), 320, g)
    s[4, 9], q[4] = 255, 0
    x[1, 5] = float('nan')
    y = mxfp4_weight_gemm(*(t.to(dev) for t in (x, q, s))).cpu()
    nan = torch.zeros(3, 20, dtype=torch.bool)
    nan[1], nan[:, 4] = True, True
    assert torch.equal(y.isnan(), nan)


def test_rows_where_they_lie(dev):
    g = torch.Generator().manual_seed(6)
    wide = torch.randn(6, 300, generator=g).to(bf16)
    q, s = codes((33, ), 192, g)
    qd, sd = q.to(dev), s.to(dev)
    for off in (0, 1, 2, 3):
        x = wide[:, off:off + 192]
        inside(mxfp4_weight_gemm(wide.to(dev)[:, off:off + 192], qd, sd), *weight_reference(x, q, s), f'offset {off}')
    x = wide[:, :192].contiguous()
    want = mxfp4_weight_gemm(x.to(dev), qd, sd)
    assert torch.equal(mxfp4_weight_gemm(x.to(dev).view(2, 3, 192), qd, sd).view(6, 33), want)
    assert torch.equal(mxfp4_weight_gemm(x.to(dev)[0], qd, sd), want[0])
    assert torch.equal(mxfp4_weight_gemm(x.t().contiguous().to(dev).t(), qd, sd), want)
    assert mxfp4_weight_gemm(x.to(dev)[:0], qd, sd).shape == (0, 33)

    def moved(t, n):
        flat = torch.zeros(t.numel() + n, dtype=u8, device=dev)
        flat[n:] = t.flatten().to(dev)
        return flat[n:].view(t.shape)

    assert torch.equal(mxfp4_weight_gemm(x.to(dev), moved(q, 3), moved(s, 1)), want)


# ---- experts ----


def weights_of(kind, E, H, I, g):
    """(w13, w2) as the call takes them, and their numbers."""
    if kind == 'f4':
        up, down = codes((E, 2 * I), H, g), codes((E, H), I, g)
        return up, down, orc.values(*up), orc.values(*down)

    def f8_of(n, k):
        q = (torch.randn(E, n, k, generator=g) * 60).clamp(-448, 448).to(f8)
        return q, (0.5 + torch.rand(E, -(-n // 128), k // 128, generator=g)) / (60 * k**0.5)

    up, down = f8_of(2 * I, H), f8_of(H, I)
    return up, down, orc.e4m3_values(*up), orc.e4m3_values(*down)


def on(dev, *things):
    return [tuple(t.to(dev) for t in v) if isinstance(v, tuple) else v.to(dev) for v in things]


CASES = [(1, 4, 2, 128, 128), (1, 40, 8, 256, 128), (3, 2, 2, 384, 256), (5, 8, 2, 256, 384), (16, 8, 4, 128, 128), (17, 4, 3, 256, 128), (33, 3, 2, 128, 256), (64, 2, 2, 128, 128),
         (64, 70, 5, 128, 128), (7, 600, 16, 128, 128), (64, 5, 1, 2048, 128)]


@pytest.mark.parametrize('dtype', [bf16, f16])
@pytest.mark.parametrize('kind', ['f8', 'f4'])
@pytest.mark.parametrize('T,E,topk,H,I', CASES)
def test_experts(dev, T, E, topk, H, I, kind, dtype):
    print(f'case experts T={T} E={E} topk={topk} H={H} I={I} {kind} {dtype}', flush=True)
    g = torch.Generator().manual_seed(T + E + topk + H)
    if kind == 'f4':
        H, I = H + 32, I + 96
    x = torch.randn(T, H, generator=g).to(dtype)
    up, down, w13, w2 = weights_of(kind, E, H, I, g)
    # distinct experts of twice as many, some of them elsewhere
    ids = torch.stack([torch.randperm(max(E + E // 3, topk), generator=g)[:topk] for _ in range(T)])
    ids = torch.where(ids < E, ids, torch.full_like(ids, -1)).to(torch.int32 if T % 2 else torch.int64)
    weights = torch.rand(T, topk, generator=g)
    out = few_token_experts(*on(dev, x, ids, weights, up, down))
    assert out.dtype == dtype and out.shape == (T, H)
    inside(out, *orc.experts(x, ids, weights, w13, w2), f'{T} tokens')


@pytest.mark.parametrize('kind', ['f8', 'f4'])
def test_routing_at_its_edges(dev, kind):
    """Every token to one expert, no expert here at all, an expert twice in a token, ids far outside, strided ids."""
    g = torch.Generator().manual_seed(11)
    E, H, I, T = 6, 128, 128, 40
    x = torch.randn(T, H, generator=g).to(bf16)
    up, down, w13, w2 = weights_of(kind, E, H, I, g)
    weights = torch.rand(T, 3, generator=g)
    some = torch.randint(0, E, (T, 3), generator=g)
    table = {
        'one expert': torch.full((T, 3), 5),
        'nowhere': torch.full((T, 3), -1),
        'twice': torch.stack([some[:, 0], some[:, 1], some[:, 0]], 1),
        'outside': torch.where(some < 3, some, torch.full_like(some, 1 << 40)),
        'below': torch.where(some < 3, some, torch.full_like(some, -(1 << 40))),
    }
    for name, ids in table.items():
        out = few_token_experts(*on(dev, x, ids, weights, up, down))
        inside(out, *orc.experts(x, ids, weights, w13, w2), name)
    assert float(few_token_experts(*on(dev, x, table['nowhere'], weights, up, down)).abs().max()) == 0.0
    strided = some.t().contiguous().to(dev).t()
    assert torch.equal(few_token_experts(x.to(dev), strided, *on(dev, weights, up, down)), few_token_experts(*on(dev, x, some, weights, up, down)))
    small = [t[:2].contiguous() for t in up], [t[:2].contiguous() for t in down]
    ids = torch.tensor([[0, 1, 0], [1, 1, 1]])  # more slots than experts, all named twice
    inside(few_token_experts(*on(dev, x[:2], ids, weights[:2], tuple(small[0]), tuple(small[1]))), *orc.experts(x[:2], ids, weights[:2], w13[:2], w2[:2]), 'two experts')
    ids = torch.tensor([[4, 4, 4]])  # fewer slots than experts
    inside(few_token_experts(*on(dev, x[:1], ids, weights[:1], up, down)), *orc.experts(x[:1], ids, weights[:1], w13, w2), 'three times')


def test_no_tokens_and_values_that_are_no_numbers(dev):
    g = torch.Generator().manual_seed(12)
    up, down, _, _ = weights_of('f8', 4, 256, 128, g)
    x = torch.randn(5, 256, generator=g).to(bf16)
    ids = torch.tensor([[0, 1], [1, 2], [2, 3], [3, 0], [1, 3]], dtype=torch.int32)
    weights = torch.rand(5, 2, generator=g)
    assert few_token_experts(*on(dev, x[:0], ids[:0], weights[:0], up, down)).shape == (0, 256)
    want = few_token_experts(*on(dev, x, ids, weights, up, down)).cpu()
    x[2, 7] = float('nan')
    out = few_token_experts(*on(dev, x, ids, weights, up, down)).cpu()
    assert bool(out[2].isnan().all()) and torch.equal(out[[0, 1, 3, 4]], want[[0, 1, 3, 4]])  # the other tokens of its experts keep theirs
    bad = up[0].clone().view(u8)
    bad[3, 5, 9] = 0x7f  # a weight of expert 3
    out = few_token_experts(*on(dev, torch.randn(5, 256, generator=g).to(bf16), ids, weights, (bad.view(f8), up[1]), down)).cpu()
    assert out.isnan().all(1).tolist() == [False, False, True, True, True]


@pytest.mark.parametrize('kind', ['f8', 'f4'])
def test_both_paths_give_the_same_bits(dev, monkeypatch, kind):
    g = torch.Generator().manual_seed(13)
    up, down, _, _ = weights_of(kind, 4, 256, 128, g)
    args = on(dev, torch.randn(9, 256, generator=g).to(bf16), torch.randint(-1, 4, (9, 2), generator=g), torch.rand(9, 2, generator=g), up, down)
    x, (q, s) = args[0], on(dev, codes((70, ), 256, g))[0]
    a, a_s = per_group_quant_mxfp4(x)
    calls = [lambda: few_token_experts(*args), lambda: mxfp4_weight_gemm(x, q, s), lambda: per_group_quant_mxfp4(x)[0], lambda: per_group_quant_mxfp4(x)[1],
             lambda: mod.mxfp4_gemm(a, q, a_s, s), lambda: mod.mxfp4_gemm(a, q, a_s, s, f16)]
    assert mod._fast.few_token_experts(*args) is not None and mod._fast.mxfp4_weight_gemm(x, q, s) is not None
    assert mod._fast.per_group_quant_mxfp4(x) is not None and mod._fast.mxfp4_gemm(a, q, a_s, s, None) is not None
    fast = [call() for call in calls]
    for name in ('few_token_experts', 'mxfp4_weight_gemm', 'per_group_quant_mxfp4', 'mxfp4_gemm'):
        monkeypatch.setattr(mod._fast, name, lambda *a: None)
    for want, call in zip(fast, calls):
        got = call()
        assert got.dtype == want.dtype and torch.equal(got, want)


def test_registry(dev):
    g = torch.Generator().manual_seed(14)
    q, s = on(dev, codes((70, ), 256, g))[0]
    x = torch.randn(4, 256, generator=g).to(bf16).to(dev)
    assert torch.equal(dlblas_amd.get_op('mxfp4_weight_gemm', (x, q, s))(x, q, s), mxfp4_weight_gemm(x, q, s))
    assert experts_mod.few_token_experts is few_token_experts
