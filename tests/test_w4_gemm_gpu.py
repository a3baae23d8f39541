"""Products with 4-bit weights against the definition in 64 bits; the bound on the fp32 sums is derived in oracle/decoder.py, the result's
rounding adds half a step of its type."""
import pytest
import torch

import dlblas_amd
from dlblas_amd.kernels import w4_gemm as mod
from dlblas_amd.kernels.w4_gemm import per_group_quant_w4, w4_gemm, w4_gemm_grouped
from oracle import decoder as orc

pytestmark = pytest.mark.gpu
bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope='module')
def dev():
    return torch.device('cuda:0')


def half_step(t):
    return torch.finfo(t).eps / 2


def weights(E, N, K, group, zeros, s_dtype, seed=0):
    g = torch.Generator().manual_seed(E + N + K + seed)
    lead = (N, ) if E is None else (E, N)
    q = torch.randint(0, 256, lead + (K // 2, ), dtype=torch.uint8, generator=g)
    s = ((0.5 + torch.rand(lead + (K // group, ), generator=g)) * 0.01).to(s_dtype)
    z = torch.randint(0, 16, lead + (K // group, ), dtype=torch.uint8, generator=g) if zeros else None
    return q, s, z


def on(dev, *tensors):
    return [None if t is None else t.to(dev) for t in tensors]


def check(y, x, q, s, z, what):
    ref, bound = orc.w4_gemm(x, q, s, z)
    off = (y.cpu().double() - ref).abs() - (half_step(y.dtype) * (ref.abs() + bound) + bound + torch.finfo(y.dtype).smallest_normal * half_step(y.dtype))
    assert float(off.max()) <= 0, f'{what}: {float(off.max()):.3e} beyond the bound'


SHAPES = [  # M, N, K, group
    (1, 1, 32, 32), (1, 16, 128, 128), (1, 2112, 7168, 128), (2, 17, 64, 64), (3, 33, 96, 32), (5, 100, 160, 32), (7, 48, 1088, 64), (15, 31, 2944, 128), (16, 64, 4096, 64),
    (17, 65, 256, 128), (31, 20, 1056, 32), (32, 96, 512, 128), (33, 40, 704, 64), (64, 130, 1152, 128), (65, 18, 416, 32), (200, 24, 384, 128), (1, 5, 18432, 128),
    # more than 8 MB of weights: tiles that share x, whole and in slices of K, a last chunk that is short
    (3, 4096, 4224, 128), (4, 2049, 8224, 32), (5, 2100, 8320, 64), (16, 1100, 16512, 128), (20, 2048, 9280, 64), (33, 1030, 17152, 128), (64, 9000, 2208, 32),
]


@pytest.mark.parametrize('dtype', [bf16, f16])
@pytest.mark.parametrize('zeros', [False, True])
@pytest.mark.parametrize('M,N,K,group', SHAPES)
def test_product(dev, M, N, K, group, zeros, dtype):
    q, s, z = weights(1, N, K, group, zeros, dtype)
    q, s, z = q[0], s[0], None if z is None else z[0]
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(dtype)
    y = w4_gemm(*on(dev, x, q, s, z))
    assert y.dtype == dtype and tuple(y.shape) == (M, N)
    check(y, x, q, s, z, f'{M}x{N}x{K}/{group}')


@pytest.mark.parametrize('s_dtype', [bf16, f16])
@pytest.mark.parametrize('dtype', [bf16, f16])
def test_types_of_scales(dev, dtype, s_dtype):
    q, s, z = (t[0] for t in weights(1, 70, 320, 64, True, s_dtype))
    x = torch.randn(4, 320, generator=torch.Generator().manual_seed(0)).to(dtype)
    check(w4_gemm(*on(dev, x, q, s, z)), x, q, s, z, f'{dtype} {s_dtype}')


@pytest.mark.parametrize('dtype', [bf16, f16])
def test_every_code_of_every_place(dev, dtype):
    """One column of x at a time picks one code: the results are the weights themselves, exactly."""
    K = 160
    q, s, z = (t[0] for t in weights(1, 48, K, 32, True, f16, seed=9))
    s = torch.full_like(s, 0.5)
    x = torch.eye(K).to(dtype)
    y = w4_gemm(*on(dev, x, q, s, z)).cpu().double()
    assert torch.equal(y, orc.w4_weights(q, s, z).t())
    y = w4_gemm(*on(dev, x, q, s)).cpu().double()
    assert torch.equal(y, orc.w4_weights(q, s, None).t())


def test_rows_where_they_lie(dev):
    q, s, _ = weights(1, 40, 256, 128, False, bf16)
    q, s = q[0], s[0]
    wide = torch.randn(6, 300, generator=torch.Generator().manual_seed(4)).to(bf16)
    for off in (0, 1, 3, 8):
        check(w4_gemm(wide.to(dev)[:, off:off + 256], *on(dev, q, s)), wide[:, off:off + 256], q, s, None, f'offset {off}')
    t = torch.randn(256, 5, generator=torch.Generator().manual_seed(5)).to(bf16)
    check(w4_gemm(t.to(dev).t(), *on(dev, q, s)), t.t(), q, s, None, 'transposed')
    cube = torch.randn(2, 3, 256, generator=torch.Generator().manual_seed(6)).to(bf16)
    y = w4_gemm(cube.to(dev), *on(dev, q, s))
    assert tuple(y.shape) == (2, 3, 40)
    check(y.view(6, 40), cube.view(6, 256), q, s, None, 'three dimensions')
    vec = w4_gemm(cube[0, 0].to(dev), *on(dev, q, s))
    assert tuple(vec.shape) == (40, )
    check(vec.view(1, 40), cube[0, :1], q, s, None, 'a vector')
    one = wide[:1, :256]
    check(w4_gemm(one.to(dev).expand(20, 256), *on(dev, q, s)), one.expand(20, 256), q, s, None, 'broadcast')
    assert tuple(w4_gemm(torch.empty(0, 256, dtype=bf16, device=dev), *on(dev, q, s)).shape) == (0, 40)


def test_numbers_that_are_none_stay_in_their_row(dev):
    q, s, _ = weights(1, 40, 256, 64, False, f16)
    q, s = on(dev, q[0], s[0])
    x = torch.randn(20, 256, device=dev, dtype=f16)
    ref = w4_gemm(x, q, s)
    bad = x.clone()
    bad[3, 7], bad[18, 200] = float('nan'), float('inf')
    y = w4_gemm(bad, q, s)
    keep = torch.ones(20, dtype=torch.bool)
    keep[3] = keep[18] = False
    assert torch.equal(y[keep.to(dev)], ref[keep.to(dev)])
    assert bool(y[3].isnan().all()) and not bool(y[18].isfinite().any())


def ranges(counts, gaps=0):
    start, end, at = [], [], 0
    for c in counts:
        start.append(at)
        end.append(at + c)
        at += c + gaps
    return torch.tensor(start, dtype=torch.int32), torch.tensor(end, dtype=torch.int32), at


@pytest.mark.parametrize('dtype', [bf16, f16])
@pytest.mark.parametrize('counts,gaps,N,K,group,zeros', [
    ([1], 0, 16, 128, 128, False), ([0, 3, 0, 1], 0, 40, 256, 64, True), ([5, 0, 0, 16, 17, 2, 0], 3, 33, 160, 32, True), ([40, 1, 70, 0], 0, 64, 384, 128, False),
    ([1] * 70 + [0] * 70 + [2] * 3, 0, 17, 128, 64, False), ([0, 0, 0], 2, 16, 128, 128, False), ([2] * 8, 1, 96, 2048, 128, True),
    ([3, 0, 20, 1], 1, 1056, 8288, 32, True), ([40, 0, 9, 33, 12], 0, 1000, 4224, 64, False), ([1, 2, 1, 0, 0, 5, 1, 1], 2, 1025, 4480, 128, True),
    ([3, 0, 20, 1], 1, 4105, 544, 32, True), ([1, 2, 1, 0, 0, 5, 1, 1], 0, 5003, 1056, 32, False), ([1] * 12, 0, 2051, 1088, 64, True), ([2, 1, 4, 0] * 4, 2, 4100, 640, 128, False),
])
def test_product_by_expert(dev, counts, gaps, N, K, group, zeros, dtype):
    start, end, rows = ranges(counts, gaps)
    rows = max(rows, 1)
    q, s, z = weights(len(counts), N, K, group, zeros, dtype)
    x = torch.randn(rows, K, generator=torch.Generator().manual_seed(rows)).to(dtype)
    y = w4_gemm_grouped(*on(dev, x, q, s, start, end, z))
    assert y.dtype == dtype and tuple(y.shape) == (rows, N)
    for e, (a, b) in enumerate(zip(start.tolist(), end.tolist())):
        if a < b:
            check(y[a:b], x[a:b], q[e], s[e], None if z is None else z[e], f'expert {e}')


def test_rows_of_no_expert_are_not_written_and_ranges_are_clamped(dev):
    """Through the binding, into an output with a known content; ranges that reach past either end of the rows."""
    from dlblas_amd import _decoder
    q, s, _ = weights(3, 24, 128, 128, False, bf16)
    x = torch.randn(12, 128, generator=torch.Generator().manual_seed(0)).to(bf16)
    start = torch.tensor([-5, 6, 11], dtype=torch.int32)
    end = torch.tensor([2, 6, 1000], dtype=torch.int32)
    y = torch.full((12, 24), 7.0, dtype=bf16, device=dev)
    _decoder.w4_gemm(*on(dev, x, q, s), None, y, *on(dev, start, end), 128)
    y = y.cpu()
    assert bool((y[2:11] == 7).all())
    check(y[:2], x[:2], q[0], s[0], None, 'first')
    check(y[11:], x[11:], q[2], s[2], None, 'last')


@pytest.mark.parametrize('dtype', [bf16, f16])
@pytest.mark.parametrize('group', [32, 64, 128])
@pytest.mark.parametrize('zero_points', [False, True])
@pytest.mark.parametrize('shape', [(1, 128), (7, 384), (3, 5, 256)])
def test_quantiser(dev, shape, group, zero_points, dtype):
    w = torch.randn(*shape, generator=torch.Generator().manual_seed(shape[-1])).to(dtype)
    w[..., :group] = 0
    w[..., group:2 * group] = w[..., group:2 * group].abs()
    q, s, z = per_group_quant_w4(w.to(dev), group, zero_points)
    assert q.dtype == torch.uint8 and s.dtype == dtype and (z is None) == (not zero_points)
    assert tuple(q.shape) == shape[:-1] + (shape[-1] // 2, ) and tuple(s.shape) == shape[:-1] + (shape[-1] // group, )
    g = w.double().reshape(shape[:-1] + (-1, group))
    hi, lo = g.amax(-1).clamp_min(0), g.amin(-1).clamp_max(0)
    want = (hi - lo) / 15 if zero_points else torch.maximum(hi, -lo) / 7
    sc = s.cpu().double()
    assert float(((sc - want).abs() - (half_step(dtype) + 3 * 2.0**-24) * want).max()) <= 0
    zero = torch.full_like(sc, 8.0) if z is None else z.cpu().double()
    codes = orc.w4_codes(q.cpu()).double().reshape(g.shape)
    safe = sc.clamp_min(1e-300)[..., None]
    # nearest code, or the nearest end of the codes; a quotient within fp32's rounding of a border may go to either side
    ideal = (g / safe + zero[..., None]).clamp(0, 15)
    err = torch.where(sc[..., None] > 0, (codes - ideal).abs(), (codes - zero[..., None]).abs())
    assert float(err.max()) <= 0.5 + 16 * 2.0**-23
    if zero_points:
        assert float((zero - torch.where(sc > 0, -lo / sc.clamp_min(1e-300), torch.zeros_like(sc)).clamp(0, 15)).abs().max()) <= 0.5 + 16 * 2.0**-23
    view = torch.zeros(shape[:-1] + (shape[-1] + 5, ), dtype=dtype, device=dev)
    view[..., 3:3 + shape[-1]] = w.to(dev)
    again = per_group_quant_w4(view[..., 3:3 + shape[-1]], group, zero_points)
    assert torch.equal(again[0], q) and torch.equal(again[1], s)


def test_quantised_weights_multiply_like_the_weights(dev):
    """The whole way: |W - W_4| is at most half a scale (7 / 6 of it at the lower end of the symmetric codes is not reached), so a
    product is off by at most sum |x| s / 2 and the rounding."""
    w = torch.randn(64, 512, generator=torch.Generator().manual_seed(1)).to(bf16)
    x = torch.randn(3, 512, generator=torch.Generator().manual_seed(2)).to(bf16)
    for zp in (False, True):
        q, s, z = per_group_quant_w4(w.to(dev), 64, zp)
        y = w4_gemm(x.to(dev), q, s, z).cpu().double()
        # with zero points the range is cut on a grid through zero: a value at its end may lie half a step past the last code
        half = (1.0 if zp else 0.5) * s.cpu().double() * (1 + 2.0**-6)
        bound = x.double().abs().reshape(3, -1, 64).sum(-1) @ half.t()
        ref = x.double() @ w.double().t()
        assert float(((y - ref).abs() - bound - 2.0**-8 * ref.abs() - 1e-3).max()) <= 0


def test_both_paths_give_the_same_bits(dev, monkeypatch):
    q, s, z = on(dev, *weights(3, 40, 256, 64, True, bf16))
    x = torch.randn(20, 256, device=dev, dtype=bf16)
    start, end = on(dev, *ranges([4, 0, 16])[:2])
    calls = lambda: (w4_gemm(x, q[0], s[0], z[0]), w4_gemm(x, q[1], s[1]), w4_gemm(x.view(4, 5, 256), q[1], s[1]), w4_gemm_grouped(x, q, s, start, end, z),
                     w4_gemm_grouped(x, q, s, start, end))
    fast = calls()
    monkeypatch.setattr(mod._fast, 'w4_gemm', lambda *a: None)
    monkeypatch.setattr(mod._fast, 'w4_gemm_grouped', lambda *a: None)
    for a, b in zip(fast, calls()):
        assert a.shape == b.shape and torch.equal(a, b)


def test_native_path_takes_plain_calls_and_registry(dev):
    q, s, z = on(dev, *weights(3, 40, 256, 64, True, bf16))
    x = torch.randn(20, 256, device=dev, dtype=bf16)
    start, end = on(dev, *ranges([4, 0, 16])[:2])
    assert mod._fast.w4_gemm(x, q[0], s[0], None) is not None and mod._fast.w4_gemm_grouped(x, q, s, start, end, z) is not None
    assert torch.equal(dlblas_amd.get_op('w4_gemm', (x, q[0], s[0]))(x, q[0], s[0]), w4_gemm(x, q[0], s[0]))


@pytest.mark.parametrize('zeros', [False, True])
@pytest.mark.parametrize('M,N,K,group', [(20, 3, 288, 32), (33, 1, 544, 32), (17, 2, 320, 64), (40, 129, 96, 32), (3, 8203, 2080, 32), (16, 8195, 2112, 64),
                                         (2, 8193, 2176, 128), (3, 203, 18464, 32), (16, 195, 12352, 64), (2, 193, 9344, 128), (3, 16401, 544, 32), (16, 9003, 608, 32)])
def test_scales_at_the_end_of_their_tensor(dev, M, N, K, group, zeros):
    """A lane reads several scales at once: rows with an odd number of groups, and a last row whose scales are the last bytes there are
    (a NaN behind them would show)."""
    q, s, z = (None if t is None else t[0] for t in weights(1, N, K, group, zeros, bf16))
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(N)).to(bf16)
    room = torch.full((s.numel() + 8, ), float('nan'), dtype=bf16, device=dev)
    sd = room[:s.numel()].view(s.shape).copy_(s)
    qd, zd, xd = on(dev, q, z, x)
    check(w4_gemm(xd, qd, sd, zd), x, q, s, z, f'{M}x{N}x{K}/{group}')
    room = torch.full((s.numel() + 8, ), float('nan'), dtype=bf16, device=dev)
    check(w4_gemm(xd, qd, room[7:7 + s.numel()].view(s.shape).copy_(s), zd), x, q, s, z, f'{M}x{N}x{K}/{group}, other place')


@pytest.mark.parametrize('N,K', [(48, 256), (4105, 544)])
def test_ranges_outside_the_rows_take_no_place(dev, N, K):
    """One row and eight experts: seven ranges name rows that there are not, and only the last one's is there."""
    q, s, _ = weights(8, N, K, 32, False, bf16)
    x = torch.randn(1, K, generator=torch.Generator().manual_seed(8)).to(bf16)
    start = torch.tensor([1, 5, -4, 1000, 2, 3, 1, 0], dtype=torch.int32)
    end = torch.tensor([4, 9, 0, 2000, 3, 9, 2, 1], dtype=torch.int32)
    y = w4_gemm_grouped(*on(dev, x, q, s, start, end))
    check(y, x, q[7], s[7], None, f'{N}x{K}')
