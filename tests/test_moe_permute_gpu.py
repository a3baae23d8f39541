"""Tokens sorted by expert and back: tables and copies exactly, sums and gradients against the definitions in 64 bits.

Tolerances, u = half a step of the stored type: the FMA chain over the slots of a token is off by 2^-24 of the magnitudes of its terms per
slot; the product of a row and a gradient has at most 32 terms a lane, 6 steps over the wave and 16 waves: below 60 * 2^-24."""
import pytest
import torch

from dlblas_amd.kernels import moe_permute as mod
from dlblas_amd.kernels.fp8 import per_token_group_quant_fp8
from dlblas_amd.kernels.moe_permute import MoePermutation, moe_permute, moe_unpermute
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
    return torch.finfo(t).smallest_normal * half_step(t)


def routing(T, topk, E, seed=0, elsewhere=0.25, dtype=torch.int32):
    """Ids of all kinds: experts here, -1, beyond the last, and the same expert twice in a token."""
    g = torch.Generator().manual_seed(100 * T + 10 * topk + E + seed)
    ids = torch.randint(0, E, (T, topk), generator=g)
    off = torch.rand(T, topk, generator=g) < elsewhere
    far = torch.where(torch.rand(T, topk, generator=g) < 0.5, torch.full_like(ids, -1), ids + E)
    return torch.where(off, far, ids).to(dtype)


def tables_equal(p, ref):
    for name, got, want in zip(MoePermutation._fields, p, ref):
        assert got.dtype == torch.int32 and torch.equal(got.cpu(), want), name


CASES = [  # T, topk, E, alignment, H
    (1, 1, 1, 1, 8), (1, 8, 32, 1, 64), (3, 2, 4, 16, 33), (16, 8, 32, 1, 256), (17, 3, 5, 128, 1), (128, 8, 8, 1, 40), (129, 8, 256, 1, 72),
    (400, 5, 3, 7, 96), (1024, 1, 64, 16, 17), (1025, 1, 64, 1, 128), (700, 6, 160, 128, 50), (5000, 2, 1024, 1, 24), (2, 64, 6, 4, 31),
]


@pytest.mark.parametrize('dtype', [bf16, f16, f32])
@pytest.mark.parametrize('T,topk,E,alignment,H', CASES)
def test_permute(dev, T, topk, E, alignment, H, dtype):
    ids = routing(T, topk, E)
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(T)).to(dtype)
    rows, p = moe_permute(x.to(dev), ids.to(dev), E, alignment)
    ref = orc.sort_tables(ids, E, alignment, rows.size(0))
    tables_equal(p, ref)
    assert torch.equal(rows.cpu(), orc.permute(x, ref[1], topk))


@pytest.mark.parametrize('T,topk,E,alignment', [(40, 4, 8, 1), (40, 4, 8, 16), (600, 4, 8, 128)])
@pytest.mark.parametrize('share', [0, 1, 7, 8, 13])
def test_rows_that_find_no_room(dev, T, topk, E, alignment, share):
    """num_rows cuts the order anywhere: slots behind it are dropped, the ranges end at it."""
    ids = routing(T, topk, E, elsewhere=0.0)
    full = int(orc.sort_tables(ids, E, alignment, 1 << 14)[4].max())
    n = full * share // 8
    x = torch.randn(T, 24, generator=torch.Generator().manual_seed(1)).to(bf16)
    rows, p = moe_permute(x.to(dev), ids.to(dev), E, alignment, num_rows=n)
    ref = orc.sort_tables(ids, E, alignment, n)
    tables_equal(p, ref)
    assert torch.equal(rows.cpu(), orc.permute(x, ref[1], topk))
    out = moe_unpermute(rows, p)
    sums, mag = orc.unpermute(rows.cpu(), ref[0], None)
    assert float(((out.cpu().double() - sums).abs() - half_step(bf16) * sums.abs() - topk * FP32 * mag).max()) <= 0


def test_ids_in_any_layout(dev):
    ids = routing(37, 6, 9)
    x = torch.randn(37, 16).to(bf16).to(dev)
    ref = orc.sort_tables(ids, 9, 1, 37 * 6)
    wide = torch.zeros(37, 13, dtype=torch.int32)
    wide[:, 1::2] = ids
    for given in (ids.long().to(dev), ids.t().contiguous().to(dev).t(), wide.to(dev)[:, 1::2], torch.full((37, 6), 2**40) * (ids.long() < 0) + ids.long().clamp_min(0)):
        rows, p = moe_permute(x, given.to(dev), 9)
        if given.dtype == torch.int64 and int(given.max()) > 2**32:  # an id whose low half would be an expert
            assert torch.equal(p.row_index.cpu() < 0, (given.cpu() >= 9))
            continue
        tables_equal(p, ref)
    one = torch.tensor([[3]], dtype=torch.int32).expand(37, 6)
    tables_equal(moe_permute(x, one.to(dev), 9)[1], orc.sort_tables(one, 9, 1, 37 * 6))


def test_no_tokens_no_experts_here(dev):
    x = torch.randn(0, 16, device=dev, dtype=bf16)
    rows, p = moe_permute(x, torch.zeros(0, 2, dtype=torch.int32, device=dev), 4)
    assert rows.shape == (0, 16) and p.row_index.shape == (0, 2) and p.row_start.tolist() == [0] * 4 and p.row_end.tolist() == [0] * 4
    assert moe_unpermute(rows, p).shape == (0, 16)
    x = torch.randn(5, 16, device=dev, dtype=bf16)
    rows, p = moe_permute(x, torch.full((5, 2), -1, device=dev), 4, num_rows=6)
    assert float(rows.abs().max()) == 0 and p.source.tolist() == [-1] * 6 and p.m_indices.tolist() == [-1] * 6
    assert float(moe_unpermute(rows, p).abs().max()) == 0
    rows, p = moe_permute(torch.randn(0, 16, device=dev, dtype=bf16), torch.zeros(0, 2, dtype=torch.int32, device=dev), 4, num_rows=3)
    assert float(rows.abs().max()) == 0 and p.source.tolist() == [-1] * 3
    rows, p = moe_permute(x, torch.zeros(5, 1, dtype=torch.int32, device=dev), 4, num_rows=0)
    assert rows.shape == (0, 16) and p.row_index.flatten().tolist() == [-1] * 5 and float(moe_unpermute(rows, p).abs().max()) == 0


@pytest.mark.parametrize('dtype', [bf16, f32])
def test_rows_where_they_lie(dev, dtype):
    """Tokens in a wider tensor at any element offset, transposed and broadcast ones."""
    ids = routing(11, 3, 4)
    wide = torch.randn(11, 80, generator=torch.Generator().manual_seed(2)).to(dtype)
    ref = orc.sort_tables(ids, 4, 1, 33)
    for off in (0, 1, 2, 3, 8):
        rows, p = moe_permute(wide.to(dev)[:, off:off + 70], ids.to(dev), 4)
        assert torch.equal(rows.cpu(), orc.permute(wide[:, off:off + 70], ref[1], 3))
        out = moe_unpermute(torch.cat([rows, rows], 1)[:, off:off + 70], p)
        sums, mag = orc.unpermute(torch.cat([rows, rows], 1)[:, off:off + 70].cpu(), ref[0], None)
        assert float(((out.cpu().double() - sums).abs() - half_step(dtype) * sums.abs() - 3 * FP32 * mag).max()) <= 0
    t = wide.t().contiguous()
    rows, _ = moe_permute(t.to(dev).t(), ids.to(dev), 4)
    assert torch.equal(rows.cpu(), orc.permute(wide, ref[1], 3))
    rows, _ = moe_permute(wide[:1].to(dev).expand(11, 80), ids.to(dev), 4)
    assert torch.equal(rows.cpu(), orc.permute(wide[:1].expand(11, 80), ref[1], 3))


@pytest.mark.parametrize('T,H,alignment', [(1, 128, 1), (33, 256, 16), (150, 1152, 128)])
@pytest.mark.parametrize('column_major', [False, True])
def test_quantised_tokens(dev, T, H, alignment, column_major):
    ids = routing(T, 4, 6)
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(3)).to(bf16).to(dev)
    q, s = per_token_group_quant_fp8(x, 128, column_major_scales=column_major)
    (rows, rows_s), p = moe_permute((q, s), ids.to(dev), 6, alignment)
    ref = orc.sort_tables(ids, 6, alignment, rows.size(0))
    tables_equal(p, ref)
    assert torch.equal(rows.view(torch.uint8).cpu(), orc.permute(q.view(torch.uint8).cpu(), ref[1], 4))
    assert torch.equal(rows_s.cpu(), orc.permute(s.cpu(), ref[1], 4))
    # rows that are not on 16 bytes
    wide = torch.zeros(T, H + 24, dtype=torch.uint8, device=dev)
    wide[:, 3:3 + H] = q.view(torch.uint8)
    (rows2, _), _ = moe_permute((wide[:, 3:3 + H].view(torch.float8_e4m3fn), s), ids.to(dev), 6, alignment)
    assert torch.equal(rows2.view(torch.uint8), rows.view(torch.uint8))


@pytest.mark.parametrize('dtype', [bf16, f16, f32])
@pytest.mark.parametrize('weighted', [False, True])
@pytest.mark.parametrize('T,topk,E,alignment,H', CASES)
def test_unpermute(dev, T, topk, E, alignment, H, weighted, dtype):
    ids = routing(T, topk, E, seed=1)
    n = T * topk + E * alignment
    ref = orc.sort_tables(ids, E, alignment, n)
    g = torch.Generator().manual_seed(T)
    rows = torch.randn(n, H, generator=g).to(dtype)
    rows[ref[1] < 0] = float('nan')  # never read
    w = torch.randn(T, topk, generator=g) if weighted else None
    out = moe_unpermute(rows.to(dev), ref[0].to(dev), None if w is None else w.to(dev))
    sums, mag = orc.unpermute(rows, ref[0], w)
    off = (out.cpu().double() - sums).abs() - (half_step(dtype) * sums.abs() + (topk + 1) * FP32 * mag + tiny(dtype))
    assert float(off.max()) <= 0


def test_table_entries_outside_the_rows_name_none(dev):
    rows = torch.randn(5, 8, device=dev)
    table = torch.tensor([[0, 7], [-3, 4], [5, 2**31 - 1], [1, 1]], dtype=torch.int32, device=dev)
    out = moe_unpermute(rows, table)
    assert torch.equal(out, torch.stack([rows[0], rows[4], torch.zeros_like(rows[0]), rows[1] + rows[1]]))


@pytest.mark.parametrize('dtype', [bf16, f16, f32])
@pytest.mark.parametrize('T,topk,E,alignment,H', CASES + [(9, 4, 5, 16, 7168), (3, 2, 4, 1, 9001)])
def test_gradients(dev, T, topk, E, alignment, H, dtype):
    ids = routing(T, topk, E, seed=2)
    g = torch.Generator().manual_seed(T + H)
    x, dout = (torch.randn(T, H, generator=g).to(dtype) for _ in range(2))
    w = torch.randn(T, topk, generator=g)
    xl, wl = x.to(dev).requires_grad_(), w.to(dev).requires_grad_()
    rows, p = moe_permute(xl, ids.to(dev), E, alignment)
    out = moe_unpermute(rows, p, wl)
    drows, dw = torch.autograd.grad([out], [rows, wl], [dout.to(dev)], retain_graph=True)
    dx, = torch.autograd.grad([out], [xl], [dout.to(dev)])
    row_index, source = (t.cpu() for t in p[:2])
    # a row's gradient is one fp32 product, rounded
    there = source >= 0
    want = torch.zeros(rows.shape, dtype=dtype)
    slot = source[there].long()
    want[there] = (w.flatten()[slot, None] * dout[slot // topk].float()).to(dtype)
    assert torch.equal(drows.cpu(), want)
    sums, mag = orc.unpermute(want, row_index, None)
    assert float(((dx.cpu().double() - sums).abs() - half_step(dtype) * sums.abs() - topk * FP32 * mag - tiny(dtype)).max()) <= 0
    terms = torch.zeros(T, topk, H, dtype=torch.float64)
    here = row_index >= 0
    terms[here] = rows.detach().cpu().double()[row_index[here].long()] * dout.double()[:, None].expand(T, topk, H)[here]
    assert float(((dw.cpu().double() - terms.sum(-1)).abs() - 60 * FP32 * terms.abs().sum(-1)).max()) <= 0
    assert bool((dw.cpu()[~here] == 0).all())
    sums, mag = orc.unpermute(rows.detach().cpu(), row_index, w)
    assert float(((out.detach().cpu().double() - sums).abs() - half_step(dtype) * sums.abs() - (topk + 1) * FP32 * mag - tiny(dtype)).max()) <= 0


def test_gradients_by_differences(dev):
    """The sum over a token's slots is linear in the rows and in the weights, so a difference over any step is the derivative: off by the
    roundings of fp32 alone, 64 * 5 * 24 terms of size one at 2^-24 of a few."""
    T, topk, E, H = 24, 5, 6, 64
    ids = routing(T, topk, E, seed=3).to(dev)
    g = torch.Generator().manual_seed(1)
    x, ex, d = (torch.randn(T, H, generator=g).to(dev) for _ in range(3))
    w, ew = (torch.randn(T, topk, generator=g).to(dev) for _ in range(2))
    xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()

    def value(a, b):
        rows, p = moe_permute(a, ids, E, 4)
        return moe_unpermute(rows, p, b)

    dx, dw = torch.autograd.grad([value(xl, wl)], [xl, wl], [d])
    loss = lambda a, b: float((value(a, b).double() * d.double()).sum())
    assert abs((loss(x + ex, w) - loss(x - ex, w)) / 2 - float((dx.double() * ex.double()).sum())) < 0.02
    assert abs((loss(x, w + ew) - loss(x, w - ew)) / 2 - float((dw.double() * ew.double()).sum())) < 0.02


def test_gradients_that_are_not_asked_for_and_layouts(dev):
    T, topk, E, H = 20, 3, 4, 48
    ids = routing(T, topk, E, seed=4).to(dev)
    x = torch.randn(T, H, device=dev, dtype=bf16)
    w = torch.randn(T, topk, device=dev)
    rows, p = moe_permute(x, ids, E)
    dout = torch.randn(T, H, device=dev, dtype=bf16)
    rl, wl = rows.clone().requires_grad_(), w.clone().requires_grad_()
    both = torch.autograd.grad(moe_unpermute(rl, p, wl), [rl, wl], [dout])
    assert torch.equal(torch.autograd.grad(moe_unpermute(rl, p, w), [rl], [dout])[0], both[0])
    assert torch.equal(torch.autograd.grad(moe_unpermute(rows, p, wl), [wl], [dout])[0], both[1])
    plain, = torch.autograd.grad(moe_unpermute(rl, p), [rl], [dout])
    ones, = torch.autograd.grad(moe_unpermute(rl, p, torch.ones_like(w)), [rl], [dout])
    assert torch.equal(plain, ones)
    # weights and gradients in other layouts: transposed, broadcast
    wt = w.t().contiguous().t().requires_grad_()
    other = torch.autograd.grad(moe_unpermute(rl, p, wt), [rl, wt], [dout.t().contiguous().t()])
    assert torch.equal(other[0], both[0]) and torch.equal(other[1], both[1])
    s1, = torch.autograd.grad(moe_unpermute(rl, p, w).sum(), [rl])
    s2, = torch.autograd.grad(moe_unpermute(rl, p, w), [rl], [torch.ones_like(dout)])
    assert torch.equal(s1, s2)
    wide = torch.randn(rows.size(0), H + 5, device=dev, dtype=bf16)
    cut = wide[:, 3:3 + H].detach().requires_grad_()
    a = torch.autograd.grad(moe_unpermute(cut, p, wl), [cut, wl], [dout])
    whole = wide[:, 3:3 + H].contiguous().requires_grad_()
    b = torch.autograd.grad(moe_unpermute(whole, p, wl), [whole, wl], [dout])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_both_paths_give_the_same_bits(dev, monkeypatch):
    ids = routing(50, 4, 7).to(dev)
    x = torch.randn(50, 256, device=dev, dtype=bf16)
    q = per_token_group_quant_fp8(x, 128)
    w = torch.randn(50, 4, device=dev)

    def calls():
        rows, p = moe_permute(x, ids, 7, 16)
        (f, s), p2 = moe_permute(q, ids, 7, 1, 150)
        return (rows, f.view(torch.uint8), s, moe_unpermute(rows, p, w), moe_unpermute(rows, p.row_index)) + tuple(p) + tuple(p2)

    fast = calls()
    monkeypatch.setattr(mod._fast, 'moe_permute', lambda *a: None)
    monkeypatch.setattr(mod._fast, 'moe_unpermute', lambda *a: None)
    for a, b in zip(fast, calls()):
        assert a.shape == b.shape and torch.equal(a, b)


def test_native_path_takes_plain_calls(dev):
    x = torch.randn(5, 128, device=dev, dtype=bf16)
    ids = torch.zeros(5, 2, dtype=torch.int64, device=dev)
    assert mod._fast.moe_permute(x, None, ids, 4, 1, None) is not None
    assert mod._fast.moe_permute(*per_token_group_quant_fp8(x, 128), ids, 4, 128, 256) is not None
    assert mod._fast.moe_unpermute(x, ids.int(), None, None) is not None
    w = torch.ones(5, 2, device=dev, requires_grad=True)
    assert mod._fast.moe_unpermute(x, ids.int(), w, None) is None  # no gradient from a table alone
    rows, p = moe_permute(x, ids, 4)
    assert mod._fast.moe_unpermute(rows, p.row_index, w, p.source).grad_fn is not None
    assert mod._fast.moe_permute(x.requires_grad_(), None, ids, 4, 1, None)[0].grad_fn is not None


def test_gradients_are_those_of_the_python_path(dev, monkeypatch):
    T, topk, E, H = 30, 3, 4, 72
    ids = routing(T, topk, E, seed=5).to(dev)
    x, dout = (torch.randn(T, H, device=dev, dtype=bf16) for _ in range(2))
    w = torch.randn(T, topk, device=dev)

    def passes():
        xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
        rows, p = moe_permute(xl, ids, E, 8)
        out = moe_unpermute(rows, p, wl)
        return (out, ) + torch.autograd.grad([out], [xl, wl], [dout])

    fast = passes()
    monkeypatch.setattr(mod._fast, 'moe_permute', lambda *a: None)
    monkeypatch.setattr(mod._fast, 'moe_unpermute', lambda *a: None)
    for a, b in zip(fast, passes()):
        assert torch.equal(a, b)


def test_a_second_derivative_raises(dev):
    ids = routing(6, 2, 3).to(dev)
    x = torch.randn(6, 16, device=dev).requires_grad_()
    w = torch.randn(6, 2, device=dev).requires_grad_()
    rows, p = moe_permute(x, ids, 3)
    dx, dw = torch.autograd.grad([moe_unpermute(rows, p, w).sum()], [x, w], create_graph=True)
    with pytest.raises(RuntimeError):
        (dx.sum() + dw.sum()).backward()
