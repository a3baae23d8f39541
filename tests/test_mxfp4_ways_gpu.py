"""Every kernel that ``mxfp4_gemm`` chooses from, with scales over the whole range, scales that are no numbers and all three types of output, against the definition in 64 bits: sums over
K / 32 groups take at most K / 32 + 8 additions, each off by at most 2^-23 of the sum of magnitudes, then half a step of the stored type.

Where a row of scales ends inside the window that a kernel reads, what follows are the next row's: finite ones meet codes of zero and would not show."""
import pytest
import torch

from dlblas_amd import _lib
from dlblas_amd.kernels.few_token_experts import few_token_experts
from dlblas_amd.kernels.moe_permute import moe_permute, moe_unpermute
from dlblas_amd.kernels.mxfp4_gemm import mxfp4_gemm, per_group_quant_mxfp4
from oracle import mxfp4 as orc

pytestmark = pytest.mark.gpu
bf16, f16, f32, u8 = torch.bfloat16, torch.float16, torch.float32, torch.uint8

SPLIT, TILES_64, TILES_128, TILES_256 = 'split', '64', '128', '256'
# rows and columns that get to each, with rows and columns off the tiles
EXTENTS = [(3, 40, SPLIT), (20, 200, SPLIT), (50, 6500, SPLIT), (200, 2100, TILES_64), (1000, 2900, TILES_128), (2100, 3801, TILES_256)]
# 12 groups (whole words, three quarters of a window of 16), 13 (laid out anew for the largest tiles), 33, 35, 36 and 48 (whole windows)
COLUMNS = [384, 416, 1056, 1120, 1152, 1536]


def way(M, N):
    """The rule of the C entry point, by the numbers of tiles."""
    tiles = lambda size: -(-M // size) * -(-N // size)
    if M <= 64 or tiles(32) <= 256:
        return SPLIT
    return TILES_64 if tiles(64) <= 512 else TILES_256 if tiles(256) >= 128 else TILES_128


@pytest.fixture(scope='module')
def dev():
    return torch.device('cuda:0')


@pytest.fixture(scope='module', autouse=True)
def ways():
    for M, N, name in EXTENTS:
        assert way(M, N) == name
        # scratch for scales of 13 groups: the largest tiles alone
        assert (_lib.load().dlb_mxfp4_gemm_workspace_bytes(M, N, 416) > 0) == (name == TILES_256)


def operand(rows, K, g, low, high):
    return torch.randint(0, 256, (rows, K // 2), generator=g, dtype=u8), torch.randint(low, high, (rows, K // 32), generator=g, dtype=u8)


def inside(c, a, a_s, b, b_s, K, dev, what):
    """On the device."""
    x, w = orc.values(a, a_s).to(dev), orc.values(b, b_s).to(dev)
    want, mag = x @ w.t(), x.abs() @ w.abs().t()
    step = torch.finfo(c.dtype).eps / 2
    off = (c.double() - want).abs() - (step * want.abs() + (K // 32 + 8) * 2 * orc.FP32 * mag * (1 + step) + torch.finfo(c.dtype).smallest_normal * step)
    assert float(off.max()) <= 0, f'{what}: {float(off.max()):.3e} beyond the bound'


@pytest.mark.parametrize('K', COLUMNS)
@pytest.mark.parametrize('M,N,name', EXTENTS)
def test_scales_over_the_whole_range(dev, M, N, name, K):
    print(f'case {name} {M}x{N}x{K}', flush=True)
    g = torch.Generator().manual_seed(M + K)
    (a, a_s), (b, b_s) = operand(M, K, g, 77, 177), operand(N, K, g, 77, 177)
    inside(mxfp4_gemm(*(t.to(dev) for t in (a, b, a_s, b_s)), f32), a, a_s, b, b_s, K, dev, name)


@pytest.mark.parametrize('out', [bf16, f16])
@pytest.mark.parametrize('M,N,name', EXTENTS)
def test_types_of_output(dev, M, N, name, out):
    g = torch.Generator().manual_seed(M)
    for K in (384, 416):
        (a, a_s), (b, b_s) = operand(M, K, g, 121, 128), operand(N, K, g, 121, 128)
        c = mxfp4_gemm(*(t.to(dev) for t in (a, b, a_s, b_s)), out)
        assert c.dtype == out
        inside(c, a, a_s, b, b_s, K, dev, f'{name} {out}')


@pytest.mark.parametrize('K', COLUMNS)
@pytest.mark.parametrize('M,N,name', EXTENTS)
def test_scales_that_are_no_numbers(dev, M, N, name, K):
    """In the first group of some rows and columns, behind which the windows of those in front end, and in the last of others; beside codes of zero."""
    print(f'case {name} {M}x{N}x{K}', flush=True)
    g = torch.Generator().manual_seed(M + K)
    (a, a_s), (b, b_s) = operand(M, K, g, 120, 130), operand(N, K, g, 120, 130)
    rows, cols = sorted({1, M // 2, M - 1}), sorted({2, N // 3, N - 1})
    nan = torch.zeros(M, N, dtype=torch.bool)
    for i, m in enumerate(rows):
        a_s[m, 0 if i < 2 else -1] = 255
        a[m] = 0 if i == 0 else a[m]
        nan[m] = True
    for i, n in enumerate(cols):
        b_s[n, 0 if i < 2 else -1] = 255
        b[n] = 0 if i == 0 else b[n]
        nan[:, n] = True
    c = mxfp4_gemm(*(t.to(dev) for t in (a, b, a_s, b_s)), f32)
    assert torch.equal(c.isnan().cpu(), nan)
    kept_rows, kept_cols = [torch.tensor([i for i in range(n) if i not in out]) for n, out in ((M, rows), (N, cols))]
    inside(c[kept_rows.to(dev)][:, kept_cols.to(dev)], a[kept_rows], a_s[kept_rows], b[kept_cols], b_s[kept_cols], K, dev, name)


def test_prompts_of_4_bit_experts_one_after_the_other(dev):
    """What is left for more tokens than ``few_token_experts`` takes: rows by expert, and products of two 4-bit operands on each expert's.  Against the definition on the values that were multiplied last."""
    g = torch.Generator().manual_seed(9)
    T, E, topk, H, I = 300, 4, 2, 256, 128
    x = torch.randn(T, H, generator=g).to(bf16).to(dev)
    ids = torch.stack([torch.randperm(E, generator=g)[:topk] for _ in range(T)]).to(torch.int32).to(dev)
    weights = torch.rand(T, topk, generator=g).to(dev)
    w13, w2 = ((torch.randint(0, 256, (E, n, k // 2), generator=g, dtype=u8).to(dev), torch.randint(118, 124, (E, n, k // 32), generator=g, dtype=u8).to(dev)) for n, k in ((2 * I, H), (H, I)))
    with pytest.raises(ValueError, match='mxfp4_gemm'):
        few_token_experts(x, ids, weights, w13, w2)
    rows, perm = moe_permute(x, ids, E)
    down = torch.zeros(rows.shape[0], H, dtype=bf16, device=dev)
    exact = torch.zeros(rows.shape[0], H, dtype=torch.float64)
    for e, (start, end) in enumerate(zip(perm.row_start.tolist(), perm.row_end.tolist())):
        q, s = per_group_quant_mxfp4(rows[start:end])
        both = mxfp4_gemm(q, w13[0][e], s, w13[1][e], f32)
        mid, mid_s = per_group_quant_mxfp4(torch.nn.functional.silu(both[:, :I]) * both[:, I:])
        down[start:end] = mxfp4_gemm(mid, w2[0][e], mid_s, w2[1][e], bf16)
        exact[start:end] = orc.values(mid.cpu(), mid_s.cpu()) @ orc.values(w2[0][e].cpu(), w2[1][e].cpu()).t()
    out = moe_unpermute(down, perm, weights).cpu().double()
    parts = exact[perm.row_index.cpu().long()] * weights.cpu().double()[:, :, None]
    # every part rounded to bf16, their sum once more; in between a dozen roundings of fp32
    step = torch.finfo(bf16).eps / 2
    assert bool(((out - parts.sum(1)).abs() <= step * parts.sum(1).abs() + (step + 16 * orc.FP32) * (1 + step) * parts.abs().sum(1)).all())
