"""What lies between the two products of ``few_token_experts`` is fp32: seen where the parts of a token's slots nearly cancel, so that the rounding of the output, to 16 bits,
hides nothing.

A token names two experts with weights w and -(1 - 2^-14) w.  Their rows have one non-zero column, and those of the second matrix one non-zero weight, so that sums
add zeros but for what is counted here.  M is the magnitude of one slot's part, v w2 with v = w silu(g) u."""
import math

import pytest
import torch

from dlblas_amd.kernels.few_token_experts import few_token_experts
from oracle import mxfp4 as orc

pytestmark = pytest.mark.gpu
bf16, f16, f32, f64, u8, f8 = torch.bfloat16, torch.float16, torch.float32, torch.float64, torch.uint8, torch.float8_e4m3fn
FP32 = orc.FP32


@pytest.fixture(scope='module')
def dev():
    return torch.device('cuda:0')


def half_step(t):
    return torch.finfo(t).eps / 2


def coded(kind, v):
    """Weights that hold the numbers v [E, N, K], multiples of 1/2 up to 2 in magnitude, as the call takes them."""
    E, N, K = v.shape
    if kind == 'f8':
        return v.to(f8), torch.ones(E, -(-N // 128), K // 128)
    code = (2 * v.abs()).to(u8) + 8 * (v < 0).to(u8)  # 0 0.5 1 1.5 2 are codes 0 to 4
    assert torch.equal(orc.values(code[..., ::2] + 16 * code[..., 1::2], torch.full((E, N, K // 32), 127, dtype=u8)), v.double())
    return code[..., ::2] + 16 * code[..., 1::2], torch.full((E, N, K // 32), 127, dtype=u8)


def some(size, g):
    """Non-zero ones of those numbers."""
    return (torch.randint(1, 5, size, generator=g) / 2) * (1 - 2 * torch.randint(0, 2, size, generator=g))


def one_column(E, N, K, values):
    v = torch.zeros(E, N, K)
    v[:, :, 0] = values
    return v


def one_weight(E, H, I, values):
    v = torch.zeros(E, H, I)
    v[:, torch.arange(H), torch.arange(H) % I] = values
    return v


@pytest.mark.parametrize('dtype', [bf16, f16])
@pytest.mark.parametrize('kind', ['f8', 'f4'])
@pytest.mark.parametrize('T', [1, 2, 3, 13, 40])
def test_parts_that_nearly_cancel(dev, T, kind, dtype):
    """v is rounded once per slot (2^-24).  A slot's sum over the columns is one product, cut or rounded where it is put together from parts (2^-23), and two additions of them
    (2^-24 each), both slots' difference is exact: 2 (2^-24 + 2^-23 + 2 2^-24) M = 5 2^-23 M in all, and the half step of what is left.  silu(g) u is the same for both slots, and what it is
    off by, at most 2^-20, counts 2^-14 as much."""
    print(f'case T={T} {kind} {dtype}', flush=True)
    g = torch.Generator().manual_seed(T)
    E, H, I = 2, 512, 384
    rows, down = some((1, 2 * I), g), some((1, H), g)
    x = torch.zeros(T, H)
    x[:, 0] = 1 + torch.rand(T, generator=g)
    x = x.to(dtype)
    w = 1 + torch.rand(T, generator=g)
    weights = torch.stack([w, -w * (1 - 2.0**-14)], 1)
    ids = torch.tensor([[0, 1]]).expand(T, 2).contiguous()
    out = few_token_experts(x.to(dev), ids.to(dev), weights.to(dev), *(tuple(t.to(dev) for t in coded(kind, v)) for v in (one_column(E, 2 * I, H, rows), one_weight(E, H, I, down)))).cpu()
    both = x[:, :1].double() * rows.double()
    a = both[:, :I] / (1 + torch.exp(-both[:, :I])) * both[:, I:]
    part = a[:, torch.arange(H) % I] * down.double()
    want = part * weights.double().sum(1, keepdim=True)
    magnitude = part.abs() * w.double()[:, None]
    off = (out.double() - want).abs() - (5 * 2 * FP32 + 2.0**-34) * magnitude * (1 + half_step(dtype)) - half_step(dtype) * want.abs()
    assert float((off / magnitude).max()) <= 0, f'{float((off / magnitude).max()):.3e} of a part beyond the bound'


@pytest.mark.parametrize('kind', ['f8', 'f4'])
@pytest.mark.parametrize('T', [2, 4, 16, 40])
def test_infinities_and_the_largest_numbers(dev, T, kind):
    """A gate of 2^129 is an infinity, and so is what lies between, of the sign of the other half; the tokens beside it, with numbers up to 2^127, keep theirs to the bit."""
    g = torch.Generator().manual_seed(T)
    E, H, I = 1, 128, 128
    rows, down = torch.zeros(1, 2 * I), some((1, H), g)
    rows[0, 5], rows[0, I + 5] = 2.0, -0.5
    x = torch.zeros(T, H)
    x[:, 0] = 2.0**torch.randint(-3, 64, (T, ), generator=g)
    weight = lambda v: tuple(t.to(dev) for t in coded(kind, v))
    down_all = torch.zeros(E, H, I)
    down_all[:, :, 5] = down
    call = lambda x: few_token_experts(x.to(bf16).to(dev), torch.zeros(T, 1, dtype=torch.int32, device=dev), torch.ones(T, 1, device=dev), weight(one_column(E, 2 * I, H, rows)), weight(down_all)).cpu()
    before = call(x)
    assert bool(before.isfinite().all())
    x[T // 2, 0] = 2.0**127 * 1.5
    out = call(x)
    assert torch.equal(out[T // 2], torch.full((H, ), -math.inf).mul(down[0].sign()).to(bf16))
    others = torch.arange(T) != T // 2
    assert torch.equal(out[others], before[others])


def test_gates_far_below_zero(dev):
    """Of one expert g is -20 ... -84, of the other as near to 0, weighted so that the parts nearly cancel.  exp is off by 2^-23 of itself, whatever its size; the sum with 1, the division, the products
    with u and the weight by 2^-24 each: 3 2^-23 a slot, and what the sums add, as above, 2^-23 + 2 2^-24: 10 2^-23 M for both."""
    g = torch.Generator().manual_seed(2)
    T, H, I = 40, 128, 128
    x = torch.zeros(T, H)
    x[:, 0] = -10 - 32 * torch.rand(T, generator=g)
    x = x.to(bf16)
    gates = torch.tensor([2.0, 2.0**-7])
    rows = torch.ones(2, 2 * I)
    rows[:, :I] = gates[:, None]
    down = some((1, H), g)
    both = x[:, :1].double() * gates.double()  # g of both
    a = both / (1 + torch.exp(-both)) * x[:, :1].double()
    weights = (torch.tensor([1.0, -(1 - 2.0**-12)], dtype=f64) / a).float()
    assert bool(weights.isfinite().all())
    ids = torch.tensor([[0, 1]]).expand(T, 2).contiguous()
    out = few_token_experts(x.to(dev), ids.to(dev), weights.to(dev), *(tuple(t.to(dev) for t in coded('f8', v)) for v in (one_column(2, 2 * I, H, rows), one_weight(2, H, I, down)))).cpu()
    want = (a * weights.double()).sum(1, keepdim=True) * down.double()
    off = (out.double() - want).abs() - 10 * 2 * FP32 * down.double().abs() * (1 + half_step(bf16)) - half_step(bf16) * want.abs()
    assert float(off.max()) <= 0, f'{float(off.max()):.3e} beyond the bound'
