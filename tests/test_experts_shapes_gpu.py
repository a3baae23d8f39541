"""The layer of experts for a few tokens with few and with many workgroups, for every number of rows that the first product takes at a time, and experts with one token to more than a
pass of the second; against the definition in 64 bits under its bound."""
import pytest
import torch

from dlblas_amd.kernels.few_token_experts import few_token_experts
from oracle import mxfp4 as orc

pytestmark = pytest.mark.gpu
bf16, f16, u8, f8 = torch.bfloat16, torch.float16, torch.uint8, torch.float8_e4m3fn


@pytest.fixture(scope='module')
def dev():
    return torch.device('cuda:0')


def weights_of(kind, E, N, K, g):
    if kind == 'f4':
        q, s = torch.randint(0, 256, (E, N, K // 2), generator=g, dtype=u8), torch.randint(119, 123, (E, N, K // 32), generator=g, dtype=u8)
        return (q, s), orc.values(q, s)
    q, s = (torch.randn(E, N, K, generator=g) * 60).clamp(-448, 448).to(f8), (0.5 + torch.rand(E, -(-N // 128), K // 128, generator=g)) / (60 * K**0.5)
    return (q, s), orc.e4m3_values(q, s)


@pytest.mark.parametrize('dtype', [bf16, f16])
@pytest.mark.parametrize('kind', ['f8', 'f4'])
@pytest.mark.parametrize('T,E,topk,H,I', [(3, 4, 2, 256, 128), (3, 4, 2, 256, 1664), (7, 4, 2, 384, 1664), (12, 3, 2, 128, 2176), (40, 4, 2, 256, 640), (40, 4, 2, 256, 3328), (64, 2, 1, 128, 6272)])
def test_few_and_many_workgroups(dev, T, E, topk, H, I, kind, dtype):
    print(f'case T={T} E={E} topk={topk} H={H} I={I} {kind} {dtype}', flush=True)
    g = torch.Generator().manual_seed(T + I)
    if kind == 'f4':
        H, I = H + 32, I - 32
    x = torch.randn(T, H, generator=g).to(dtype)
    (up, w13), (down, w2) = weights_of(kind, E, 2 * I, H, g), weights_of(kind, E, H, I, g)
    ids = torch.stack([torch.randperm(E + 1, generator=g)[:topk] for _ in range(T)])  # expert E is elsewhere
    weights = torch.rand(T, topk, generator=g)
    put = lambda v: tuple(t.to(dev) for t in v)
    out = few_token_experts(x.to(dev), ids.to(dev), weights.to(dev), put(up), put(down))
    want, bound = orc.experts(x, ids, weights, w13, w2)
    step = torch.finfo(dtype).eps / 2
    off = (out.cpu().double() - want).abs() - (step * want.abs() + bound * (1 + step) + torch.finfo(dtype).smallest_normal * step)
    assert float(off.max()) <= 0, f'{float(off.max()):.3e} beyond the bound'
