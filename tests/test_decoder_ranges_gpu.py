"""The row ranges that moe_permute leaves, read by the FP8 products on row ranges: spans that begin at any row, experts without one."""
import pytest
import torch

import helpers
from dlblas_amd import _lib
from dlblas_amd.kernels.fp8_gemm_grouped import m_grouped_fp8_gemm_nt_contiguous
from dlblas_amd.kernels.moe_permute import moe_permute
from oracle import fp8_block_gemm as orc

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def dev():
    return torch.device('cuda:0')


@pytest.mark.parametrize('alignment', [1, 16, 128])
@pytest.mark.parametrize('T,K,N,E,topk', [(1, 512, 256, 8, 2), (33, 512, 384, 8, 2), (40, 1024, 256, 40, 8)])
def test_products_on_the_ranges_of_the_permutation(dev, T, K, N, E, topk, alignment):
    """Row by row the bits of the expert-contiguous product on 128-row spans; rows of no slot keep what they hold."""
    g = helpers.gen(T + K)
    q, s = (t.to(dev) for t in orc.quant_act_1x128(torch.randn(T, K, generator=g).to(torch.bfloat16)))
    weights = [orc.quant_weight_128x128((torch.randn(N, K, generator=g) * 0.05).to(torch.bfloat16)) for _ in range(3)]
    w, w_s = (torch.stack([weights[e % 3][i] for e in range(E)]).to(dev) for i in (0, 1))
    ids = torch.randint(-1, E - 1, (T, topk), generator=g).to(dev)  # the last expert has none
    (rows, rows_s), p = moe_permute((q, s), ids, E, alignment)
    out = torch.full((rows.size(0), N), -7.0, dtype=torch.bfloat16, device=dev)
    assert _lib.gemm_ragged(rows, w, rows_s, w_s, out, p.row_start, p.row_end, max(1, T * topk // E))
    whole, pw = moe_permute((q, s), ids, E, 128)
    ref = torch.zeros(whole[0].size(0), N, dtype=torch.bfloat16, device=dev)
    m_grouped_fp8_gemm_nt_contiguous(whole, (w, w_s), ref, pw.m_indices)
    here = p.row_index >= 0
    assert torch.equal(here, pw.row_index >= 0) and torch.equal(here, ids >= 0)
    assert torch.equal(out[p.row_index[here].long()], ref[pw.row_index[here].long()])
    assert bool((out[p.source < 0] == -7).all())
