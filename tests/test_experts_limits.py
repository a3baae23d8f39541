"""The limit of ``few_token_experts`` on the numbers between its products: header and binding, and its refusal without a GPU."""
import os
import re

import pytest
import torch

from dlblas_amd import _mxfp4
from dlblas_amd.kernels.few_token_experts import few_token_experts

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'include', 'dlblas_mxfp4.h')


def test_header_and_binding_agree():
    assert re.search(r'#define DLB_FEW_NUMBERS \(1 << 29\)', open(HEADER).read()) and _mxfp4.FEW_NUMBERS == 1 << 29


def test_too_many_numbers_between_the_products():
    meta = lambda *size, dtype: torch.empty(size, dtype=dtype, device='meta')
    T, topk, H, I = 64, 16, 32, (1 << 19) + 32
    u8 = torch.uint8
    with pytest.raises(ValueError, match='tokens'):
        few_token_experts(meta(T, H, dtype=torch.bfloat16), meta(T, topk, dtype=torch.int32), meta(T, topk, dtype=torch.float32), (meta(1, 2 * I, H // 2, dtype=u8), meta(1, 2 * I, H // 32, dtype=u8)),
                          (meta(1, H, I // 2, dtype=u8), meta(1, H, I // 32, dtype=u8)))


@pytest.mark.parametrize('bits', [8, 4])
def test_a_prompt_is_sent_to_a_call_that_takes_its_weights(bits):
    T, topk, E, H, I = 65, 2, 4, 256, 128
    zeros = lambda *size, dtype: torch.zeros(size, dtype=dtype)
    if bits == 4:
        w13, w2 = ((zeros(E, n, k // 2, dtype=torch.uint8), zeros(E, n, k // 32, dtype=torch.uint8)) for n, k in ((2 * I, H), (H, I)))
    else:
        w13, w2 = ((zeros(E, n, k, dtype=torch.uint8).view(torch.float8_e4m3fn), zeros(E, n // 128, k // 128, dtype=torch.float32)) for n, k in ((2 * I, H), (H, I)))
    with pytest.raises(ValueError, match='fused_moe_v3' if bits == 8 else 'mxfp4_gemm'):
        few_token_experts(zeros(T, H, dtype=torch.bfloat16), zeros(T, topk, dtype=torch.int32), zeros(T, topk, dtype=torch.float32), w13, w2)
