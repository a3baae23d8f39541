"""What ``few_token_experts`` refuses costs no memory: neither the native path nor the Python one allocates for a call that is too large."""
import pytest
import torch

from dlblas_amd.kernels.few_token_experts import few_token_experts

pytestmark = pytest.mark.gpu
bf16, u8, f8 = torch.bfloat16, torch.uint8, torch.float8_e4m3fn


@pytest.mark.parametrize('T,topk,E', [(16384, 8, 2), (64, 17, 2), (8, 2, 1025)])
def test_no_memory_for_what_is_refused(T, topk, E):
    dev = torch.device('cuda:0')
    H = I = 128
    x = torch.zeros(T, H, dtype=bf16, device=dev)
    ids, weights = torch.zeros(T, topk, dtype=torch.int32, device=dev), torch.zeros(T, topk, device=dev)
    w13 = torch.zeros(E, 2 * I, H, dtype=u8, device=dev).view(f8), torch.zeros(E, 2, 1, device=dev)
    w2 = torch.zeros(E, H, I, dtype=u8, device=dev).view(f8), torch.zeros(E, 1, 1, device=dev)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with pytest.raises(ValueError):
        few_token_experts(x, ids, weights, w13, w2)
    assert torch.cuda.max_memory_allocated() == before

