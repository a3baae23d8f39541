"""What the steps around the products refuse, beside tests/test_decoder_steps.py: without a GPU."""
import ctypes

import pytest
import torch

from dlblas_amd import _lib
from dlblas_amd.kernels.moe_permute import MoePermutation, moe_permute, moe_unpermute


@pytest.mark.parametrize('which', ['scales', 'codes', 'both'])
def test_quantised_tokens_have_no_gradient(which):
    """They came back without one where their scales were leaves of a graph."""
    codes, scales = torch.zeros(2, 128, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.ones(2, 1)
    for t, name in ((codes, 'codes'), (scales, 'scales')):
        if which in (name, 'both'):
            t.requires_grad_()
    with pytest.raises(NotImplementedError, match='no gradient'):
        moe_permute((codes, scales), torch.zeros(2, 1, dtype=torch.int32), 4)


def test_the_4_bit_quantiser_takes_the_types_that_scales_have():
    """Its scales have the type of the weights, and no product takes scales in 32 bits."""
    fake, null = ctypes.c_void_p(4096), ctypes.c_void_p(0)
    assert _lib.load().dlb_w4_quant(fake, 256, _lib.IN_CODES[torch.float32], fake, fake, null, 4, 256, 128, null) == _lib.ERR_BAD_DTYPE


def test_a_permutation_of_another_type_has_no_gradient():
    """Its source would be read as int32."""
    p = MoePermutation(torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int64), None, None, None)
    with pytest.raises(TypeError, match='int32'):
        moe_unpermute(torch.zeros(2, 8, requires_grad=True), p)
