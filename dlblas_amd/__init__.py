"""MI355X-native FP8 block-scaled GEMM behind DLBlas' entry points.

    from dlblas_amd.kernels.fp8_gemm import fp8_gemm            # dlblas.kernels.fp8_gemm.fp8_gemm
    from dlblas_amd import get_op                                # dlblas.get_op / dlblas.utils.get_op
    op = get_op('fp8_gemm', (a, b, a_s, b_s)); c = op(a, b, a_s, b_s)

``dlblas_amd.compat.install()`` additionally publishes the same modules under the ``dlblas`` and ``deep_gemm``
names for code that imports those.
"""
from . import kernels  # noqa: F401  (registers the ops)
from ._lib import prepare
from .kernels.few_token_experts import few_token_experts
from .kernels.fp8 import per_token_group_quant_fp8
from .kernels.fp8_gemm import fp8_gemm
from .kernels.fp8_gemm_grouped import (fp8_gemm_grouped_contiguous, fp8_gemm_grouped_masked,
                                       m_grouped_fp8_gemm_nt_contiguous, m_grouped_fp8_gemm_nt_masked)
from .kernels.layer_norm import layer_norm
from .kernels.moe_permute import MoePermutation, moe_permute, moe_unpermute
from .kernels.mxfp4_gemm import mxfp4_gemm, mxfp4_weight_gemm, per_group_quant_mxfp4
from .kernels.rms_norm import rms_norm, rms_norm_quant
from .kernels.w4_gemm import per_group_quant_w4, w4_gemm, w4_gemm_grouped
from .utils import get_args_from_op_name, get_list_op_names, get_op, register_dlblas_op

__version__ = '0.1.0'

__all__ = [
    'fp8_gemm', 'prepare', 'per_token_group_quant_fp8', 'fp8_gemm_grouped_contiguous', 'fp8_gemm_grouped_masked', 'm_grouped_fp8_gemm_nt_contiguous',
    'm_grouped_fp8_gemm_nt_masked', 'rms_norm', 'rms_norm_quant', 'layer_norm', 'MoePermutation', 'moe_permute', 'moe_unpermute', 'w4_gemm', 'w4_gemm_grouped',
    'per_group_quant_w4', 'mxfp4_gemm', 'mxfp4_weight_gemm',
    'per_group_quant_mxfp4', 'few_token_experts', 'get_op', 'get_list_op_names', 'get_args_from_op_name', 'register_dlblas_op'
]
