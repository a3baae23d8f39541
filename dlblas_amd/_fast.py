"""The entry points as native calls (csrc/host_calls.cpp, host_steps.cpp): ``_fast.fp8_gemm(a, b, a_s, b_s)`` and so on return the result of
the Python function of that name, or None without having done anything when the call is not a plain one; the Python function
then takes its own path.  The module is loaded at the first use.  It is built for one torch version, unlike the C library
behind both paths: without it (not built, or built for another torch) every call takes the Python path, after one warning."""
import importlib.util
import os
import warnings

from . import _lib
from ._build import HOST_PATH

# the library's entry points in the order of the Abi struct in csrc/host_calls.cpp
_ABI = ('dlb_last_error', 'dlb_workspace_lock', 'dlb_workspace_unlock', 'dlb_fp8_gemm', 'dlb_fp8_gemm_grouped_contiguous', 'dlb_fp8_gemm_grouped_contiguous_same_rows',
        'dlb_fp8_gemm_grouped_contiguous_gather_silu_quant', 'dlb_fp8_gemm_grouped_masked',
        'dlb_expert_gate_up_masked', 'dlb_fp8_gemm_grouped_ragged', 'dlb_expert_gate_up_ragged', 'dlb_expert_plan', 'dlb_fp8_quant_group',
        'dlb_silu_mul_quant_masked', 'dlb_ep_scatter_workspace_bytes', 'dlb_ep_scatter_rows_host', 'dlb_ep_gather')


_FUNCTIONS = ('fp8_gemm', 'quant', 'grouped_contiguous', 'grouped_masked', 'low_latency_experts', 'ep_gather', 'fused_moe_v3')

# the same for the StepAbi struct and the functions of csrc/host_steps.cpp
_STEP_ABI = ('dlb_last_error', 'dlb_rms_norm_backward_workspace_bytes', 'dlb_rms_norm_backward', 'dlb_moe_unpermute_backward', 'dlb_rms_norm', 'dlb_rms_norm_quant', 'dlb_moe_permute_workspace_bytes', 'dlb_moe_permute', 'dlb_moe_unpermute', 'dlb_w4_gemm_workspace_bytes',
             'dlb_w4_gemm', 'dlb_layer_norm', 'dlb_layer_norm_backward_workspace_bytes', 'dlb_layer_norm_backward',
             'dlb_mxfp4_quant', 'dlb_mxfp4_gemm_workspace_bytes', 'dlb_mxfp4_gemm',
             'dlb_mxfp4_weight_gemm', 'dlb_few_token_experts_workspace_bytes', 'dlb_few_token_experts')
_STEP_FUNCTIONS = ('rms_norm', 'rms_norm_quant', 'layer_norm', 'moe_permute', 'moe_unpermute', 'w4_gemm', 'w4_gemm_grouped', 'per_group_quant_mxfp4', 'mxfp4_gemm', 'mxfp4_weight_gemm',
                   'few_token_experts')


def _declined(*args):
    return None


def _load():
    import ctypes
    lib = _lib.load()
    try:
        if not os.path.exists(HOST_PATH):
            raise ImportError('it has not been built')
        spec = importlib.util.spec_from_file_location('dlblas_amd._host', HOST_PATH)
        host = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(host)
        address = lambda name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value
        host.init([address(name) for name in _ABI], _lib.workspace)
        host.init_steps([address(name) for name in _STEP_ABI])
    except (ImportError, ValueError, AttributeError) as exc:
        warnings.warn(f'cannot use {HOST_PATH} ({exc}): calls cost more host time; run `python -m dlblas_amd._build`', RuntimeWarning)
        return None
    return host


def __getattr__(name):
    if name not in _FUNCTIONS + _STEP_FUNCTIONS:
        raise AttributeError(name)
    try:
        host = _load()
    except ImportError:  # no library: the Python path says so as soon as it needs it
        return _declined
    for fn in _FUNCTIONS + _STEP_FUNCTIONS:
        globals()[fn] = getattr(host, fn) if host is not None else _declined
    return globals()[name]
