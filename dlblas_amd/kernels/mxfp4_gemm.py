"""Microscaled 4-bit floating point (the OCP format MXFP4): quantiser and products, beside the FP8 block-scaled products at half their bytes and
twice their matrix rate.

    groups of 32 columns of a row share a scale 2^(s - 127), one byte s (255 = NaN); an element is e2m1: 0 0.5 1 1.5 2 3 4 6 with a sign
    mxfp4_gemm          y = a b^T of two quantised operands
    mxfp4_weight_gemm   y = x w^T of a few 16-bit rows and quantised weights

Codes are uint8 [..., K / 2], two a byte, the even column in the low half; scales uint8 [..., K / 32].  Tensors of torch's float4_e2m1fn_x2 and
float8_e8m0fnu hold the same bytes: ``view(torch.uint8)``.  The reference has no counterpart.
"""
from typing import Optional

import torch

from .. import _decoder, _fast, _lib, _mxfp4
from ..utils import SymVar, Tensor, register_dlblas_op
from .rms_norm import _bench, _rows

GROUP = _mxfp4.GROUP


@torch.library.custom_op('dlblas::per_group_quant_mxfp4', mutates_args=('q', 's'), device_types='cuda')
def _quant_op(x: torch.Tensor, q: torch.Tensor, s: torch.Tensor) -> None:
    _mxfp4.quant(x, q, s)


@torch.library.custom_op('dlblas::mxfp4_gemm', mutates_args=('c', ), device_types='cuda')
def _gemm_op(a: torch.Tensor, b: torch.Tensor, a_s: torch.Tensor, b_s: torch.Tensor, c: torch.Tensor) -> None:
    _mxfp4.gemm(a, b, a_s, b_s, c)


@torch.library.custom_op('dlblas::mxfp4_weight_gemm', mutates_args=('y', ), device_types='cuda')
def _weight_op(x: torch.Tensor, w_q: torch.Tensor, w_s: torch.Tensor, y: torch.Tensor) -> None:
    _mxfp4.weight_gemm(x, w_q, w_s, y)


def _check_columns(K):
    if K % GROUP != 0:
        raise ValueError(f'the last dimension {K} must be divisible by {GROUP}, the columns of a scale')
    if K > _mxfp4.MAX_COLUMNS:
        raise ValueError(f'at most {_mxfp4.MAX_COLUMNS} columns are implemented, got {K}')


def _check_operand(q, s, name, dims):
    """Codes and scales of an operand; returns its columns.  dims None: any number, at least one."""
    for t, what in ((q, 'codes'), (s, 'scales')):
        if t.dtype != torch.uint8:
            raise TypeError(f'{what} of {name} must be uint8, got {t.dtype}')
        assert t.is_contiguous(), f'{what} of {name} must be contiguous'
    if q.dim() != s.dim() or q.dim() < 1 or (dims is not None and q.dim() != dims) or q.shape[:-1] != s.shape[:-1]:
        raise ValueError(f'codes and scales of {name} must have {dims or "the same"} dimensions, all but the last alike, got {list(q.shape)} and {list(s.shape)}')
    K = 2 * q.size(-1)
    _check_columns(K)
    if s.size(-1) != K // GROUP:
        raise ValueError(f'{name} has {K} columns and scales for {s.size(-1)} groups: one per {GROUP} columns')
    return K


def per_group_quant_mxfp4(x: torch.Tensor):
    """Codes and scales of ``x`` [..., K] (bf16 / fp16 / fp32, K a multiple of 32): ``(q, s)`` with q uint8 [..., K / 2] and s uint8 [..., K / 32].

    The scale of a group is the power of two two octaves below its largest magnitude's (``2^(floor(log2 amax) - 2)``), elements are rounded to
    nearest, ties to even, and what lies above 6 scales becomes 6.  A group that holds an infinity or a NaN gets the scale NaN.
    """
    if not torch.compiler.is_compiling():
        out = _fast.per_group_quant_mxfp4(x)
        if out is not None:
            return out
    _decoder.no_tangents(x)
    if x.dtype not in _lib.IN_CODES:
        raise TypeError(f'x must be bfloat16, float16 or float32, got {x.dtype}')
    if x.dim() < 1 or x.size(-1) < 1:
        raise ValueError('x must be [..., K] with at least one group of columns')
    K = x.size(-1)
    _check_columns(K)
    if torch.is_grad_enabled() and x.requires_grad:
        raise NotImplementedError('per_group_quant_mxfp4 has no gradient: call it under torch.no_grad()')
    q = torch.empty(x.shape[:-1] + (K // 2, ), dtype=torch.uint8, device=x.device)
    s = torch.empty(x.shape[:-1] + (K // GROUP, ), dtype=torch.uint8, device=x.device)
    _quant_op(_rows(x), q.view(-1, K // 2), s.view(-1, K // GROUP))
    return q, s


def mxfp4_gemm(a: torch.Tensor, b: torch.Tensor, a_s: torch.Tensor, b_s: torch.Tensor, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """
    Matrix product of operands in 4-bit floating point, ``a @ b.T``; operands in the order of ``fp8_gemm``.

    Args:
        a: codes of the activations ``[..., K / 2]`` uint8, contiguous; leading dimensions are flattened into M.
        b: codes of the weights ``[N, K / 2]`` uint8, contiguous.
        a_s: their scales ``[..., K / 32]`` uint8, contiguous.
        b_s: ``[N, K / 32]`` uint8, contiguous.
        out_dtype: bfloat16, float16 or float32; None: ``torch.get_default_dtype()``.

    Returns:
        ``[..., N]``, newly allocated, enqueued on the current stream; fp32 sums, one rounding.  A scale of 255 makes its row or column NaN.
    """
    if not torch.compiler.is_compiling():
        c = _fast.mxfp4_gemm(a, b, a_s, b_s, out_dtype)
        if c is not None:
            return c
    if out_dtype is None:
        out_dtype = torch.get_default_dtype()
    if out_dtype not in _lib.IN_CODES:
        raise TypeError(f'out_dtype must be bfloat16, float16 or float32, got {out_dtype}')
    K = _check_operand(b, b_s, 'b', 2)
    if _check_operand(a, a_s, 'a', None) != K:
        raise ValueError(f'a has {2 * a.size(-1)} columns and b {K}')
    N = b.size(0)
    c = torch.empty(a.shape[:-1] + (N, ), dtype=out_dtype, device=a.device)
    if c.numel() > 0:
        _gemm_op(a, b, a_s, b_s, c.view(-1, N))
    return c


def mxfp4_weight_gemm(x: torch.Tensor, w_q: torch.Tensor, w_s: torch.Tensor) -> torch.Tensor:
    """``x`` [..., K] (bf16 / fp16) times weights in 4-bit floating point, ``w_q`` [N, K / 2] uint8 with scales ``w_s`` [N, K / 32] uint8 as
    ``per_group_quant_mxfp4`` makes them: [..., N] in the type of x; fp32 sums, one rounding.

    For up to a few dozen rows, which stay unquantised: the weights are read once per 16 of them.
    """
    if not torch.compiler.is_compiling():
        y = _fast.mxfp4_weight_gemm(x, w_q, w_s)
        if y is not None:
            return y
    _decoder.no_tangents(x)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f'x must be bfloat16 or float16, got {x.dtype}')
    K = _check_operand(w_q, w_s, 'w', 2)
    if x.dim() < 1 or x.size(-1) != K:
        raise ValueError(f'x must be [..., {K}], got {list(x.shape)}')
    if torch.is_grad_enabled() and x.requires_grad:
        raise NotImplementedError('products with 4-bit weights have no gradient: call them under torch.no_grad()')
    N = w_q.size(0)
    y = torch.empty(x.shape[:-1] + (N, ), dtype=x.dtype, device=x.device)
    if y.numel() > 0:
        _weight_op(x if x.dim() == 2 else x.reshape(-1, K), w_q, w_s, y.view(-1, N))
    return y


def _register():
    m, n, k, kh, g = (SymVar(s) for s in 'm n k kh g'.split())
    u8 = lambda *size: Tensor(size, dtype=torch.uint8, device='cuda')
    register_dlblas_op('mxfp4_gemm', None, (u8(m, kh), u8(n, kh), u8(m, g), u8(n, g)), mxfp4_gemm, _bench(mxfp4_gemm), mxfp4_gemm)
    for dt in (torch.bfloat16, torch.float16):
        register_dlblas_op('mxfp4_weight_gemm', None, (Tensor((m, k), dtype=dt, device='cuda'), u8(n, kh), u8(n, g)), mxfp4_weight_gemm, _bench(mxfp4_weight_gemm),
                           mxfp4_weight_gemm)
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        register_dlblas_op('per_group_quant_mxfp4', None, (Tensor((m, k), dtype=dt, device='cuda'), ), per_group_quant_mxfp4, _bench(per_group_quant_mxfp4),
                           per_group_quant_mxfp4)


_register()
