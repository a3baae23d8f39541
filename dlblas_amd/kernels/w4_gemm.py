"""Products of a few rows with 4-bit weights: the decode side of a layer whose weights are kept at half the bytes of e4m3.  That is what
they are for: against ``fp8_gemm`` they are faster where few rows meet many weights (1 x 7168 x 18432 22 and 24 us, 32 experts x 4 rows x
4096 x 7168 119 and 147) and slower elsewhere (1 x 2112 x 7168 7.6 and 6.3 us, 32 x 7168 x 7168 18 and 14, 64 x 7168 x 18432 48 and 39).

    y[m, n] = sum over the groups g of w_s[n, g] * sum_{k in g} x[m, k] * (w_q[n, k] - w_z[n, g])

``w_q`` holds two codes a byte, the even column in the low half; groups are 32, 64 or 128 columns of a row; without zero points
``w_z`` is 8.  The reference has no counterpart.
"""
from typing import Optional

import torch

from .. import _decoder, _fast
from ..utils import SymVar, Tensor, register_dlblas_op
from .rms_norm import _bench

GROUP_SIZES = (32, 64, 128)


def _columns_whole(t):
    return t if t.stride(1) == 1 or t.size(1) == 1 else t.contiguous()


def _on_dwords(t):
    """Rows as the kernel reads them: on 4 bytes and less than 2^25 bytes apart.  Inside the op, because an address is none that a compiled
    caller has."""
    t = _columns_whole(t)
    if t.data_ptr() % 4 != 0 or t.stride(0) % 2 != 0 or t.stride(0) > 1 << 24:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


@torch.library.custom_op('dlblas::w4_gemm', mutates_args=('y', ), device_types='cuda')
def _w4_op(x: torch.Tensor, w_q: torch.Tensor, w_s: torch.Tensor, w_z: Optional[torch.Tensor], y: torch.Tensor, row_start: Optional[torch.Tensor],
           row_end: Optional[torch.Tensor], group_size: int) -> None:
    _decoder.w4_gemm(_on_dwords(x), w_q, w_s, w_z, y, row_start, row_end, group_size)


@torch.library.custom_op('dlblas::per_group_quant_w4', mutates_args=('w_q', 'w_s', 'w_z'), device_types='cuda')
def _quant_op(w: torch.Tensor, w_q: torch.Tensor, w_s: torch.Tensor, w_z: Optional[torch.Tensor], group_size: int) -> None:
    _decoder.w4_quant(w, w_q, w_s, w_z, group_size)


def _check(x, w_q, w_s, w_z, dims):
    """Types, shapes and layouts of a product; returns the group size."""
    _decoder.no_tangents(x, w_s)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f'x must be bfloat16 or float16, got {x.dtype}')
    if w_q.dtype != torch.uint8:
        raise TypeError(f'w_q must be uint8 (two codes a byte), got {w_q.dtype}')
    if w_s.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f'w_s must be bfloat16 or float16, got {w_s.dtype}')
    if w_z is not None and w_z.dtype != torch.uint8:
        raise TypeError(f'w_z must be uint8, got {w_z.dtype}')
    if w_q.dim() != dims or w_s.dim() != dims or tuple(w_s.shape[:-1]) != tuple(w_q.shape[:-1]):
        raise ValueError(f'w_q and w_s must have {dims} dimensions, all but the last alike, got {list(w_q.shape)} and {list(w_s.shape)}')
    if w_z is not None and w_z.shape != w_s.shape:
        raise ValueError(f'w_z must be like w_s {list(w_s.shape)}, got {list(w_z.shape)}')
    K = 2 * w_q.size(-1)
    if K > 1 << 24:
        raise ValueError(f'at most 2^24 columns are implemented, got {K}')
    if x.size(-1) != K:
        raise ValueError(f'x has {x.size(-1)} columns and w_q {K}')
    groups = w_s.size(-1)
    if groups == 0 or K % groups != 0 or K // groups not in GROUP_SIZES:
        raise ValueError(f'{groups} groups over {K} columns: a group is one of {GROUP_SIZES} columns')
    assert all(t is None or t.is_contiguous() for t in (w_q, w_s, w_z)), 'Weight tensors must be contiguous'
    if torch.is_grad_enabled() and (x.requires_grad or w_s.requires_grad):
        raise NotImplementedError('products with 4-bit weights have no gradient: call them under torch.no_grad()')
    return K // groups


def w4_gemm(x: torch.Tensor, w_q: torch.Tensor, w_s: torch.Tensor, w_z: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x`` [..., K] (bf16 / fp16) times the 4-bit weights ``w_q`` [N, K / 2] uint8 with scales ``w_s`` [N, K / group] (bf16 or fp16)
    and zero points ``w_z`` (uint8 like w_s, 0 ... 16, or None: 8; a byte above 16 makes its column NaN): [..., N] in the type of x; fp32
    sums, one rounding.

    For up to a few dozen rows: the weights are read once per 32 of them.  A product of N(0, 1)-like rows is as exact as its rounding;
    see include/dlblas_decoder.h for rows that are nearly constant or close to the end of fp32.  An infinity in a row of x makes that
    row of the product NaN.
    """
    if not torch.compiler.is_compiling():
        y = _fast.w4_gemm(x, w_q, w_s, w_z)
        if y is not None:
            return y
    if x.dim() < 1:
        raise ValueError('x must be [..., K]')
    group = _check(x, w_q, w_s, w_z, 2)
    x2d = x if x.dim() == 2 else x.reshape(-1, x.size(-1))
    y = torch.empty(x.shape[:-1] + (w_q.size(0), ), dtype=x.dtype, device=x.device)
    _w4_op(x2d, w_q, w_s, w_z, y.view(-1, w_q.size(0)), None, None, group)
    return y


def w4_gemm_grouped(x: torch.Tensor, w_q: torch.Tensor, w_s: torch.Tensor, row_start: torch.Tensor, row_end: torch.Tensor,
                    w_z: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``w4_gemm`` by expert: the rows [row_start[e], row_end[e]) of ``x`` [R, K] times the weights of expert e, w_q [E, N, K / 2] and so on.
    The ranges (int32 [E] on the device, clamped to 0 ... R, no row in two of them) are those of ``moe_permute``; rows of no expert are not written.  For a decode
    step: an expert's weights are read once per 16 or 32 of its rows, and those of experts without a row not at all."""
    if not torch.compiler.is_compiling():
        y = _fast.w4_gemm_grouped(x, w_q, w_s, row_start, row_end, w_z)
        if y is not None:
            return y
    if x.dim() != 2:
        raise ValueError(f'x must be [R, K], got {list(x.shape)}')
    group = _check(x, w_q, w_s, w_z, 3)
    for name, t in (('row_start', row_start), ('row_end', row_end)):
        if t.dtype != torch.int32:
            raise TypeError(f'{name} must be int32, got {t.dtype}')
        if tuple(t.shape) != (w_q.size(0), ):
            raise ValueError(f'{name} must be [{w_q.size(0)}], got {list(t.shape)}')
    y = torch.empty((x.size(0), w_q.size(1)), dtype=x.dtype, device=x.device)
    _w4_op(x, w_q, w_s, w_z, y, row_start.contiguous(), row_end.contiguous(), group)
    return y


def per_group_quant_w4(w: torch.Tensor, group_size: int = 128, zero_points: bool = False):
    """4-bit codes of a weight ``w`` [N, K] or [E, N, K] (bf16 / fp16) for ``w4_gemm`` / ``w4_gemm_grouped``: returns
    ``(w_q, w_s, w_z)`` with w_q [..., K / 2] uint8, w_s [..., K / group_size] in the type of w and w_z uint8 like it, or None.

    Without zero points ``w_s = amax / 7`` and codes around 8; with them the range of a group from its lowest (at most 0) to its highest value
    (at least 0) is cut into 15 steps.  A group that holds an infinity or a NaN gets a scale of NaN, so its products show it.
    """
    _decoder.no_tangents(w)
    if w.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f'w must be bfloat16 or float16 (the type of its scales), got {w.dtype}')
    if w.dim() not in (2, 3):
        raise ValueError('w must be [N, K] or [E, N, K]')
    if group_size not in GROUP_SIZES:
        raise NotImplementedError(f'a group is one of {GROUP_SIZES} columns, got {group_size}')
    K = w.size(-1)
    assert K % group_size == 0, f'the last dimension of w {K} must be divisible by group_size {group_size}'
    if torch.is_grad_enabled() and w.requires_grad:
        raise NotImplementedError('per_group_quant_w4 has no gradient: call it under torch.no_grad()')
    w_q = torch.empty(w.shape[:-1] + (K // 2, ), dtype=torch.uint8, device=w.device)
    w_s = torch.empty(w.shape[:-1] + (K // group_size, ), dtype=w.dtype, device=w.device)
    w_z = torch.empty(w_s.shape, dtype=torch.uint8, device=w.device) if zero_points else None
    w2d = _columns_whole(w) if w.dim() == 2 else w.contiguous().view(-1, K)
    _quant_op(w2d, w_q.view(-1, K // 2), w_s.view(-1, K // group_size), None if w_z is None else w_z.view(-1, K // group_size), int(group_size))
    return w_q, w_s, w_z


def _register():
    m, n, k, kh, g = (SymVar(s) for s in 'm n k kh g'.split())
    for dt in (torch.bfloat16, torch.float16):
        register_dlblas_op('w4_gemm', None, (Tensor((m, k), dtype=dt, device='cuda'), Tensor((n, kh), dtype=torch.uint8, device='cuda'),
                                             Tensor((n, g), dtype=dt, device='cuda')), w4_gemm, _bench(w4_gemm), w4_gemm)


_register()
