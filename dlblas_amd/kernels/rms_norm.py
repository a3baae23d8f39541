"""Root-mean-square norm with the residual's addition, for training, and the form that leaves the (a, a_s) operands of the FP8
block-scaled products, for serving.  The reference has the norms as dlblas/kernels/rms_norm.py and add_rms_norm.py.

    h = x + residual, rounded to the type of x          (without a residual h = x)
    y = h / sqrt(mean(h^2) + eps) * weight              in fp32, rounded once

``h`` is rounded before the norm reads it, because it is what the next layer adds to and what the gradient starts from.  The sum of
squares is held in fp32: rows whose sum passes 2^128 give zeros.
"""
from typing import Optional

import torch

from .. import _decoder, _fast, _lib
from ..utils import SymVar, Tensor, register_dlblas_op


@torch.library.custom_op('dlblas::rms_norm', mutates_args=('y', 'summed'), device_types='cuda')
def _norm_op(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor], y: torch.Tensor, summed: Optional[torch.Tensor],
             eps: float) -> None:
    _decoder.rms_norm(x, weight, residual, y, summed, eps)


@torch.library.custom_op('dlblas::rms_norm_quant', mutates_args=('q', 's', 'summed'), device_types='cuda')
def _norm_quant_op(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor], q: torch.Tensor, s: torch.Tensor,
                   summed: Optional[torch.Tensor], eps: float, quant_eps: float) -> None:
    _decoder.rms_norm_quant(x, weight, residual, q, s, summed, eps, quant_eps)


@torch.library.custom_op('dlblas::rms_norm_backward', mutates_args=('dx', 'dw'), device_types='cuda')
def _norm_backward_op(dy: torch.Tensor, dsum: Optional[torch.Tensor], h: torch.Tensor, weight: torch.Tensor, dx: torch.Tensor,
                      dw: Optional[torch.Tensor], eps: float) -> None:
    _decoder.rms_norm_backward(dy, dsum, h, weight, dx, dw, eps)


def _check(x, weight, residual, eps):
    _decoder.no_tangents(x, weight, residual)
    if x.dtype not in _lib.IN_CODES:
        raise TypeError(f'x must be bfloat16, float16 or float32, got {x.dtype}')
    if x.dim() < 1 or x.size(-1) < 1:
        raise ValueError('x must be [..., H] with at least one column')
    if x.size(-1) > _decoder.NORM_MAX_COLUMNS:
        raise ValueError(f'rows of at most {_decoder.NORM_MAX_COLUMNS} columns are implemented, got {x.size(-1)}')
    if weight.dtype not in (x.dtype, torch.float32):
        raise TypeError(f'weight must have the type of x or float32, got {weight.dtype}')
    if tuple(weight.shape) != (x.size(-1), ):
        raise ValueError(f'weight must be [{x.size(-1)}], got {list(weight.shape)}')
    if residual is not None and (residual.dtype != x.dtype or residual.shape != x.shape):
        raise ValueError('residual must have the shape and type of x')
    if not eps >= 0:
        raise ValueError(f'eps must not be negative, got {eps}')


def _rows(t):
    """[rows, H] with contiguous columns: a view where t allows it."""
    if t is None:
        return None
    if t.dim() == 2 and t.stride(1) == 1:
        return t
    return t.contiguous().view(-1, t.size(-1))


def _forward(x, weight, residual, eps):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    summed = None if residual is None else torch.empty_like(y)
    H = x.size(-1)
    _norm_op(_rows(x), weight.contiguous(), _rows(residual), y.view(-1, H), None if summed is None else summed.view(-1, H), float(eps))
    return y, summed


class _RmsNorm(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, summed = _forward(x, weight, residual, eps)
        ctx.set_materialize_grads(False)
        ctx.eps = eps
        ctx.save_for_backward(x if summed is None else summed, weight)
        return y if summed is None else (y, summed)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dsum=None):
        _decoder.no_tangents(dy, dsum)
        h, weight = ctx.saved_tensors
        if dy is None:  # only the sum went on
            return dsum, None, dsum if ctx.needs_input_grad[2] else None, None
        H = dy.size(-1)
        h = _decoder.given_back(h, dy, dy.dtype, dy.shape)
        weight = _decoder.given_back(weight, dy, torch.float32 if weight.dtype == torch.float32 else dy.dtype, (H, ))
        dx = torch.empty(h.shape, dtype=h.dtype, device=h.device)
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=weight.device) if ctx.needs_input_grad[1] else None
        _norm_backward_op(_rows(dy), _rows(dsum), _rows(h), weight.contiguous(), dx.view(-1, H), dw, float(ctx.eps))
        return dx, dw, dx if ctx.needs_input_grad[2] else None, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None):
    """RMS norm of ``x`` [..., H] (bf16 / fp16 / fp32) with ``weight`` [H] of the same type or fp32, in the type of x.

    Returns ``y``; with a ``residual`` like x ``(y, h)``, where ``h = x + residual`` is what the next residual starts from.
    Differentiable in x, weight and residual, once and in reverse mode; sums over rows are added in a fixed order.
    """
    if not torch.compiler.is_compiling():
        out = _fast.rms_norm(x, weight, eps, residual)
        if out is not None:
            return out
    _check(x, weight, residual, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        return _RmsNorm.apply(x, weight, residual, eps)
    y, summed = _forward(x, weight, residual, eps)
    return y if residual is None else (y, summed)


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None,
                   group_size: int = 128, quant_eps: float = 1e-10, column_major_scales: bool = False):
    """``rms_norm`` whose ``y`` leaves as float8_e4m3fn with one fp32 scale per 128 columns, in one pass over the rows: what
    ``fp8_gemm``, the grouped products and ``fused_moe_v3`` take.  y goes into the quantiser unrounded.

    Returns ``(q, s)``, with a residual ``(q, s, h)``: q like x in fp8, s [..., H / 128] with ``s = max(amax, quant_eps) / 448`` (a
    column-major view when ``column_major_scales``, as ``per_token_group_quant_fp8`` makes it).  A group with an infinity or a NaN
    dequantises to NaN.  Not differentiable.
    """
    if not torch.compiler.is_compiling():
        out = _fast.rms_norm_quant(x, weight, eps, residual, group_size, quant_eps, column_major_scales)
        if out is not None:
            return out
    _check(x, weight, residual, eps)
    if group_size != 128:
        raise NotImplementedError(f'only group_size 128 is implemented, got {group_size}')
    H = x.size(-1)
    assert H % group_size == 0, f'the last dimension of x {H} must be divisible by group_size {group_size}'
    if not quant_eps >= 1e-30:
        raise ValueError(f'quant_eps must be at least 1e-30, got {quant_eps}')
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise NotImplementedError('rms_norm_quant has no gradient: call it under torch.no_grad(), or rms_norm')
    rows = x.numel() // H
    q = torch.empty(x.shape, device=x.device, dtype=torch.float8_e4m3fn)
    if column_major_scales:
        buf = torch.empty((H // group_size, rows), device=x.device, dtype=torch.float32)
        s2d = buf.t()
        s = buf.reshape((H // group_size, ) + x.shape[:-1]).movedim(0, -1)
    else:
        s = torch.empty(x.shape[:-1] + (H // group_size, ), device=x.device, dtype=torch.float32)
        s2d = s.view(rows, H // group_size)
    summed = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _norm_quant_op(_rows(x), weight.contiguous(), _rows(residual), q.view(-1, H), s2d, None if summed is None else summed.view(-1, H), float(eps),
                   float(quant_eps))
    return (q, s) if residual is None else (q, s, summed)


def _bench(fn):

    def bench(*args, warmup: int = 3, rep: int = 10) -> float:
        for _ in range(warmup):
            fn(*args)
        times = []
        for _ in range(rep):
            start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            fn(*args)
            stop.record()
            stop.synchronize()
            times.append(start.elapsed_time(stop))
        times.sort()
        return times[len(times) // 2]

    return bench


def _register():
    m, k = SymVar('m'), SymVar('k')
    for fn in (rms_norm, rms_norm_quant):
        for dt in (torch.bfloat16, torch.float16, torch.float32):
            register_dlblas_op(fn.__name__, None, (Tensor((m, k), dtype=dt, device='cuda'), Tensor((k, ), dtype=dt, device='cuda')), fn, _bench(fn), fn)


_register()
