"""Layer norm with the residual's addition, for training and serving: the norm of models that centre their rows, beside ``rms_norm``.  The
reference has the norm without a residual under dlblas/kernels/layer_norm/.

    h = x + residual, rounded to the type of x                            (without a residual h = x)
    y = (h - mean(h)) / sqrt(mean((h - mean(h))^2) + eps) * weight + bias in fp32, rounded once

``h`` is rounded before the norm reads it, because it is what the next layer adds to and what the gradient starts from.  The squares are those
of the centred row, in fp32: rows whose sum passes 2^130 give the bias.
"""
from typing import Optional

import torch

from .. import _decoder, _fast
from ..utils import SymVar, Tensor, register_dlblas_op
from .rms_norm import _bench, _rows
from .rms_norm import _check as _check_rows


@torch.library.custom_op('dlblas::layer_norm', mutates_args=('y', 'summed', 'stats'), device_types='cuda')
def _norm_op(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], residual: Optional[torch.Tensor], y: torch.Tensor,
             summed: Optional[torch.Tensor], stats: Optional[torch.Tensor], eps: float) -> None:
    _decoder.layer_norm(x, weight, bias, residual, y, summed, stats, eps)


@torch.library.custom_op('dlblas::layer_norm_backward', mutates_args=('dx', 'dw', 'db'), device_types='cuda')
def _norm_backward_op(dy: torch.Tensor, dsum: Optional[torch.Tensor], h: torch.Tensor, weight: torch.Tensor, stats: torch.Tensor, dx: torch.Tensor,
                      dw: Optional[torch.Tensor], db: Optional[torch.Tensor]) -> None:
    _decoder.layer_norm_backward(dy, dsum, h, weight, stats, dx, dw, db)


def _check(x, weight, bias, residual, eps):
    _check_rows(x, weight, residual, eps)
    _decoder.no_tangents(bias)
    if bias is not None:
        if bias.dtype != weight.dtype:
            raise TypeError(f'bias must have the type of weight, {weight.dtype}, got {bias.dtype}')
        if bias.shape != weight.shape:
            raise ValueError(f'bias must be [{weight.size(0)}], got {list(bias.shape)}')


def _forward(x, weight, bias, residual, eps, with_stats):
    H = x.size(-1)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    summed = None if residual is None else torch.empty_like(y)
    stats = torch.empty((x.numel() // H, 2), dtype=torch.float32, device=x.device) if with_stats else None
    _norm_op(_rows(x), weight.contiguous(), None if bias is None else bias.contiguous(), _rows(residual), y.view(-1, H),
             None if summed is None else summed.view(-1, H), stats, float(eps))
    return y, summed, stats


class _LayerNorm(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps):
        y, summed, stats = _forward(x, weight, bias, residual, eps, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x if summed is None else summed, weight, stats)
        return y if summed is None else (y, summed)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dsum=None):
        _decoder.no_tangents(dy, dsum)
        h, weight, stats = ctx.saved_tensors
        want_x, want_w, want_b, want_res, _ = ctx.needs_input_grad
        if dy is None:  # only the sum went on
            return dsum, None, None, dsum if want_res else None, None
        H = dy.size(-1)
        h = _decoder.given_back(h, dy, dy.dtype, dy.shape)
        weight = _decoder.given_back(weight, dy, torch.float32 if weight.dtype == torch.float32 else dy.dtype, (H, ))
        stats = _decoder.given_back(stats, dy, torch.float32, (dy.numel() // H, 2)).contiguous()
        dx = torch.empty(h.shape, dtype=h.dtype, device=h.device)
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=weight.device) if want_w or want_b else None
        db = torch.empty_like(dw) if want_b else None
        _norm_backward_op(_rows(dy), _rows(dsum), _rows(h), weight.contiguous(), stats, dx.view(-1, H), dw, db)
        return dx, dw if want_w else None, db, dx if want_res else None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               residual: Optional[torch.Tensor] = None):
    """Layer norm of ``x`` [..., H] (bf16 / fp16 / fp32) with ``weight`` and ``bias`` [H] (or no bias) of the same type or both fp32, in the
    type of x.

    Returns ``y``; with a ``residual`` like x ``(y, h)``, where ``h = x + residual`` is what the next residual starts from.
    Differentiable in x, weight, bias and residual, once and in reverse mode; sums over rows are added in a fixed order.
    """
    if not torch.compiler.is_compiling():
        out = _fast.layer_norm(x, weight, bias, eps, residual)
        if out is not None:
            return out
    _check(x, weight, bias, residual, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return _LayerNorm.apply(x, weight, bias, residual, eps)
    y, summed, _ = _forward(x, weight, bias, residual, eps, False)
    return y if residual is None else (y, summed)


def _register():
    m, k = SymVar('m'), SymVar('k')
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        row = Tensor((k, ), dtype=dt, device='cuda')
        register_dlblas_op('layer_norm', None, (Tensor((m, k), dtype=dt, device='cuda'), row, row), layer_norm, _bench(layer_norm), layer_norm)


_register()
