"""A layer of experts for the few tokens of a decode step: two kernels instead of a sort, two grouped products, an activation and a gather.

    out[t] = sum over the slots j of topk_weights[t, j] * W2[e] (silu(gate) * up),   gate, up = halves of W13[e] x[t],   e = topk_ids[t, j]

Beside ``fused_moe_v3`` and ``low_latency_experts``, which take quantised tokens that are sorted or laid out by expert, and hold what lies between the
products in e4m3: here tokens come as they are in 16 bits, routing is read on the device, and what lies between the products is fp32.  Weights are
those calls' e4m3 ones or the 4-bit ones of ``per_group_quant_mxfp4``.  The reference has no counterpart.
"""
from typing import Tuple

import torch

from .. import _decoder, _fast, _mxfp4

BLOCK = 128


@torch.library.custom_op('dlblas::few_token_experts', mutates_args=('out', ), device_types='cuda')
def _experts_op(x: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor, w13: torch.Tensor, w13_s: torch.Tensor, w2: torch.Tensor,
                w2_s: torch.Tensor, out: torch.Tensor) -> None:
    _mxfp4.few_token_experts(x, topk_ids, topk_weights, w13, w13_s, w2, w2_s, out)


def _check_weights(name, q, s, columns):
    """Types and layouts of [E, rows, columns] weights."""
    if q.dim() != 3 or s.dim() != 3:
        raise ValueError(f'{name} and its scales must have three dimensions, got {list(q.shape)} and {list(s.shape)}')
    assert q.is_contiguous() and s.is_contiguous(), 'Weight tensors must be contiguous'
    if q.dtype == torch.uint8:
        if s.dtype != torch.uint8:
            raise TypeError(f'scales of 4-bit {name} must be uint8, got {s.dtype}')
        unit, need, held = _mxfp4.GROUP, (q.size(0), q.size(1), columns // _mxfp4.GROUP), 2 * q.size(2)
    elif q.dtype == torch.float8_e4m3fn:
        if s.dtype != torch.float32:
            raise TypeError(f'scales of {name} must be float32, got {s.dtype}')
        unit, need, held = BLOCK, (q.size(0), -(-q.size(1) // BLOCK), columns // BLOCK), q.size(2)
    else:
        raise TypeError(f'{name} must be float8_e4m3fn or uint8 (4-bit codes), got {q.dtype}')
    if held != columns:
        raise ValueError(f'{name} has {held} columns where {columns} are expected')
    if columns == 0 or columns % unit != 0 or columns > 1 << 20:
        raise ValueError(f'columns of {name} must be a multiple of {unit}, at most 2^20, got {columns}')
    if tuple(s.shape) != need:
        raise ValueError(f'scales of {name} must be {list(need)}, got {list(s.shape)}')


def few_token_experts(x: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor, w13_weight: Tuple[torch.Tensor, torch.Tensor],
                      w2_weight: Tuple[torch.Tensor, torch.Tensor]) -> torch.Tensor:
    """
    Args:
        x: tokens ``[T, H]`` in bfloat16 or float16, at most 64.
        topk_ids: ``[T, topk]`` int32 or int64, at most 16 experts a token; values outside ``0 ... E - 1`` (other GPUs' experts, -1) are left out.
        topk_weights: ``[T, topk]`` float32.
        w13_weight: ``(w, s)``, gate rows and behind them up rows: ``[E, 2 I, H]`` float8_e4m3fn with float32 scales
            ``[E, ceil(2 I / 128), H / 128]``, or 4-bit codes ``[E, 2 I, H / 2]`` uint8 with scales ``[E, 2 I, H / 32]`` uint8; contiguous, E at most 1024.
        w2_weight: ``[E, H, I]`` in the same form.

    Returns:
        ``[T, H]`` in the type of x; fp32 sums, one rounding; zeros for a token without an expert here.  Not differentiable.  For more tokens:
        ``fused_moe_v3`` with e4m3 weights; no call takes 4-bit ones by expert for a prompt, which leaves ``mxfp4_gemm`` on the rows of one expert after the other.
    """
    if not torch.compiler.is_compiling():
        out = _fast.few_token_experts(x, topk_ids, topk_weights, w13_weight, w2_weight)
        if out is not None:
            return out
    (w13, w13_s), (w2, w2_s) = w13_weight, w2_weight
    _decoder.no_tangents(x, topk_weights, w13_s if w13_s.is_floating_point() else None, w2_s if w2_s.is_floating_point() else None)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f'x must be bfloat16 or float16, got {x.dtype}')
    if x.dim() != 2 or topk_ids.dim() != 2 or topk_ids.size(0) != x.size(0):
        raise ValueError(f'x must be [T, H] and topk_ids [T, topk], got {list(x.shape)} and {list(topk_ids.shape)}')
    if topk_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f'topk_ids must be int32 or int64, got {topk_ids.dtype}')
    if topk_weights.dtype != torch.float32:
        raise TypeError(f'topk_weights must be float32, got {topk_weights.dtype}')
    if topk_weights.shape != topk_ids.shape:
        raise ValueError(f'topk_weights must be like topk_ids {list(topk_ids.shape)}, got {list(topk_weights.shape)}')
    T, H = x.shape
    if T > _mxfp4.FEW_TOKENS:
        more = 'fused_moe_v3 takes more' if w13.dtype != torch.uint8 else 'of 4-bit experts more go through mxfp4_gemm, expert by expert'
        raise ValueError(f'at most {_mxfp4.FEW_TOKENS} tokens are implemented, got {T}: {more}')
    if not 1 <= topk_ids.size(1) <= _mxfp4.FEW_TOPK:
        raise ValueError(f'1 to {_mxfp4.FEW_TOPK} experts a token are implemented, got {topk_ids.size(1)}')
    if w13.dtype != w2.dtype:
        raise TypeError(f'w13_weight and w2_weight must have one type, got {w13.dtype} and {w2.dtype}')
    if w13.dim() != 3 or w13.size(1) % 2 != 0:
        raise ValueError(f'w13_weight must be [E, 2 I, H], got {list(w13.shape)}')
    E, I = w13.size(0), w13.size(1) // 2
    if not 1 <= E <= _mxfp4.FEW_EXPERTS:
        raise ValueError(f'1 to {_mxfp4.FEW_EXPERTS} experts are implemented, got {E}')
    _check_weights('w13_weight', w13, w13_s, H)
    _check_weights('w2_weight', w2, w2_s, I)
    if w2.size(0) != E or w2.size(1) != H:
        raise ValueError(f'w2_weight must be [{E}, {H}, {I}], got {list(w2.shape)}')
    if T * topk_ids.size(1) * I > _mxfp4.FEW_NUMBERS:
        raise ValueError(f'tokens * topk * I is {T * topk_ids.size(1) * I}, at most {_mxfp4.FEW_NUMBERS} are implemented')
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, topk_weights, w13, w13_s, w2, w2_s)):
        raise NotImplementedError('few_token_experts has no gradient: call it under torch.no_grad()')
    out = torch.empty((T, H), dtype=x.dtype, device=x.device)
    if T > 0:
        _experts_op(x, topk_ids, topk_weights.contiguous(), w13, w13_s, w2, w2_s, out)
    return out
