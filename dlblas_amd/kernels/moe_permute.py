"""Tokens sorted by expert and back, with gradients.

``ep_scatter`` and ``ep_gather`` (fused_moe_v3) do this for a dispatcher that knows every expert's count on the host; ``moe_permute``
counts on the device, so nothing waits for it, and both directions are differentiable.  The tables it leaves are the ones the
products take: ``m_indices`` with ``alignment=128`` for ``m_grouped_fp8_gemm_nt_contiguous``, ``row_start`` / ``row_end`` for the ragged
products and ``w4_gemm_grouped``.  The reference has the pair as dlblas/kernels/permute/moe_triton_kernels.py.
"""
from typing import NamedTuple, Optional, Tuple, Union

import torch

from .. import _decoder, _fast, _lib


class MoePermutation(NamedTuple):
    """Which slot lies where (all int32): a slot is a (token, j) of topk_ids.  The tables may lie behind each other in one allocation, on 4
    bytes each: keeping one keeps all of them."""
    row_index: torch.Tensor  # [T, topk] row of every slot, -1 where it has none
    source: torch.Tensor     # [rows] slot t * topk + j of every row, -1 where it holds none
    m_indices: torch.Tensor  # [rows] expert of every row of a span, -1 past the last span
    row_start: torch.Tensor  # [experts] first row of every expert's span
    row_end: torch.Tensor    # [experts] one past its last row that holds a slot


@torch.library.custom_op('dlblas::moe_permute', mutates_args=('row_index', 'source', 'm_indices', 'row_start', 'row_end', 'rows', 'rows_s'),
                         device_types='cuda')
def _permute_op(topk_ids: torch.Tensor, x: torch.Tensor, x_s: Optional[torch.Tensor], row_index: torch.Tensor, source: torch.Tensor,
                m_indices: torch.Tensor, row_start: torch.Tensor, row_end: torch.Tensor, rows: torch.Tensor, rows_s: Optional[torch.Tensor],
                alignment: int) -> None:
    # inside the op, because an address is none that a compiled caller has
    if x_s is not None and (x.stride(1) != 1 or x.stride(0) % 16 != 0 or x.data_ptr() % 16 != 0):
        x = x.clone(memory_format=torch.contiguous_format)
    _decoder.moe_permute(topk_ids, x, x_s, row_index, source, m_indices, row_start, row_end, rows, rows_s, alignment)


@torch.library.custom_op('dlblas::moe_unpermute', mutates_args=('out', ), device_types='cuda')
def _unpermute_op(rows: torch.Tensor, row_index: torch.Tensor, weights: Optional[torch.Tensor], out: torch.Tensor) -> None:
    _decoder.moe_unpermute(rows, row_index, weights, out)


@torch.library.custom_op('dlblas::moe_unpermute_backward', mutates_args=('drows', 'dweights'), device_types='cuda')
def _unpermute_backward_op(dout: torch.Tensor, rows: Optional[torch.Tensor], row_index: torch.Tensor, source: torch.Tensor,
                           weights: Optional[torch.Tensor], drows: torch.Tensor, dweights: Optional[torch.Tensor]) -> None:
    _decoder.moe_unpermute_backward(dout, rows, row_index, source, weights, drows, dweights)


def _columns_whole(t):
    return t if t is None or t.stride(1) == 1 or t.size(1) == 1 else t.contiguous()


def _permuted(x, x_s, topk_ids, num_experts, alignment, num_rows):

    def table(*size):
        return torch.empty(size, dtype=torch.int32, device=x.device)

    p = MoePermutation(table(*topk_ids.shape), table(num_rows), table(num_rows), table(num_experts), table(num_experts))
    rows = torch.empty((num_rows, x.size(1)), dtype=x.dtype, device=x.device)
    rows_s = None if x_s is None else torch.empty((num_rows, x_s.size(1)), dtype=torch.float32, device=x.device)
    _permute_op(topk_ids, x, x_s, *p, rows, rows_s, alignment)
    return rows, rows_s, p


def _unpermuted(rows, row_index, weights):
    out = torch.empty((row_index.size(0), rows.size(1)), dtype=rows.dtype, device=rows.device)
    _unpermute_op(rows, row_index, weights, out)
    return out


class _Permute(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, topk_ids, num_experts, alignment, num_rows):
        rows, _, p = _permuted(_columns_whole(x), None, topk_ids, num_experts, alignment, num_rows)
        ctx.save_for_backward(p.row_index)
        ctx.slots = topk_ids.shape
        ctx.mark_non_differentiable(*p)
        return (rows, ) + tuple(p)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, drows, *_):
        _decoder.no_tangents(drows)
        row_index = _decoder.given_back(ctx.saved_tensors[0], drows, torch.int32, ctx.slots).contiguous()
        return _unpermuted(_columns_whole(drows), row_index, None), None, None, None, None


class _Unpermute(torch.autograd.Function):

    @staticmethod
    def forward(ctx, rows, weights, row_index, source):
        ctx.save_for_backward(rows if weights is not None and weights.requires_grad else None, weights, row_index, source)
        ctx.num_rows, ctx.slots = rows.size(0), row_index.shape
        return _unpermuted(_columns_whole(rows), row_index, None if weights is None else weights.contiguous())

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        _decoder.no_tangents(dout)
        rows, weights, row_index, source = ctx.saved_tensors
        row_index = _decoder.given_back(row_index, dout, torch.int32, ctx.slots).contiguous()
        source = _decoder.given_back(source, dout, torch.int32, (ctx.num_rows, )).contiguous()
        weights = None if weights is None else _decoder.given_back(weights, dout, torch.float32, ctx.slots).contiguous()
        drows = torch.empty((ctx.num_rows, dout.size(1)), dtype=dout.dtype, device=dout.device)
        dweights = torch.empty(weights.shape, dtype=torch.float32, device=dout.device) if ctx.needs_input_grad[1] else None
        if dweights is not None:
            rows = _columns_whole(_decoder.given_back(rows, dout, dout.dtype, drows.shape))
        _unpermute_backward_op(_columns_whole(dout), rows if dweights is not None else None, row_index, source, weights, drows, dweights)
        return drows if ctx.needs_input_grad[0] else None, dweights, None, None


def _worst_rows(slots, num_experts, alignment):
    """Rows that suffice whatever the routing: the spans of as many experts as there are slots are each a row short of a block too long."""
    return -(-(slots + min(num_experts, slots) * (alignment - 1)) // alignment) * alignment


def moe_permute(x: Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]], topk_ids: torch.Tensor, num_experts: int, alignment: int = 1,
                num_rows: Optional[int] = None):
    """Copies every token next to the other tokens of each expert it is routed to: returns ``(rows, permutation)``.

    x          [T, H] bf16 / fp16 / fp32, or the pair ``(q, s)`` of ``per_token_group_quant_fp8`` / ``rms_norm_quant`` (float8_e4m3fn and its
               [T, H / 128] scales); rows is the pair then too, its scales row-major
    topk_ids   [T, topk] int32 / int64, topk at most 64; ids below 0 or from num_experts (at most 1024) on name no expert here
    alignment  every expert's span is a multiple of this many rows
    num_rows   rows to return; slots whose row would lie past them are dropped (row_index -1).  By default enough for any routing, which
               with many experts and a large alignment is far more than one routing fills

    Rows are in the order of (expert, token, j); rows that hold no slot are zero.  Differentiable in x, once and
    in reverse mode; quantised tokens are not.
    """
    quantised = isinstance(x, (tuple, list))
    x, x_s = x if quantised else (x, None)
    if not torch.compiler.is_compiling():
        out = _fast.moe_permute(x, x_s, topk_ids, num_experts, alignment, num_rows)
        if out is not None:
            rows = (out[0], out[1]) if quantised else out[0]
            return rows, MoePermutation(*out[2:])
    _decoder.no_tangents(x, x_s)
    if x.dim() != 2 or topk_ids.dim() != 2 or topk_ids.size(0) != x.size(0):
        raise ValueError(f'x must be [T, H] and topk_ids [T, topk], got {list(x.shape)} and {list(topk_ids.shape)}')
    if topk_ids.dtype not in _lib.IDX_CODES:
        raise TypeError(f'topk_ids must be int32 or int64, got {topk_ids.dtype}')
    if not 1 <= topk_ids.size(1) <= _decoder.SORT_MAX_TOPK:
        raise ValueError(f'1 to {_decoder.SORT_MAX_TOPK} experts a token are implemented, got {topk_ids.size(1)}')
    if not 1 <= num_experts <= _decoder.SORT_MAX_EXPERTS:
        raise ValueError(f'1 to {_decoder.SORT_MAX_EXPERTS} experts are implemented, got {num_experts}')
    if alignment < 1:
        raise ValueError(f'alignment must be at least 1, got {alignment}')
    if num_rows is None:
        num_rows = _worst_rows(topk_ids.numel(), num_experts, alignment)
    if num_rows < 0:
        raise ValueError(f'num_rows must not be negative, got {num_rows}')
    if quantised:
        if x.dtype != torch.float8_e4m3fn or x_s.dtype != torch.float32:
            raise TypeError(f'quantised tokens must be float8_e4m3fn with float32 scales, got {x.dtype} and {x_s.dtype}')
        assert x.size(1) % 128 == 0, f'the last dimension of x {x.size(1)} must be divisible by 128'
        if tuple(x_s.shape) != (x.size(0), x.size(1) // 128):
            raise ValueError(f'scales must be {[x.size(0), x.size(1) // 128]}, got {list(x_s.shape)}')
        if torch.is_grad_enabled() and (x.requires_grad or x_s.requires_grad):
            raise NotImplementedError('quantised tokens have no gradient: permute them under torch.no_grad()')
        rows, rows_s, p = _permuted(x, x_s, topk_ids, num_experts, alignment, num_rows)
        return (rows, rows_s), p
    if x.dtype not in _lib.IN_CODES:
        raise TypeError(f'x must be bfloat16, float16 or float32, or float8_e4m3fn with its scales, got {x.dtype}')
    if torch.is_grad_enabled() and x.requires_grad:
        out = _Permute.apply(x, topk_ids, num_experts, alignment, num_rows)
        return out[0], MoePermutation(*out[1:])
    rows, _, p = _permuted(_columns_whole(x), None, topk_ids, num_experts, alignment, num_rows)
    return rows, p


def moe_unpermute(rows: torch.Tensor, permutation: Union[MoePermutation, torch.Tensor], topk_weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[t] = sum_j topk_weights[t, j] * rows[row_index[t, j]]`` over the slots that have a row: [T, H] in the type of rows.

    rows [R, H] bf16 / fp16 / fp32; permutation as ``moe_permute`` returned it, or any int32 [T, topk] table of rows (entries outside
    0 ... R - 1 name none); topk_weights [T, topk] float32, all one by default.  fp32 sums in slot order, one rounding; a token without a
    row gets zeros.  Differentiable in rows and topk_weights, once and in reverse mode, for which it needs the permutation, not a table alone.
    """
    whole = isinstance(permutation, MoePermutation)
    row_index = permutation.row_index if whole else permutation
    if not torch.compiler.is_compiling():
        out = _fast.moe_unpermute(rows, row_index, topk_weights, permutation.source if whole else None)
        if out is not None:
            return out
    _decoder.no_tangents(rows, topk_weights)
    if rows.dtype not in _lib.IN_CODES:
        raise TypeError(f'rows must be bfloat16, float16 or float32, got {rows.dtype}')
    if row_index.dtype != torch.int32:
        raise TypeError(f'the table of rows must be int32, got {row_index.dtype}')
    if rows.dim() != 2 or row_index.dim() != 2 or not 1 <= row_index.size(1) <= _decoder.SORT_MAX_TOPK:
        raise ValueError(f'rows must be [R, H] and the table [T, 1 ... {_decoder.SORT_MAX_TOPK}], got {list(rows.shape)} and {list(row_index.shape)}')
    if topk_weights is not None:
        if topk_weights.dtype != torch.float32:
            raise TypeError(f'topk_weights must be float32, got {topk_weights.dtype}')
        if topk_weights.shape != row_index.shape:
            raise ValueError(f'topk_weights must be {list(row_index.shape)}, got {list(topk_weights.shape)}')
    row_index = row_index.contiguous()
    if torch.is_grad_enabled() and (rows.requires_grad or (topk_weights is not None and topk_weights.requires_grad)):
        if not whole:
            raise ValueError('the gradients need the MoePermutation of moe_permute: a table of rows may name a row twice')
        if permutation.source.dtype != torch.int32:
            raise TypeError(f'the permutation holds int32 tables, got a source of {permutation.source.dtype}')
        if tuple(permutation.source.shape) != (rows.size(0), ):
            raise ValueError(f'the permutation is one of {permutation.source.numel()} rows, got {rows.size(0)}')
        if rows.size(1) > _decoder.NORM_MAX_COLUMNS:
            raise ValueError(f'gradients of at most {_decoder.NORM_MAX_COLUMNS} columns are implemented, got {rows.size(1)}')
        return _Unpermute.apply(rows, topk_weights, row_index, permutation.source)
    return _unpermuted(_columns_whole(rows), row_index, None if topk_weights is None else topk_weights.contiguous())
