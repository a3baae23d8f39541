"""The calls of include/dlblas_decoder.h on torch tensors: pointers, strides, device and stream.  Shapes and types are the business of
the functions in kernels/, which call these through their custom ops."""
import torch
from torch.autograd import forward_ad

from ._lib import IDX_CODES, IN_CODES, _ptr, _require_gpu, _stream, check, load

ROWS_E4M3 = 3  # DLB_ROWS_E4M3
NORM_MAX_COLUMNS = 32768
SORT_MAX_EXPERTS = 1024
SORT_MAX_TOPK = 64


def _present(*tensors):
    return [t for t in tensors if t is not None]


def _require_one_gpu(*tensors):
    _require_gpu(*tensors)
    for t in tensors:
        if t.device != tensors[0].device:
            raise RuntimeError(f'all tensors of a call must be on one GPU, got {tensors[0].device} and {t.device}')


def no_tangents(*tensors):
    """Forward-mode derivatives are not implemented, and the ops write into outputs that no tangent follows: without this a tensor with a
    tangent would come back as one whose derivative is zero."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError('forward-mode derivatives of the steps around the products are not implemented')


def given_back(t, grad, dtype, shape):
    """A saved tensor as a hook on saved tensors gave it back: the kernels are told nothing but its address."""
    if t.device != grad.device or t.dtype != dtype or tuple(t.shape) != tuple(shape):
        raise RuntimeError('a tensor saved for a gradient of dlblas_amd came back from its hook on another device, of another type or with other '
                           f'sizes: {t.device}, {t.dtype}, {list(t.shape)}')
    return t


def _rs(t):
    """Row stride of a [rows, columns] tensor; 0 for none."""
    return 0 if t is None else t.stride(0)


def rms_norm(x, weight, residual, y, summed, eps):
    _require_one_gpu(*_present(x, weight, residual, y, summed))
    with torch.cuda.device(x.device):
        check(load().dlb_rms_norm(_ptr(x), _rs(x), _ptr(residual), _rs(residual), IN_CODES[x.dtype], _ptr(weight), IN_CODES[weight.dtype], _ptr(y),
                                  _rs(y), _ptr(summed), _rs(summed), x.size(0), x.size(1), float(eps), _stream(x)))


def rms_norm_quant(x, weight, residual, q, s, summed, eps, quant_eps):
    _require_one_gpu(*_present(x, weight, residual, q, s, summed))
    with torch.cuda.device(x.device):
        check(load().dlb_rms_norm_quant(_ptr(x), _rs(x), _ptr(residual), _rs(residual), IN_CODES[x.dtype], _ptr(weight), IN_CODES[weight.dtype],
                                        _ptr(q), _ptr(s), s.stride(0), s.stride(1), _ptr(summed), _rs(summed), x.size(0), x.size(1), float(eps),
                                        float(quant_eps), _stream(x)))


def rms_norm_backward(dy, dsum, h, weight, dx, dw, eps):
    _require_one_gpu(*_present(dy, dsum, h, weight, dx, dw))
    lib = load()
    with torch.cuda.device(h.device):
        rows, H = h.shape
        # scratch of its own, so that two captured graphs never share it
        need = lib.dlb_rms_norm_backward_workspace_bytes(rows, H) if dw is not None else 0
        ws = torch.empty(need, dtype=torch.uint8, device=h.device)
        check(lib.dlb_rms_norm_backward(_ptr(dy), _rs(dy), _ptr(dsum), _rs(dsum), _ptr(h), _rs(h), IN_CODES[h.dtype], _ptr(weight),
                                        IN_CODES[weight.dtype], _ptr(dx), _rs(dx), _ptr(dw), rows, H, float(eps), _ptr(ws), need, _stream(h)))


def layer_norm(x, weight, bias, residual, y, summed, stats, eps):
    _require_one_gpu(*_present(x, weight, bias, residual, y, summed, stats))
    with torch.cuda.device(x.device):
        check(load().dlb_layer_norm(_ptr(x), _rs(x), _ptr(residual), _rs(residual), IN_CODES[x.dtype], _ptr(weight), _ptr(bias), IN_CODES[weight.dtype],
                                    _ptr(y), _rs(y), _ptr(summed), _rs(summed), _ptr(stats), x.size(0), x.size(1), float(eps), _stream(x)))


def layer_norm_backward(dy, dsum, h, weight, stats, dx, dw, db):
    _require_one_gpu(*_present(dy, dsum, h, weight, stats, dx, dw, db))
    lib = load()
    with torch.cuda.device(h.device):
        rows, H = h.shape
        # scratch of its own, so that two captured graphs never share it
        need = lib.dlb_layer_norm_backward_workspace_bytes(rows, H, db is not None) if dw is not None else 0
        ws = torch.empty(need, dtype=torch.uint8, device=h.device)
        check(lib.dlb_layer_norm_backward(_ptr(dy), _rs(dy), _ptr(dsum), _rs(dsum), _ptr(h), _rs(h), IN_CODES[h.dtype], _ptr(weight),
                                          IN_CODES[weight.dtype], _ptr(stats), _ptr(dx), _rs(dx), _ptr(dw), _ptr(db), rows, H, _ptr(ws), need,
                                          _stream(h)))


def moe_permute(ids, x, x_s, row_index, source, m_indices, row_start, row_end, rows, rows_s, alignment):
    _require_one_gpu(*_present(ids, x, x_s, row_index, source, m_indices, row_start, row_end, rows, rows_s))
    code = ROWS_E4M3 if x.dtype == torch.float8_e4m3fn else IN_CODES[x.dtype]
    lib = load()
    with torch.cuda.device(x.device):
        (T, topk), E = ids.shape, row_start.numel()
        need = lib.dlb_moe_permute_workspace_bytes(T, topk, E)
        ws = torch.empty(need, dtype=torch.uint8, device=x.device)
        check(lib.dlb_moe_permute(_ptr(ids), IDX_CODES[ids.dtype], ids.stride(0), ids.stride(1), _ptr(x), _rs(x), code, _ptr(x_s), _rs(x_s),
                                  0 if x_s is None else x_s.stride(1), _ptr(row_index), _ptr(source), _ptr(m_indices), _ptr(row_start), _ptr(row_end),
                                  _ptr(rows), _ptr(rows_s), T, x.size(1), topk, E, alignment, source.numel(), _ptr(ws), need, _stream(x)))


def moe_unpermute(rows, row_index, weights, out):
    _require_one_gpu(*_present(rows, row_index, weights, out))
    with torch.cuda.device(rows.device):
        check(load().dlb_moe_unpermute(_ptr(rows), _rs(rows), IN_CODES[rows.dtype], _ptr(row_index), _ptr(weights), _ptr(out), _rs(out), out.size(0),
                                       out.size(1), row_index.size(1), rows.size(0), _stream(rows)))


def moe_unpermute_backward(dout, rows, row_index, source, weights, drows, dweights):
    _require_one_gpu(*_present(dout, rows, row_index, source, weights, drows, dweights))
    with torch.cuda.device(dout.device):
        check(load().dlb_moe_unpermute_backward(_ptr(dout), _rs(dout), _ptr(rows), _rs(rows), IN_CODES[dout.dtype], _ptr(row_index), _ptr(source),
                                                _ptr(weights), _ptr(drows), _rs(drows), _ptr(dweights), dout.size(0), dout.size(1),
                                                row_index.size(1), drows.size(0), _stream(dout)))


def w4_gemm(x, w_q, w_s, w_z, y, row_start, row_end, group):
    _require_one_gpu(*_present(x, w_q, w_s, w_z, y, row_start, row_end))
    lib = load()
    E = w_q.size(0) if w_q.dim() == 3 else 1
    with torch.cuda.device(x.device):
        need = lib.dlb_w4_gemm_workspace_bytes(x.size(0), w_q.size(-2), x.size(1), 0 if row_start is None else E)
        ws = torch.empty(need, dtype=torch.uint8, device=x.device)
        check(lib.dlb_w4_gemm(_ptr(x), _rs(x), IN_CODES[x.dtype], _ptr(w_q), _ptr(w_s), IN_CODES[w_s.dtype], _ptr(w_z), _ptr(y), _rs(y),
                              _ptr(row_start), _ptr(row_end), x.size(0), w_q.size(-2), x.size(1), group, E, _ptr(ws), need, _stream(x)))


def w4_quant(w, q, s, z, group):
    _require_one_gpu(*_present(w, q, s, z))
    with torch.cuda.device(w.device):
        check(load().dlb_w4_quant(_ptr(w), _rs(w), IN_CODES[w.dtype], _ptr(q), _ptr(s), _ptr(z), w.size(0), w.size(1), group, _stream(w)))
