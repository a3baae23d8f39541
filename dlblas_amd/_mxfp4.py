"""The calls of include/dlblas_mxfp4.h on torch tensors: pointers, strides, device and stream.  Shapes and types are the business of the functions
in kernels/, which call these through their custom ops."""
import torch

from ._decoder import _present, _require_one_gpu, _rs
from ._lib import IDX_CODES, IN_CODES, _ptr, _stream, check, load

GROUP = 32  # columns that share a scale
MAX_COLUMNS = 1 << 22
FEW_TOKENS, FEW_TOPK, FEW_EXPERTS, FEW_NUMBERS = 64, 16, 1024, 1 << 29
WEIGHTS_E4M3, WEIGHTS_MXFP4 = 0, 1


def on_bytes(t, n):
    """A contiguous tensor that starts on n bytes.  Inside the ops, because an address is none that a compiled caller has."""
    return t if t.data_ptr() % n == 0 else t.clone(memory_format=torch.contiguous_format)


def quant(x, q, s):
    _require_one_gpu(x, q, s)
    with torch.cuda.device(x.device):
        check(load().dlb_mxfp4_quant(_ptr(x), _rs(x), IN_CODES[x.dtype], _ptr(q), _ptr(s), x.size(0), x.size(1), _stream(x)))


def gemm(a, b, a_s, b_s, c):
    _require_one_gpu(a, b, a_s, b_s, c)
    lib = load()
    with torch.cuda.device(a.device):
        M, N, K = c.size(0), c.size(1), 2 * b.size(1)
        # scratch of its own, so that two captured graphs never share it
        need = lib.dlb_mxfp4_gemm_workspace_bytes(M, N, K)
        ws = torch.empty(need, dtype=torch.uint8, device=a.device)
        a, b, a_s, b_s = on_bytes(a, 16), on_bytes(b, 16), on_bytes(a_s, 4), on_bytes(b_s, 4)
        check(lib.dlb_mxfp4_gemm(_ptr(a), _ptr(b), _ptr(a_s), _ptr(b_s), _ptr(c), M, N, K, IN_CODES[c.dtype], _ptr(ws), need, _stream(a)))


def on_dwords(x):
    """Rows as the kernels of a few rows read them: contiguous columns, on 4 bytes, at most 2^23 elements apart."""
    if (x.stride(1) != 1 and x.size(1) > 1) or x.data_ptr() % 4 != 0 or x.stride(0) % 2 != 0 or x.stride(0) > 1 << 23:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def weight_gemm(x, w_q, w_s, y):
    _require_one_gpu(x, w_q, w_s, y)
    with torch.cuda.device(x.device):
        x, w_q = on_dwords(x), on_bytes(w_q, 16)
        check(load().dlb_mxfp4_weight_gemm(_ptr(x), _rs(x), IN_CODES[x.dtype], _ptr(w_q), _ptr(w_s), _ptr(y), x.size(0), w_q.size(0), x.size(1), _stream(x)))


def few_token_experts(x, ids, weights, up_q, up_s, down_q, down_s, out):
    _require_one_gpu(x, ids, weights, up_q, up_s, down_q, down_s, out)
    lib = load()
    f4 = up_q.dtype == torch.uint8
    with torch.cuda.device(x.device):
        (T, topk), I = ids.shape, up_q.size(1) // 2
        # scratch of its own, so that two captured graphs never share it
        need = lib.dlb_few_token_experts_workspace_bytes(T, topk, I)
        ws = torch.empty(need, dtype=torch.uint8, device=x.device)
        x, up_q, down_q = on_dwords(x), on_bytes(up_q, 16), on_bytes(down_q, 16)
        check(lib.dlb_few_token_experts(_ptr(x), _rs(x), IN_CODES[x.dtype], _ptr(ids), IDX_CODES[ids.dtype], ids.stride(0), ids.stride(1), _ptr(weights),
                                        WEIGHTS_MXFP4 if f4 else WEIGHTS_E4M3, _ptr(up_q), _ptr(up_s), _ptr(down_q), _ptr(down_s), _ptr(out), T, topk,
                                        up_q.size(0), x.size(1), I, _ptr(ws), need, _stream(x)))
