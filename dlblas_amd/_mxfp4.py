"""The calls of include/dlblas_mxfp4.h on torch tensors: pointers, strides, device and stream.  Shapes and types are the business of the functions
in kernels/, which call these through their custom ops."""
import torch

from ._decoder import _present, _require_one_gpu, _rs
from ._lib import IN_CODES, _ptr, _stream, check, load

GROUP = 32  # columns that share a scale
MAX_COLUMNS = 1 << 22


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
