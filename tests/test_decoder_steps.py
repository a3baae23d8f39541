"""The steps around the products without a GPU: the header against the binding, what the C ABI and the Python functions refuse, and the
definitions in 64 bits against differences and against each other."""
import ctypes
import os
import re

import pytest
import torch

from dlblas_amd import _decoder, _lib
from dlblas_amd.kernels.moe_permute import MoePermutation, _worst_rows, moe_permute, moe_unpermute
from dlblas_amd.kernels.rms_norm import rms_norm, rms_norm_quant
from dlblas_amd.kernels.w4_gemm import per_group_quant_w4, w4_gemm, w4_gemm_grouped
from oracle import decoder as orc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, 'include', 'dlblas_decoder.h')
bf16, f16, f32, i32, u8 = torch.bfloat16, torch.float16, torch.float32, torch.int32, torch.uint8


def test_header_binding_and_library_agree():
    text = re.sub(r'/\*.*?\*/', '', open(HEADER).read(), flags=re.S)
    declared = sorted(set(re.findall(r'\b(dlb_[a-z0-9_]+)\s*\(', text)))
    assert declared == sorted(_lib.DECODER_SYMBOLS)
    lib = _lib.load()
    for name in declared:
        assert hasattr(lib, name)
    for name, value in (('DLB_NORM_MAX_COLUMNS', _decoder.NORM_MAX_COLUMNS), ('DLB_SORT_MAX_EXPERTS', _decoder.SORT_MAX_EXPERTS),
                        ('DLB_ROWS_E4M3', _decoder.ROWS_E4M3)):
        assert int(re.search(rf'#define {name} (\d+)', text).group(1)) == value


# ---- the C ABI refuses before it touches the device --------------------------------------------------------------------

null, fake = ctypes.c_void_p(0), ctypes.c_void_p(4096)
OK, NULL, SHAPE, STRIDE, DTYPE, WORKSPACE, ALIGN = 0, _lib.ERR_NULL_POINTER, _lib.ERR_BAD_SHAPE, _lib.ERR_BAD_STRIDE, _lib.ERR_BAD_DTYPE, _lib.ERR_WORKSPACE, _lib.ERR_ALIGNMENT
at = ctypes.c_void_p


def refused(name, good, cases):
    call = getattr(_lib.load(), name)
    order = list(good)
    for changes, code in cases:
        args = dict(good, **changes)
        assert call(*(args[k] for k in order)) == code, (name, changes, _lib.last_error())


def test_norm_entry_points_refuse():
    good = dict(x=fake, x_rs=256, res=fake, res_rs=256, dtype=0, w=fake, w_dtype=0, y=fake, y_rs=256, sum=fake, sum_rs=256, rows=4, H=256, eps=1e-6, st=null)
    refused('dlb_rms_norm', good, [
        (dict(dtype=3), DTYPE), (dict(w_dtype=1), DTYPE), (dict(rows=-1), SHAPE), (dict(H=32769), SHAPE), (dict(rows=1 << 31), SHAPE), (dict(x=null), NULL),
        (dict(w=null), NULL), (dict(sum=null), NULL), (dict(y=null), NULL), (dict(y_rs=255), STRIDE), (dict(sum_rs=255), STRIDE), (dict(x_rs=-1), STRIDE),
        (dict(res_rs=-1), STRIDE), (dict(x=at(4097)), ALIGN), (dict(res=at(4097)), ALIGN), (dict(y=at(4097)), ALIGN), (dict(w=at(4098), w_dtype=2), ALIGN),
        (dict(rows=0, x=null, y=null), OK), (dict(H=0, x=null, y=null), OK)])
    good = dict(x=fake, x_rs=256, res=fake, res_rs=256, dtype=0, w=fake, w_dtype=2, q=fake, s=fake, s_m=2, s_k=1, sum=fake, sum_rs=256, rows=4, H=256, eps=1e-6,
                qeps=1e-10, st=null)
    refused('dlb_rms_norm_quant', good, [
        (dict(dtype=-1), DTYPE), (dict(H=200), SHAPE), (dict(qeps=0.0), SHAPE), (dict(qeps=float('nan')), SHAPE), (dict(q=null), NULL), (dict(s=null), NULL),
        (dict(sum=null), NULL), (dict(q=at(4100)), ALIGN), (dict(s=at(4098)), ALIGN), (dict(s_m=-1), STRIDE), (dict(s_k=-1), STRIDE), (dict(sum_rs=100), STRIDE),
        (dict(rows=0, q=null), OK)])
    lib = _lib.load()
    need = lib.dlb_rms_norm_backward_workspace_bytes(4, 256)
    assert need > 0 and lib.dlb_rms_norm_backward_workspace_bytes(0, 256) == 0
    good = dict(dy=fake, dy_rs=256, ds=fake, ds_rs=256, h=fake, h_rs=256, dtype=0, w=fake, w_dtype=0, dx=fake, dx_rs=256, dw=fake, rows=4, H=256, eps=1e-6, ws=fake,
                wsb=need, st=null)
    refused('dlb_rms_norm_backward', good, [
        (dict(dtype=7), DTYPE), (dict(w_dtype=1), DTYPE), (dict(H=40000), SHAPE), (dict(dy=null), NULL), (dict(h=null), NULL), (dict(dx=null), NULL),
        (dict(dx_rs=2), STRIDE), (dict(dy_rs=-1), STRIDE), (dict(ds_rs=-1), STRIDE), (dict(dy=at(4097)), ALIGN), (dict(dw=at(4097)), ALIGN), (dict(ws=null), WORKSPACE),
        (dict(wsb=need - 1), WORKSPACE), (dict(ws=at(4098)), ALIGN), (dict(H=0), OK), (dict(rows=0, dw=null), OK)])


def test_sort_entry_points_refuse():
    lib = _lib.load()
    need = lib.dlb_moe_permute_workspace_bytes(100000, 8, 64)
    assert need > 0 and lib.dlb_moe_permute_workspace_bytes(0, 8, 64) == 0 and lib.dlb_moe_permute_workspace_bytes(128, 8, 64) == 0
    good = dict(ids=fake, i_dt=0, s0=8, s1=1, x=fake, x_rs=256, dt=0, xs=null, xs0=0, xs1=0, ri=fake, src=fake, mi=fake, st=fake, en=fake, rows=fake, rs=null,
                T=100000, H=256, topk=8, E=64, al=1, R=100, ws=fake, wsb=need, stream=null)
    f8 = dict(dt=3, xs=fake, rs=fake, xs0=2, xs1=1)
    refused('dlb_moe_permute', good, [
        (dict(i_dt=2), DTYPE), (dict(T=-1), SHAPE), (dict(topk=0), SHAPE), (dict(topk=65), SHAPE), (dict(E=0), SHAPE), (dict(E=1025), SHAPE), (dict(al=0), SHAPE),
        (dict(al=(1 << 20) + 1), SHAPE), (dict(R=-1), SHAPE), (dict(R=1 << 31), SHAPE), (dict(T=1 << 29), SHAPE), (dict(s0=-8), STRIDE), (dict(ids=null), NULL),
        (dict(ri=null), NULL), (dict(src=null), NULL), (dict(mi=null), NULL), (dict(st=null), NULL), (dict(en=null), NULL), (dict(ws=null), WORKSPACE),
        (dict(wsb=need - 1), WORKSPACE), (dict(ids=at(4100), i_dt=1), ALIGN), (dict(src=at(4098)), ALIGN), (dict(ws=at(4098)), ALIGN),
        (dict(dt=4), DTYPE), (dict(H=-1), SHAPE), (dict(x=null), NULL), (dict(rows=null), NULL),
        (dict(x_rs=-1), STRIDE), (dict(x=at(4097)), ALIGN), (dict(f8, H=200), SHAPE), (dict(f8, xs=null), NULL), (dict(f8, rs=null), NULL), (dict(f8, x=at(4104)), ALIGN),
        (dict(f8, x_rs=264), ALIGN), (dict(f8, xs0=-1), STRIDE)])
    good = dict(rows=fake, rs=256, dt=0, ri=fake, w=fake, out=fake, o_rs=256, T=10, H=256, topk=2, R=20, st=null)
    refused('dlb_moe_unpermute', good, [
        (dict(dt=3), DTYPE), (dict(T=-1), SHAPE), (dict(topk=65), SHAPE), (dict(rows=null), NULL), (dict(ri=null), NULL), (dict(out=null), NULL), (dict(o_rs=255), STRIDE),
        (dict(rs=-1), STRIDE), (dict(rows=at(4097)), ALIGN), (dict(w=at(4098)), ALIGN), (dict(T=0, out=null), OK)])
    good = dict(do=fake, do_rs=256, rows=fake, rs=256, dt=0, ri=fake, src=fake, w=fake, dr=fake, dr_rs=256, dw=fake, T=10, H=256, topk=2, R=20, st=null)
    refused('dlb_moe_unpermute_backward', good, [
        (dict(dt=3), DTYPE), (dict(H=0), SHAPE), (dict(H=32769), SHAPE), (dict(do=null), NULL), (dict(ri=null), NULL), (dict(src=null), NULL), (dict(dr=null), NULL),
        (dict(rows=null), NULL), (dict(dr_rs=255), STRIDE), (dict(do_rs=-1), STRIDE), (dict(dr=at(4097)), ALIGN), (dict(T=0, R=0), OK)])


def test_w4_entry_points_refuse():
    good = dict(x=fake, x_rs=256, dt=0, q=fake, s=fake, s_dt=0, z=null, y=fake, y_rs=64, rs=fake, re=fake, rows=4, N=64, K=256, g=128, E=2, ws=null, wsb=0, st=null)
    refused('dlb_w4_gemm', good, [
        (dict(dt=2), DTYPE), (dict(s_dt=2), DTYPE), (dict(rows=-1), SHAPE), (dict(g=16), SHAPE), (dict(g=256), SHAPE), (dict(K=192), SHAPE), (dict(K=0), SHAPE),
        (dict(rs=null), NULL), (dict(re=null), NULL), (dict(rs=null, re=null), SHAPE), (dict(x=null), NULL), (dict(q=null), NULL), (dict(s=null), NULL), (dict(y=null), NULL),
        (dict(y_rs=63), STRIDE), (dict(x_rs=-1), STRIDE), (dict(q=at(4104)), ALIGN), (dict(x=at(4098)), ALIGN), (dict(x_rs=257), ALIGN), (dict(x_rs=(1 << 24) + 2), STRIDE), (dict(s=at(4097)), ALIGN),
        (dict(rs=at(4098)), ALIGN), (dict(rows=1 << 31), SHAPE), (dict(K=1 << 31), SHAPE), (dict(K=1 << 25), STRIDE), (dict(rows=0, x=null), OK), (dict(N=0, y=null), OK)])
    lib = _lib.load()
    need = lib.dlb_w4_gemm_workspace_bytes(16, 7168, 18432, 0)
    assert need > 0 and lib.dlb_w4_gemm_workspace_bytes(16, 7168, 18432, 32) == 0 and lib.dlb_w4_gemm_workspace_bytes(1, 16, 128, 0) == 0
    good.update(x_rs=18432, y_rs=7168, rs=null, re=null, rows=16, N=7168, K=18432, E=1, ws=fake, wsb=need)
    refused('dlb_w4_gemm', good, [(dict(ws=null), WORKSPACE), (dict(wsb=need - 1), WORKSPACE), (dict(ws=at(4098)), ALIGN)])
    good = dict(w=fake, w_rs=256, dt=0, q=fake, s=fake, z=null, rows=4, K=256, g=128, st=null)
    refused('dlb_w4_quant', good, [
        (dict(dt=3), DTYPE), (dict(rows=-1), SHAPE), (dict(g=48), SHAPE), (dict(K=300), SHAPE), (dict(w=null), NULL), (dict(q=null), NULL), (dict(s=null), NULL),
        (dict(w_rs=-1), STRIDE), (dict(q=at(4098)), ALIGN), (dict(w=at(4097)), ALIGN), (dict(rows=0, w=null), OK)])


# ---- the Python functions ------------------------------------------------------------------------------------------------


def zeros(*size, dtype=bf16):
    return torch.zeros(size, dtype=dtype)


@pytest.mark.parametrize('call,error', [
    (lambda: rms_norm(zeros(2, 8, dtype=torch.float64), zeros(8)), TypeError),
    (lambda: rms_norm(zeros(2, 8), zeros(8, dtype=f16)), TypeError),
    (lambda: rms_norm(zeros(2, 8), zeros(7)), ValueError),
    (lambda: rms_norm(zeros(2, 8), zeros(8), 1e-6, zeros(3, 8)), ValueError),
    (lambda: rms_norm(zeros(2, 8), zeros(8), 1e-6, zeros(2, 8, dtype=f16)), ValueError),
    (lambda: rms_norm(zeros(2, 8), zeros(8), -1.0), ValueError),
    (lambda: rms_norm(zeros(2, 8), zeros(8), float('nan')), ValueError),
    (lambda: rms_norm(zeros(2, 0), zeros(0)), ValueError),
    (lambda: rms_norm(zeros(1, 32769), zeros(32769)), ValueError),
    (lambda: rms_norm_quant(zeros(2, 200), zeros(200)), AssertionError),
    (lambda: rms_norm_quant(zeros(2, 256), zeros(256), group_size=64), NotImplementedError),
    (lambda: rms_norm_quant(zeros(2, 256), zeros(256), quant_eps=0.0), ValueError),
    (lambda: rms_norm_quant(zeros(2, 256).requires_grad_(), zeros(256)), NotImplementedError),
    (lambda: moe_permute(zeros(2, 3, 4), zeros(2, 1, dtype=i32), 4), ValueError),
    (lambda: moe_permute(zeros(2, 8), zeros(3, 1, dtype=i32), 4), ValueError),
    (lambda: moe_permute(zeros(2, 8), zeros(2, 1, dtype=f32), 4), TypeError),
    (lambda: moe_permute(zeros(2, 8), zeros(2, 65, dtype=i32), 4), ValueError),
    (lambda: moe_permute(zeros(2, 8), zeros(2, 0, dtype=i32), 4), ValueError),
    (lambda: moe_permute(zeros(2, 8), zeros(2, 1, dtype=i32), 0), ValueError),
    (lambda: moe_permute(zeros(2, 8), zeros(2, 1, dtype=i32), 1025), ValueError),
    (lambda: moe_permute(zeros(2, 8), zeros(2, 1, dtype=i32), 4, alignment=0), ValueError),
    (lambda: moe_permute(zeros(2, 8), zeros(2, 1, dtype=i32), 4, num_rows=-1), ValueError),
    (lambda: moe_permute(zeros(2, 8, dtype=torch.float64), zeros(2, 1, dtype=i32), 4), TypeError),
    (lambda: moe_permute((zeros(2, 128), zeros(2, 1, dtype=f32)), zeros(2, 1, dtype=i32), 4), TypeError),
    (lambda: moe_permute((zeros(2, 128, dtype=u8).view(torch.float8_e4m3fn), zeros(2, 2, dtype=f32)), zeros(2, 1, dtype=i32), 4), ValueError),
    (lambda: moe_permute((zeros(2, 100, dtype=u8).view(torch.float8_e4m3fn), zeros(2, 1, dtype=f32)), zeros(2, 1, dtype=i32), 4), AssertionError),
    (lambda: moe_unpermute(zeros(2, 8, dtype=torch.float64), zeros(2, 1, dtype=i32)), TypeError),
    (lambda: moe_unpermute(zeros(2, 8), zeros(2, 1, dtype=torch.int64)), TypeError),
    (lambda: moe_unpermute(zeros(2, 8), zeros(2, dtype=i32)), ValueError),
    (lambda: moe_unpermute(zeros(2, 8), zeros(2, 1, dtype=i32), zeros(2, 2, dtype=f32)), ValueError),
    (lambda: moe_unpermute(zeros(2, 8), zeros(2, 1, dtype=i32), zeros(2, 1)), TypeError),
    (lambda: moe_unpermute(zeros(2, 8).requires_grad_(), zeros(2, 1, dtype=i32)), ValueError),
    (lambda: moe_unpermute(zeros(2, 8).requires_grad_(), MoePermutation(*(zeros(3, 1, dtype=i32), zeros(3, dtype=i32)) + (None, ) * 3)), ValueError),
    (lambda: w4_gemm(zeros(2, 256, dtype=f32), zeros(8, 128, dtype=u8), zeros(8, 2)), TypeError),
    (lambda: w4_gemm(zeros(2, 256), zeros(8, 128, dtype=torch.int8), zeros(8, 2)), TypeError),
    (lambda: w4_gemm(zeros(2, 256), zeros(8, 128, dtype=u8), zeros(8, 2, dtype=f32)), TypeError),
    (lambda: w4_gemm(zeros(2, 256), zeros(8, 128, dtype=u8), zeros(7, 2)), ValueError),
    (lambda: w4_gemm(zeros(2, 256), zeros(8, 128, dtype=u8), zeros(8, 1)), ValueError),
    (lambda: w4_gemm(zeros(2, 256), zeros(8, 128, dtype=u8), zeros(8, 0)), ValueError),
    (lambda: w4_gemm(zeros(2, 128), zeros(8, 128, dtype=u8), zeros(8, 2)), ValueError),
    (lambda: w4_gemm(zeros(2, 256), zeros(8, 128, dtype=u8), zeros(8, 2), zeros(8, 2)), TypeError),
    (lambda: w4_gemm(zeros(2, 256), zeros(8, 128, dtype=u8), zeros(8, 2), zeros(8, 1, dtype=u8)), ValueError),
    (lambda: w4_gemm(zeros(2, 256), zeros(128, 8, dtype=u8).t(), zeros(8, 2)), AssertionError),
    (lambda: w4_gemm(zeros(2, 256).requires_grad_(), zeros(8, 128, dtype=u8), zeros(8, 2)), NotImplementedError),
    (lambda: w4_gemm_grouped(zeros(1, 2, 256), zeros(3, 8, 128, dtype=u8), zeros(3, 8, 2), zeros(3, dtype=i32), zeros(3, dtype=i32)), ValueError),
    (lambda: w4_gemm_grouped(zeros(2, 256), zeros(8, 128, dtype=u8), zeros(8, 2), zeros(3, dtype=i32), zeros(3, dtype=i32)), ValueError),
    (lambda: w4_gemm_grouped(zeros(2, 256), zeros(3, 8, 128, dtype=u8), zeros(3, 8, 2), zeros(3, dtype=torch.int64), zeros(3, dtype=i32)), TypeError),
    (lambda: w4_gemm_grouped(zeros(2, 256), zeros(3, 8, 128, dtype=u8), zeros(3, 8, 2), zeros(3, dtype=i32), zeros(2, dtype=i32)), ValueError),
    (lambda: per_group_quant_w4(zeros(8, 256, dtype=u8)), TypeError),
    (lambda: per_group_quant_w4(zeros(8, 256, dtype=f32)), TypeError),
    (lambda: per_group_quant_w4(zeros(256)), ValueError),
    (lambda: per_group_quant_w4(zeros(8, 256), 48), NotImplementedError),
    (lambda: per_group_quant_w4(zeros(8, 200), 128), AssertionError),
    (lambda: per_group_quant_w4(zeros(8, 256).requires_grad_()), NotImplementedError),
])
def test_python_functions_refuse(call, error):
    with pytest.raises(error):
        call()


@pytest.mark.parametrize('slots,experts,alignment', [(0, 4, 128), (1, 4, 1), (7, 3, 16), (64, 256, 128), (1000, 8, 128)])
def test_default_rows_are_enough_for_any_routing(slots, experts, alignment):
    rows = _worst_rows(slots, experts, alignment)
    assert rows % alignment == 0
    g = torch.Generator().manual_seed(slots)
    for spread in (1, 2, experts):
        counts = torch.bincount(torch.randint(0, spread, (slots, ), generator=g), minlength=experts).tolist()
        assert sum(-(-c // alignment) * alignment for c in counts) <= rows


# ---- the definitions ------------------------------------------------------------------------------------------------------


def test_norm_gradient_is_the_differences_of_the_norm():
    """Central differences of sum(y * dy) + sum(h * dsum) in 64 bits, step 1e-6: off by the cube of the step and 2^-52 / step."""
    g = torch.Generator().manual_seed(3)
    x, w, dy, dsum = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((3, 10), (10, ), (3, 10), (3, 10)))
    f = lambda x, w: float((orc.rms_norm(x, w, 1e-3) * dy).sum() + (x * dsum).sum())
    dx, dw = orc.rms_norm_grad(dy, dsum, x, w, 1e-3)[:2]
    step = 1e-6
    for v, d in ((x, dx), (w, dw)):
        for i in range(v.numel()):
            up, down = v.clone(), v.clone()
            up.view(-1)[i] += step
            down.view(-1)[i] -= step
            num = (f(up, w) - f(down, w)) / (2 * step) if v is x else (f(x, up) - f(x, down)) / (2 * step)
            assert abs(num - float(d.reshape(-1)[i])) < 1e-7


def test_sorted_order_is_stable_and_spans_are_aligned():
    ids = torch.tensor([[2, 0], [0, 0], [-1, 5], [2, 1]])
    row_index, source, m_indices, start, end = orc.sort_tables(ids, 3, 4, 14)
    assert start.tolist() == [0, 4, 8] and end.tolist() == [3, 5, 10]
    assert source.tolist() == [1, 2, 3, -1, 7, -1, -1, -1, 0, 6, -1, -1, -1, -1]
    assert m_indices.tolist() == [0] * 4 + [1] * 4 + [2] * 4 + [-1] * 2
    assert row_index.tolist() == [[8, 0], [1, 2], [-1, -1], [9, 4]]
    cut = orc.sort_tables(ids, 3, 4, 9)
    assert cut[0].tolist() == [[8, 0], [1, 2], [-1, -1], [-1, 4]] and cut[4].tolist() == [3, 5, 9]


def test_4_bit_codes_in_a_byte():
    assert orc.w4_codes(torch.tensor([[0x21, 0xf8]], dtype=u8)).tolist() == [[1, 2, 8, 15]]


def test_tensors_of_two_devices_are_refused():
    class On:
        is_cuda = True

        def __init__(self, index):
            self.device = torch.device('cuda', index)

    _decoder._require_one_gpu(On(0), On(0))
    with pytest.raises(RuntimeError, match='one GPU'):
        _decoder._require_one_gpu(On(0), On(0), On(1))
