"""Layer norm, 4-bit floating point and the experts for a few tokens without a GPU: the header against the binding, what the C ABI and the Python
functions refuse, and the definitions in 64 bits against differences and against each other."""
import ctypes
import math
import os
import re

import pytest
import torch

from dlblas_amd import _lib, _mxfp4
from dlblas_amd.kernels.few_token_experts import few_token_experts
from dlblas_amd.kernels.layer_norm import layer_norm
from dlblas_amd.kernels.mxfp4_gemm import mxfp4_gemm, mxfp4_weight_gemm, per_group_quant_mxfp4
from oracle import layer_norm as norm_orc
from oracle import mxfp4 as orc

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, 'include', 'dlblas_mxfp4.h')
bf16, f16, f32, f64, i32, i64, u8, f8 = torch.bfloat16, torch.float16, torch.float32, torch.float64, torch.int32, torch.int64, torch.uint8, torch.float8_e4m3fn


def test_header_binding_and_library_agree():
    source = open(HEADER).read()
    text = re.sub(r'/\*.*?\*/', '', source, flags=re.S)
    declared = sorted(set(re.findall(r'\b(dlb_[a-z0-9_]+)\s*\(', text)))
    assert declared == sorted(_lib.MXFP4_SYMBOLS)
    lib = _lib.load()
    for name in declared:
        assert hasattr(lib, name)
    for name, value in (('FEW_TOKENS', _mxfp4.FEW_TOKENS), ('FEW_TOPK', _mxfp4.FEW_TOPK), ('FEW_EXPERTS', _mxfp4.FEW_EXPERTS), ('WEIGHTS_E4M3', _mxfp4.WEIGHTS_E4M3),
                        ('WEIGHTS_MXFP4', _mxfp4.WEIGHTS_MXFP4)):
        assert int(re.search(rf'#define DLB_{name} (\d+)', text).group(1)) == value
    assert '#define DLB_MXFP4_MAX_COLUMNS (1 << 22)' in text and _mxfp4.MAX_COLUMNS == 1 << 22


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


def test_layer_norm_entry_points_refuse():
    good = dict(x=fake, x_rs=256, res=fake, res_rs=256, dtype=0, w=fake, b=fake, w_dtype=2, y=fake, y_rs=256, sum=fake, sum_rs=256, stats=fake, rows=4, H=256, eps=1e-5, st=null)
    refused('dlb_layer_norm', good, [
        (dict(dtype=3), DTYPE), (dict(w_dtype=1), DTYPE), (dict(rows=-1), SHAPE), (dict(H=-1), SHAPE), (dict(H=32769), SHAPE), (dict(rows=1 << 31), SHAPE), (dict(x=null), NULL),
        (dict(w=null), NULL), (dict(y=null), NULL), (dict(sum=null), NULL), (dict(y_rs=255), STRIDE), (dict(sum_rs=255), STRIDE), (dict(x_rs=-1), STRIDE),
        (dict(res_rs=-1), STRIDE), (dict(x=at(4097)), ALIGN), (dict(res=at(4097)), ALIGN), (dict(w=at(4098)), ALIGN), (dict(b=at(4098)), ALIGN), (dict(y=at(4097)), ALIGN),
        (dict(sum=at(4097)), ALIGN), (dict(stats=at(4098)), ALIGN), (dict(rows=0, x=null), OK), (dict(H=0, y=null), OK)])
    lib = _lib.load()
    need = lib.dlb_layer_norm_backward_workspace_bytes(4, 256, 1)
    assert need == 2 * lib.dlb_layer_norm_backward_workspace_bytes(4, 256, 0) > 0 and lib.dlb_layer_norm_backward_workspace_bytes(0, 256, 1) == 0
    good = dict(dy=fake, dy_rs=256, ds=fake, ds_rs=256, h=fake, h_rs=256, dtype=0, w=fake, w_dtype=0, stats=fake, dx=fake, dx_rs=256, dw=fake, db=fake, rows=4, H=256, ws=fake,
                wsb=need, st=null)
    refused('dlb_layer_norm_backward', good, [
        (dict(dtype=7), DTYPE), (dict(w_dtype=1), DTYPE), (dict(H=40000), SHAPE), (dict(rows=-1), SHAPE), (dict(dy=null), NULL), (dict(h=null), NULL), (dict(w=null), NULL),
        (dict(stats=null), NULL), (dict(dx=null), NULL), (dict(dw=null), NULL), (dict(dx_rs=2), STRIDE), (dict(dy_rs=-1), STRIDE), (dict(ds_rs=-1), STRIDE),
        (dict(h_rs=-1), STRIDE), (dict(dy=at(4097)), ALIGN), (dict(ds=at(4097)), ALIGN), (dict(stats=at(4098)), ALIGN), (dict(dw=at(4097)), ALIGN), (dict(db=at(4097)), ALIGN),
        (dict(ws=null), WORKSPACE), (dict(wsb=need - 1), WORKSPACE), (dict(ws=at(4098)), ALIGN), (dict(H=0), OK), (dict(rows=0, dw=null, db=null), OK)])


def test_mxfp4_entry_points_refuse():
    good = dict(x=fake, x_rs=256, dt=0, q=fake, s=fake, rows=4, K=256, st=null)
    refused('dlb_mxfp4_quant', good, [
        (dict(dt=3), DTYPE), (dict(rows=-1), SHAPE), (dict(K=-32), SHAPE), (dict(K=48), SHAPE), (dict(K=(1 << 22) + 32), SHAPE), (dict(rows=1 << 31), SHAPE), (dict(x=null), NULL),
        (dict(q=null), NULL), (dict(s=null), NULL), (dict(x_rs=-1), STRIDE), (dict(x=at(4097)), ALIGN), (dict(q=at(4098)), ALIGN), (dict(rows=0, x=null), OK), (dict(K=0, q=null), OK)])
    lib = _lib.load()
    good = dict(a=fake, b=fake, a_s=fake, b_s=fake, c=fake, M=4, N=64, K=256, dt=0, ws=null, wsb=0, st=null)
    refused('dlb_mxfp4_gemm', good, [
        (dict(dt=3), DTYPE), (dict(M=-1), SHAPE), (dict(N=-1), SHAPE), (dict(K=-32), SHAPE), (dict(K=0), SHAPE), (dict(K=100), SHAPE), (dict(K=(1 << 22) + 32), SHAPE),
        (dict(M=1 << 31), SHAPE), (dict(N=(1 << 27) + 1), SHAPE), (dict(a=null), NULL), (dict(b=null), NULL), (dict(a_s=null), NULL), (dict(b_s=null), NULL), (dict(c=null), NULL),
        (dict(a=at(4104)), ALIGN), (dict(b=at(4104)), ALIGN), (dict(a_s=at(4098)), ALIGN), (dict(b_s=at(4098)), ALIGN), (dict(c=at(4097)), ALIGN), (dict(dt=2, c=at(4098)), ALIGN),
        (dict(M=0, a=null), OK), (dict(N=0, c=null), OK)])
    need = lib.dlb_mxfp4_gemm_workspace_bytes(4096, 4096, 96)
    assert need > 0 and lib.dlb_mxfp4_gemm_workspace_bytes(4096, 4096, 256) == 0 == lib.dlb_mxfp4_gemm_workspace_bytes(4, 64, 96) and lib.dlb_mxfp4_gemm_workspace_bytes(0, 64, 96) == 0 == lib.dlb_mxfp4_gemm_workspace_bytes(-1, 64, 96)
    refused('dlb_mxfp4_gemm', dict(good, M=4096, N=4096, K=96, ws=fake, wsb=need), [(dict(ws=null), WORKSPACE), (dict(wsb=need - 1), WORKSPACE), (dict(ws=at(4104)), ALIGN)])
    good = dict(x=fake, x_rs=256, dt=0, q=fake, s=fake, y=fake, M=4, N=64, K=256, st=null)
    refused('dlb_mxfp4_weight_gemm', good, [
        (dict(dt=2), DTYPE), (dict(M=-1), SHAPE), (dict(N=-1), SHAPE), (dict(K=0), SHAPE), (dict(K=100), SHAPE), (dict(K=(1 << 22) + 32), SHAPE), (dict(M=(1 << 21) + 1), SHAPE),
        (dict(N=(1 << 23) + 1), SHAPE), (dict(x=null), NULL), (dict(q=null), NULL), (dict(s=null), NULL), (dict(y=null), NULL), (dict(x_rs=-1), STRIDE),
        (dict(x_rs=(1 << 23) + 2), STRIDE), (dict(x_rs=257), ALIGN), (dict(x=at(4098)), ALIGN), (dict(q=at(4104)), ALIGN), (dict(y=at(4097)), ALIGN), (dict(M=0, x=null), OK),
        (dict(N=0, y=null), OK)])


def test_experts_entry_point_refuses():
    lib = _lib.load()
    need = lib.dlb_few_token_experts_workspace_bytes(4, 2, 256)
    assert need == 4 * 2 * 256 * 4 and lib.dlb_few_token_experts_workspace_bytes(0, 2, 256) == 0
    good = dict(x=fake, x_rs=128, dt=0, ids=fake, i_dt=0, s0=2, s1=1, w=fake, kind=0, up=fake, up_s=fake, down=fake, down_s=fake, out=fake, T=4, topk=2, E=8, H=128, I=256, ws=fake,
                wsb=need, st=null)
    refused('dlb_few_token_experts', good, [
        (dict(dt=2), DTYPE), (dict(i_dt=2), DTYPE), (dict(kind=2), DTYPE), (dict(T=-1), SHAPE), (dict(T=65), SHAPE), (dict(topk=0), SHAPE), (dict(topk=17), SHAPE), (dict(E=0), SHAPE),
        (dict(E=1025), SHAPE), (dict(H=96), SHAPE), (dict(I=96), SHAPE), (dict(I=0), SHAPE), (dict(kind=1, H=48), SHAPE), (dict(kind=1, I=48), SHAPE), (dict(H=(1 << 20) + 128), SHAPE),
        (dict(I=(1 << 20) + 128), SHAPE), (dict(T=64, topk=16, I=1 << 20), SHAPE), (dict(x=null), NULL), (dict(ids=null), NULL), (dict(w=null), NULL), (dict(up=null), NULL),
        (dict(up_s=null), NULL), (dict(down=null), NULL), (dict(down_s=null), NULL), (dict(out=null), NULL), (dict(x_rs=-2), STRIDE), (dict(x_rs=(1 << 23) + 2), STRIDE),
        (dict(s0=-1), STRIDE), (dict(s1=-1), STRIDE), (dict(x=at(4098)), ALIGN), (dict(x_rs=129), ALIGN), (dict(ids=at(4098)), ALIGN), (dict(i_dt=1, ids=at(4100)), ALIGN),
        (dict(w=at(4098)), ALIGN), (dict(up=at(4104)), ALIGN), (dict(down=at(4104)), ALIGN), (dict(up_s=at(4098)), ALIGN), (dict(down_s=at(4098)), ALIGN), (dict(out=at(4097)), ALIGN),
        (dict(ws=null), WORKSPACE), (dict(wsb=need - 1), WORKSPACE), (dict(ws=at(4098)), ALIGN), (dict(T=0, x=null), OK), (dict(H=0, out=null), OK)])


# ---- the Python functions ----------------------------------------------------------------------------------------------


def zeros(*size, dtype=bf16):
    return torch.zeros(size, dtype=dtype)


def coded(*size):
    return zeros(*size[:-1], size[-1] // 2, dtype=u8), zeros(*size[:-1], size[-1] // 32, dtype=u8)


def f8s(E, N, K):
    return zeros(E, N, K, dtype=u8).view(f8), zeros(E, -(-N // 128), K // 128, dtype=f32)


def experts(x=None, ids=None, weights=None, w13=None, w2=None):
    pick = lambda given, otherwise: otherwise if given is None else given
    return few_token_experts(pick(x, zeros(3, 256)), pick(ids, zeros(3, 2, dtype=i32)), pick(weights, zeros(3, 2, dtype=f32)), pick(w13, f8s(4, 256, 256)), pick(w2, f8s(4, 256, 128)))


(Q, S), (A, A_S) = coded(8, 64), coded(3, 64)
STRIDED = torch.zeros(32, 8, dtype=u8).t()


@pytest.mark.parametrize('call,error', [
    (lambda: layer_norm(zeros(2, 8, dtype=f64), zeros(8)), TypeError),
    (lambda: layer_norm(zeros(2, 8), zeros(8, dtype=f16)), TypeError),
    (lambda: layer_norm(zeros(2, 8), zeros(8), zeros(8, dtype=f32)), TypeError),
    (lambda: layer_norm(zeros(2, 8), zeros(8, dtype=f32), zeros(8)), TypeError),
    (lambda: layer_norm(zeros(2, 8), zeros(7)), ValueError),
    (lambda: layer_norm(zeros(2, 8), zeros(8), zeros(7)), ValueError),
    (lambda: layer_norm(zeros(2, 8), zeros(8), zeros(1, 8)), ValueError),
    (lambda: layer_norm(zeros(2, 8), zeros(8), None, 1e-5, zeros(3, 8)), ValueError),
    (lambda: layer_norm(zeros(2, 8), zeros(8), None, 1e-5, zeros(2, 8, dtype=f16)), ValueError),
    (lambda: layer_norm(zeros(2, 8), zeros(8), None, -1.0), ValueError),
    (lambda: layer_norm(zeros(2, 8), zeros(8), None, float('nan')), ValueError),
    (lambda: layer_norm(zeros(2, 0), zeros(0)), ValueError),
    (lambda: layer_norm(zeros(2, 32776), zeros(32776)), ValueError),
    (lambda: per_group_quant_mxfp4(zeros(2, 64, dtype=f64)), TypeError),
    (lambda: per_group_quant_mxfp4(zeros(2, 48)), ValueError),
    (lambda: per_group_quant_mxfp4(zeros(2, 0)), ValueError),
    (lambda: per_group_quant_mxfp4(torch.tensor(1.0)), ValueError),
    (lambda: per_group_quant_mxfp4(torch.empty(0, (1 << 22) + 32)), ValueError),
    (lambda: per_group_quant_mxfp4(zeros(2, 64).requires_grad_()), NotImplementedError),
    (lambda: mxfp4_gemm(A, Q, A_S, S, f64), TypeError),
    (lambda: mxfp4_gemm(A.view(torch.int8), Q, A_S, S, bf16), TypeError),
    (lambda: mxfp4_gemm(A, Q, A_S, S.float(), bf16), TypeError),
    (lambda: mxfp4_gemm(A, Q, A_S, S[:7], bf16), ValueError),
    (lambda: mxfp4_gemm(A, Q, A_S[:, :1].contiguous(), S, bf16), ValueError),
    (lambda: mxfp4_gemm(A, Q[0], A_S, S[0], bf16), ValueError),
    (lambda: mxfp4_gemm(A[0], Q, A_S, S, bf16), ValueError),
    (lambda: mxfp4_gemm(A, coded(8, 128)[0], A_S, coded(8, 128)[1], bf16), ValueError),
    (lambda: mxfp4_gemm(A, STRIDED, A_S, S, bf16), AssertionError),
    (lambda: mxfp4_gemm(zeros(3, 8, dtype=u8), zeros(8, 8, dtype=u8), zeros(3, 0, dtype=u8), zeros(8, 0, dtype=u8), bf16), ValueError),
    (lambda: mxfp4_weight_gemm(zeros(3, 64, dtype=f32), Q, S), TypeError),
    (lambda: mxfp4_weight_gemm(zeros(3, 96), Q, S), ValueError),
    (lambda: mxfp4_weight_gemm(zeros(3, 64), Q, S[:, :1].contiguous()), ValueError),
    (lambda: mxfp4_weight_gemm(zeros(3, 64), STRIDED, S), AssertionError),
    (lambda: mxfp4_weight_gemm(zeros(3, 64), Q.view(1, 8, 32), S.view(1, 8, 2)), ValueError),
    (lambda: mxfp4_weight_gemm(zeros(3, 64).requires_grad_(), Q, S), NotImplementedError),
    (lambda: experts(x=zeros(3, 256, dtype=f32)), TypeError),
    (lambda: experts(x=zeros(1, 3, 256)), ValueError),
    (lambda: experts(x=zeros(4, 256)), ValueError),
    (lambda: experts(x=zeros(65, 256), ids=zeros(65, 2, dtype=i32), weights=zeros(65, 2, dtype=f32)), ValueError),
    (lambda: experts(ids=zeros(3, 17, dtype=i32), weights=zeros(3, 17, dtype=f32)), ValueError),
    (lambda: experts(ids=zeros(3, 0, dtype=i32), weights=zeros(3, 0, dtype=f32)), ValueError),
    (lambda: experts(ids=zeros(3, 2, dtype=torch.int16)), TypeError),
    (lambda: experts(weights=zeros(3, 2)), TypeError),
    (lambda: experts(weights=zeros(3, 1, dtype=f32)), ValueError),
    (lambda: experts(w13=coded(4, 256, 256)), TypeError),
    (lambda: experts(w13=f8s(4, 255, 256)), ValueError),
    (lambda: experts(w13=f8s(4, 256, 128)), ValueError),
    (lambda: experts(w13=f8s(3, 256, 256)), ValueError),
    (lambda: experts(w2=f8s(4, 128, 128)), ValueError),
    (lambda: experts(w13=(f8s(4, 256, 256)[0], zeros(4, 2, 1, dtype=f32))), ValueError),
    (lambda: experts(w13=(f8s(4, 256, 256)[0], zeros(4, 2, 2))), TypeError),
    (lambda: experts(w13=coded(4, 256, 256)[:1] + (zeros(4, 256, 8, dtype=f32), ), w2=coded(4, 256, 128)), TypeError),
    (lambda: experts(x=zeros(3, 96), w13=f8s(4, 256, 96), w2=f8s(4, 96, 128)), ValueError),
    (lambda: experts(w13=f8s(1025, 2, 256), w2=f8s(1025, 256, 1)), ValueError),
    (lambda: experts(w13=f8s(0, 256, 256), w2=f8s(0, 256, 128)), ValueError),
    (lambda: experts(w13=(f8s(4, 256, 256)[0].transpose(1, 2), f8s(4, 256, 256)[1])), AssertionError),
    (lambda: experts(x=zeros(3, 256).requires_grad_()), NotImplementedError),
    (lambda: experts(weights=zeros(3, 2, dtype=f32).requires_grad_()), NotImplementedError),
])
def test_python_functions_refuse(call, error):
    with pytest.raises(error):
        call()


# ---- the definitions -----------------------------------------------------------------------------------------------------


def test_layer_norm_gradient_is_the_differences_of_the_norm():
    """Central differences in 64 bits: a step of 1e-5 leaves h^2 / 6 times third derivatives, far below 1e-6 of numbers around one, and 1e-16 / 1e-5."""
    g = torch.Generator().manual_seed(3)
    h, dy, dsum = (torch.randn(3, 9, generator=g, dtype=f64) for _ in range(3))
    w, b = (torch.randn(9, generator=g, dtype=f64) for _ in range(2))
    grads, _ = norm_orc.layer_norm_grad(dy, dsum, h, w, 1e-5)
    value = lambda h, w, b: float((norm_orc.layer_norm(h, w, b, 1e-5)[0] * dy).sum() + (h * dsum).sum())
    for which, (t, grad) in enumerate(zip((h, w, b), grads)):
        for i in range(t.numel()):
            by = []
            for step in (1e-5, -1e-5):
                moved = [v.clone() for v in (h, w, b)]
                moved[which].view(-1)[i] += step
                by.append(value(*moved))
            assert abs((by[0] - by[1]) / 2e-5 - float(grad.reshape(-1)[i])) < 1e-6


def test_4_bit_floating_point_by_hand():
    q, s = orc.quant(torch.tensor([[6.0, -3.0, 2.5, 0.25] + [0.0] * 28, [0.7, 0.0, -0.1, 7.0] + [0.0] * 28]))
    assert s.tolist() == [[127], [127]]
    assert q[0, :2].tolist() == [0x7 | 0xd << 4, 0x4 | 0x0 << 4]  # 2.5 between 2 and 3, 0.25 between 0 and 0.5: to the even codes
    assert q[1, :2].tolist() == [0x1, 0x8 | 0x7 << 4]  # 0.7 to 0.5, -0.1 to -0, 7 to 6
    assert orc.values(q, s)[0, :4].tolist() == [6.0, -3.0, 2.0, 0.0]
    x = torch.randn(5, 96, generator=torch.Generator().manual_seed(1))
    q, s = orc.quant(x)
    scale = torch.exp2(s.double() - 127).repeat_interleave(32, 1)
    off = (orc.values(q, s) - x.double()).abs()
    assert bool((off <= torch.where(x.abs() <= 6 * scale, (x.abs().double() / 4).clamp_min(scale / 4), x.abs().double() - 6 * scale + 1e-12)).all())  # half a step of one bit, below 1 of 0.5


def test_experts_are_the_products_by_hand():
    g = torch.Generator().manual_seed(2)
    w13, w2, x = torch.randn(3, 8, 6, generator=g, dtype=f64), torch.randn(3, 6, 4, generator=g, dtype=f64), torch.randn(2, 6, generator=g, dtype=f64)
    out, bound = orc.experts(x, torch.tensor([[2, -1], [1, 1]]), torch.tensor([[0.5, 9.0], [0.25, 0.5]]), w13, w2)
    one = lambda e, v: w2[e] @ (torch.nn.functional.silu(w13[e, :4] @ v) * (w13[e, 4:] @ v))
    assert torch.allclose(out, torch.stack([0.5 * one(2, x[0]), 0.75 * one(1, x[1])]), atol=1e-12) and bool((bound > 0).all()) and math.isfinite(float(bound.max()))
