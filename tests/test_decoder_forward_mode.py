"""Forward-mode derivatives of the steps around the products: the ops write into outputs that no tangent follows, so a tensor with a
tangent is refused instead of coming back without one."""
import pytest
import torch
from torch.autograd import forward_ad

from dlblas_amd.kernels.moe_permute import MoePermutation, moe_permute, moe_unpermute
from dlblas_amd.kernels.rms_norm import rms_norm, rms_norm_quant
from dlblas_amd.kernels.w4_gemm import per_group_quant_w4, w4_gemm, w4_gemm_grouped

bf16, f32, i32, u8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8


def made(dev):
    """name -> (call of one tensor, that tensor)"""
    z = lambda *size, dtype=f32: torch.zeros(size, dtype=dtype, device=dev)
    x, w = z(4, 128) + 1, z(128) + 1
    x16, s16 = x.to(bf16), z(8, 1, dtype=bf16)
    q, q3 = z(8, 64, dtype=u8), z(2, 8, 64, dtype=u8)
    ids, start, end = z(4, 1, dtype=i32), z(2, dtype=i32), z(2, dtype=i32) + 4  # the first expert has all rows, the second none
    start[1] = 4
    p = MoePermutation(z(4, 1, dtype=i32), z(4, dtype=i32), z(4, dtype=i32), z(1, dtype=i32), z(1, dtype=i32))
    return {
        'norm x': (lambda t: rms_norm(t, w), x),
        'norm weight': (lambda t: rms_norm(x, t), w),
        'norm residual': (lambda t: rms_norm(x, w, 1e-6, t)[0], x),
        'norm with quantiser': (lambda t: rms_norm_quant(t, w)[1], x),
        'permute': (lambda t: moe_permute(t, ids, 2)[0], x),
        'permute scales': (lambda t: moe_permute((z(4, 128, dtype=u8).view(torch.float8_e4m3fn), t), ids, 2)[0][1], z(4, 1) + 1),
        'unpermute rows': (lambda t: moe_unpermute(t, p), x),
        'unpermute rows by a table': (lambda t: moe_unpermute(t, p.row_index), x),
        'unpermute weights': (lambda t: moe_unpermute(x, p, t), z(4, 1) + 1),
        'w4 x': (lambda t: w4_gemm(t, q, s16), x16),
        'w4 scales': (lambda t: w4_gemm(x16, q, t), s16),
        'w4 by expert': (lambda t: w4_gemm_grouped(t, q3, s16.expand(2, 8, 1).contiguous(), start, end), x16),
        'w4 quantiser': (lambda t: per_group_quant_w4(t)[1], x16),
    }


NAMES = list(made('cpu'))


def refused(call, x):
    """Without a gradient wanted in reverse too, and with one."""
    for leaf in (x, x.clone().requires_grad_()):
        with forward_ad.dual_level():
            with pytest.raises(NotImplementedError, match='forward-mode'):
                call(forward_ad.make_dual(leaf, torch.ones_like(x)))
    with pytest.raises(NotImplementedError, match='forward-mode'):
        torch.func.jvp(call, (x, ), (torch.ones_like(x), ))
    with pytest.raises(NotImplementedError, match='forward-mode'):
        torch.func.jacfwd(call)(x)


@pytest.mark.parametrize('name', NAMES)
def test_a_tangent_is_refused(name):
    refused(*made('cpu')[name])


@pytest.mark.gpu
@pytest.mark.parametrize('name', NAMES)
def test_a_tangent_is_refused_on_the_gpu(name):
    call, x = made(torch.device('cuda:0'))[name]
    refused(call, x)
    with forward_ad.dual_level():  # a level alone changes nothing
        assert torch.equal(call(x), call(x))


@pytest.mark.gpu
@pytest.mark.parametrize('native', [True, False])
@pytest.mark.parametrize('name', ['norm x', 'norm residual', 'permute', 'unpermute rows'])
def test_a_gradient_with_a_tangent_is_refused(name, native, monkeypatch):
    from dlblas_amd import _fast
    if not native:
        for fn in ('rms_norm', 'moe_permute', 'moe_unpermute'):
            monkeypatch.setattr(_fast, fn, lambda *a: None)
    call, x = made(torch.device('cuda:0'))[name]
    x = x.clone().requires_grad_()
    y = call(x)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match='forward-mode'):
            torch.autograd.grad(y, x, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))
