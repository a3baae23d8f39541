"""The gradients of the steps around the products inside what torch lays around a graph: hooks on saved tensors, checkpointing, anomaly
mode, gradients that are batched.  Everything is compared bit for bit with the same call without it."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from dlblas_amd.kernels.moe_permute import moe_permute, moe_unpermute
from dlblas_amd.kernels.rms_norm import rms_norm

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16
T, H, E, TOPK = 20, 136, 5, 3


@pytest.fixture(scope='module')
def dev():
    return torch.device('cuda:0')


def leaves(dev):
    g = torch.Generator().manual_seed(11)
    x, res = (torch.randn(T, H, generator=g).to(bf16).to(dev).requires_grad_() for _ in range(2))
    w = (1 + 0.1 * torch.randn(H, generator=g)).to(bf16).to(dev).requires_grad_()
    weights = torch.rand(T, TOPK, generator=g).to(dev).requires_grad_()
    return x, w, res, weights


def routing(dev):
    return torch.randint(-1, E, (T, TOPK), generator=torch.Generator().manual_seed(12)).to(dev)


def norm(x, w, res, weights):
    return rms_norm(x, w)


def norm_with_residual(x, w, res, weights):
    y, h = rms_norm(x, w, 1e-6, res)
    return y + h


def permute(x, w, res, weights):
    return moe_permute(x, routing(x.device), E, 4)[0]


def back_alone(x, w, res, weights):
    """A fixed permutation: the rows are the input."""
    with torch.no_grad():
        _, p = moe_permute(x, routing(x.device), E)
    return moe_unpermute(x.repeat(TOPK, 1)[:p.source.numel()], p, weights)


def block(x, w, res, weights):
    y, h = rms_norm(x, w, 1e-6, res)
    rows, p = moe_permute(y, routing(x.device), E, 4)
    return moe_unpermute(rows, p, weights) + h


STEPS = [norm, norm_with_residual, permute, back_alone, block]


def gradients(fn, dev, around=None):
    ins = leaves(dev)
    out = fn(*ins) if around is None else around(fn, ins)
    dout = torch.randn(out.shape, generator=torch.Generator().manual_seed(13)).to(out.dtype).to(dev)
    return [out.detach()] + [g for g in torch.autograd.grad(out, ins, dout, allow_unused=True) if g is not None]


def same(got, want):
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize('fn', STEPS)
def test_hooks_on_saved_tensors(dev, fn):
    want = gradients(fn, dev)
    packed, unpacked = [], []

    def around(fn, ins):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: (packed.append(t.shape), t.cpu())[1], lambda t: (unpacked.append(t.shape), t.to(dev))[1]):
            return fn(*ins)

    same(gradients(fn, dev, around), want)
    assert packed and unpacked


@pytest.mark.parametrize('reentrant', [False, True])
@pytest.mark.parametrize('fn', STEPS)
def test_checkpointed(dev, fn, reentrant):
    """A recomputation ends with an exception of torch's own, raised by the hook that packs the last saved tensor."""
    if reentrant:  # reaches gradients through backward() alone

        def by_backward(call):
            ins = leaves(dev)
            out = call(*ins)
            out.backward(torch.randn(out.shape, generator=torch.Generator().manual_seed(13)).to(out.dtype).to(dev))
            return [out.detach()] + [t.grad for t in ins if t.grad is not None]

        same(by_backward(lambda *ins: checkpoint(fn, *ins, use_reentrant=True)), by_backward(fn))
        return
    same(gradients(fn, dev, lambda fn, ins: checkpoint(fn, *ins, use_reentrant=False)), gradients(fn, dev))


@pytest.mark.parametrize('fn', STEPS)
def test_an_exception_of_a_hook_keeps_its_type(dev, fn):
    class Mine(Exception):
        pass

    def pack(t):
        raise Mine('while packing')

    with pytest.raises(Mine, match='while packing'):
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            fn(*leaves(dev))
    same(gradients(fn, dev), gradients(fn, dev))  # and nothing is left behind


@pytest.mark.parametrize('fn', STEPS)
def test_anomaly_mode(dev, fn):
    want = gradients(fn, dev)
    with torch.autograd.detect_anomaly(check_nan=True):
        same(gradients(fn, dev), want)


@pytest.mark.parametrize('fn', [norm, norm_with_residual, permute, back_alone])
def test_batched_gradients_are_refused(dev, fn):
    ins = leaves(dev)
    out = fn(*ins)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, ins, torch.ones((2, ) + out.shape, dtype=bf16, device=dev), is_grads_batched=True, allow_unused=True)


def spread(t):
    """The same values in another layout."""
    wide = t.new_zeros(t.shape + (3, ))
    wide[..., 1] = t
    return wide[..., 1]


CHANGES = {
    'another device': lambda t: t.cpu(),
    'another type': lambda t: t.double() if t.is_floating_point() else t.long(),
    'a narrower type': lambda t: t.half() if t.is_floating_point() else t.short(),
    'fewer elements': lambda t: t[:1],
    'another shape': lambda t: t.reshape(-1, 1),
}


@pytest.mark.parametrize('native', [True, False])
@pytest.mark.parametrize('change', list(CHANGES) + ['another layout'])
@pytest.mark.parametrize('fn,saved,which', [(fn, n, i) for fn, n in ((norm, 2), (norm_with_residual, 2), (permute, 1), (back_alone, 4)) for i in range(n)])
def test_what_a_hook_gives_back_is_looked_at(dev, fn, saved, which, change, native, monkeypatch):
    """The kernels are told nothing but addresses: a saved tensor that is another one raises before anything is enqueued, one that lies
    differently is the same."""
    if not native:
        from dlblas_amd import _fast
        for name in ('rms_norm', 'moe_permute', 'moe_unpermute'):
            monkeypatch.setattr(_fast, name, lambda *a: None)
    want = gradients(fn, dev)
    count = [0]

    def around(fn, ins):
        if fn is back_alone:  # repeat() saves nothing
            rows = ins[0].repeat(TOPK, 1)
            with torch.no_grad():
                _, p = moe_permute(ins[0], routing(dev), E)
            call = lambda: moe_unpermute(rows[:p.source.numel()], p, ins[3])
        else:
            call = lambda: fn(*ins)

        def pack(t):
            count[0] += 1
            return count[0] - 1, t

        def unpack(packed):
            n, t = packed
            if n != which:
                return t
            return spread(t) if change == 'another layout' else CHANGES[change](t)

        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            return call()

    if change == 'another layout':
        same(gradients(fn, dev, around), want)
        return
    with pytest.raises(RuntimeError, match='came back from its hook'):
        gradients(fn, dev, around)
    assert count[0] == saved
