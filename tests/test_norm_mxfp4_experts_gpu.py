"""Layer norm, products in 4-bit floating point and the experts for a few tokens together, as a layer uses them: served, captured into graphs, on other
streams, from several threads; the norm's gradient inside what torch lays around a graph; sizes at the ends of what is allowed and beyond 32 bits.

Every stage of the layer is compared with its definition in 64 bits on what the stage before it really left, so a stage's tolerance is its own: the
bounds of oracle/layer_norm.py and oracle/mxfp4.py, and half a step of the stored type."""
import threading

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils.checkpoint import checkpoint

from dlblas_amd import _fast
from dlblas_amd.kernels.few_token_experts import few_token_experts
from dlblas_amd.kernels.layer_norm import layer_norm
from dlblas_amd.kernels.mxfp4_gemm import mxfp4_gemm, mxfp4_weight_gemm, per_group_quant_mxfp4
from oracle import layer_norm as norm_orc
from oracle import mxfp4 as orc
from oracle.decoder import norm_input

pytestmark = pytest.mark.gpu
bf16, f16, f32, f64, i32, u8, f8 = torch.bfloat16, torch.float16, torch.float32, torch.float64, torch.int32, torch.uint8, torch.float8_e4m3fn
EPS = 1e-5


@pytest.fixture(scope='module')
def dev():
    return torch.device('cuda:0')


def inside(got, want, bound, what):
    step = torch.finfo(got.dtype).eps / 2
    off = (got.detach().cpu().double() - want).abs() - (bound * (1 + step) + step * want.abs() + torch.finfo(got.dtype).smallest_normal * step)
    assert float(off.max()) <= 0, f'{what}: {float(off.max()):.3e} beyond the bound'


def codes(size, K, g, middle=122, spread=2):
    return torch.randint(0, 256, size + (K // 2, ), generator=g, dtype=u8), torch.randint(middle - spread, middle + spread, size + (K // 32, ), generator=g, dtype=u8)


def product_bound(K, mag):
    """The sums over K / 32 groups: K / 32 + 8 additions, each off by at most 2^-23 of the sum of magnitudes."""
    return (K / 32 + 8) * 2 * orc.FP32 * mag


class Layer:
    """Norm, a quantised product, the residual's norm, experts and a product beside them: H columns, E experts of I."""

    def __init__(self, dev, kind, H=256, I=128, E=6, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.H, self.I, self.E = H, I, E
        self.norms = [((1 + 0.1 * torch.randn(H, generator=g)).to(bf16), (0.1 * torch.randn(H, generator=g)).to(bf16)) for _ in range(2)]
        self.mix, self.head = codes((H, ), H, g), codes((96, ), H, g)
        if kind == 'f4':
            self.up, self.down = codes((E, 2 * I), H, g), codes((E, H), I, g)
        else:
            self.up, self.down = ((torch.randn(E, n, k, generator=g).to(f8), 0.01 + 0.02 * torch.rand(E, -(-n // 128), k // 128, generator=g)) for n, k in ((2 * I, H), (H, I)))
        self.on = {k: tuple(t.to(dev) for t in getattr(self, k)) for k in ('mix', 'head', 'up', 'down')}
        self.norms_on = [tuple(t.to(dev) for t in n) for n in self.norms]

    def serve(self, x, res, ids, weights):
        y, h = layer_norm(x, *self.norms_on[0], EPS, res)
        q, s = per_group_quant_mxfp4(y)
        mixed = mxfp4_gemm(q, self.on['mix'][0], s, self.on['mix'][1], bf16)
        y2, h2 = layer_norm(mixed, *self.norms_on[1], EPS, h)
        out = dict(y=y, h=h, q=q, s=s, mixed=mixed, y2=y2, h2=h2, beside=mxfp4_weight_gemm(y2, *self.on['head']))
        if x.size(0) <= 64:
            out['out'] = few_token_experts(y2, ids, weights, self.on['up'], self.on['down'])
        return out


def batch(T, H, E, topk, seed=0):
    g = torch.Generator().manual_seed(1000 + 7 * T + seed)
    ids = torch.randint(0, E + 2, (T, topk), generator=g)  # a quarter of the slots are elsewhere
    ids[ids == E + 1] = -1
    return torch.randn(T, H, generator=g).to(bf16), torch.randn(T, H, generator=g).to(bf16), ids, torch.rand(T, topk, generator=g)


@pytest.mark.parametrize('kind', ['f8', 'f4'])
@pytest.mark.parametrize('T', [1, 7, 40, 150])
def test_a_layer(dev, T, kind):
    layer = Layer(dev, kind)
    x, res, ids, weights = batch(T, layer.H, layer.E, 3)
    on = layer.serve(*(t.to(dev) for t in (x, res, ids, weights)))
    b = {k: v.cpu() for k, v in on.items()}
    assert torch.equal(b['h'], norm_input(x, res))
    inside(on['y'], *norm_orc.layer_norm(b['h'], *layer.norms[0], EPS), 'norm')
    q, s = orc.quant(b['y'])
    assert torch.equal(b['q'], q) and torch.equal(b['s'], s)
    want, mag = orc.gemm(q, s, *layer.mix)
    inside(on['mixed'], want, product_bound(layer.H, mag), 'product')
    assert torch.equal(b['h2'], norm_input(b['mixed'], b['h']))
    inside(on['y2'], *norm_orc.layer_norm(b['h2'], *layer.norms[1], EPS), 'second norm')
    w, rows = orc.values(*layer.head), b['y2'].double()
    inside(on['beside'], rows @ w.t(), (layer.H + 16) * 2 * orc.FP32 * (rows.abs() @ w.abs().t()), 'product beside them')
    if T <= 64:
        numbers = (orc.values if kind == 'f4' else orc.e4m3_values)
        inside(on['out'], *orc.experts(b['y2'], ids, weights, numbers(*layer.up), numbers(*layer.down)), 'experts')


@pytest.mark.parametrize('kind', ['f8', 'f4'])
@pytest.mark.parametrize('T', [1, 20, 200])
def test_a_captured_layer_replays(dev, T, kind):
    layer = Layer(dev, kind, H=288 if kind == 'f4' else 256)  # 288: scales in rows that are no whole words
    fixed = [t.to(dev) for t in batch(T, layer.H, layer.E, 2)]
    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        layer.serve(*fixed)
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = layer.serve(*fixed)
    for seed in range(4):
        fresh = [t.to(dev) for t in batch(T, layer.H, layer.E, 2, seed)]
        for to, t in zip(fixed, fresh):
            to.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want = layer.serve(*fresh)  # eager work of the same kind between the replays
        torch.cuda.synchronize()
        for name in want:
            assert torch.equal(held[name], want[name]), (seed, name)


def test_a_captured_gradient_replays(dev):
    g = torch.Generator().manual_seed(1)
    start = [torch.randn(50, 264, generator=g).to(dev) for _ in range(4)] + [torch.randn(264, generator=g).to(dev) for _ in range(2)]

    def step(x, res, gy, gh, w, b):
        return torch.autograd.grad(layer_norm(x, w, b, EPS, res), (x, res, w, b), (gy, gh))

    def fresh(scale):
        """Leaves of their own: no eager graph of them is alive when the capture runs."""
        t = [v.clone() for v in start]
        t[0].mul_(scale)
        for i in (0, 1, 4, 5):
            t[i].requires_grad_()
        return t

    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step(*fresh(1.0))
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    fixed = fresh(1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(*fixed)
    for scale in (1.0, 0.5, 3.0, 1.0):
        with torch.no_grad():
            fixed[0].copy_(start[0] * scale)
        graph.replay()
        torch.cuda.synchronize()
        want = step(*fresh(scale))
        torch.cuda.synchronize()
        for got, ref in zip(held, want):
            assert torch.equal(got, ref), scale


@pytest.mark.parametrize('which', ['experts', 'scales laid out anew'])
def test_two_graphs_in_flight_at_once(dev, which):
    """What lies between two kernels is in scratch of the call's own."""
    g = torch.Generator().manual_seed(0)
    calls = []
    for i in range(2):
        if which == 'experts':
            up, down = (tuple(t.to(dev) for t in codes((8, n), k, g)) for n, k in ((1024, 1024), (1024, 512)))
            args = (torch.randn(16, 1024, generator=g).to(bf16).to(dev), torch.randint(0, 8, (16, 4), generator=g).to(dev), torch.rand(16, 4, generator=g).to(dev), up, down)
            calls.append(lambda args=args: few_token_experts(*args))
        else:
            a, b = (tuple(t.to(dev) for t in codes((n, ), 1056, g)) for n in (3000, 2900))
            calls.append(lambda a=a, b=b: mxfp4_gemm(a[0], b[0], a[1], b[1], bf16))
    want = [call() for call in calls]
    graphs, held = [], []
    for call in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(call())
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    for _ in range(5):
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for got, ref in zip(held, want):
            assert torch.equal(got, ref)


def test_a_layer_on_a_stream_of_its_own(dev):
    layer = Layer(dev, 'f8')
    inputs = [t.to(dev) for t in batch(60, layer.H, layer.E, 4)]
    want = layer.serve(*inputs)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(device=dev)
    with torch.cuda.stream(side):
        late = [t.clone() for t in inputs]  # made on that stream, so a call on another one would come too early
        got = layer.serve(*late)
    side.synchronize()
    for name in want:
        assert torch.equal(got[name], want[name]), name


def test_layers_from_threads(dev):
    layers = [Layer(dev, kind) for kind in ('f8', 'f4', 'f4')]
    sets = [[t.to(dev) for t in batch(T, 256, 6, 4)] for T in (3, 50, 300)]
    want = [layer.serve(*s) for layer, s in zip(layers, sets)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream(device=dev)):
                for _ in range(5):
                    got = layers[i].serve(*sets[i])
                    torch.cuda.current_stream().synchronize()
                    wrong.extend((i, name) for name in got if not torch.equal(got[name], want[i][name]))
        except Exception as e:  # noqa: BLE001
            wrong.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i, )) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize('kind', ['serve', 'train'])
def test_under_the_tracing_compiler(dev, kind):
    """The Python functions trace into one graph of the registered ops; the numbers are those of the native calls."""
    layer = Layer(dev, 'f8')
    x, res, ids, weights = (t.to(dev) for t in batch(20, layer.H, layer.E, 2))

    def train(x):
        y, h = layer_norm(x, *layer.norms_on[0], EPS, res)
        return layer_norm(y + h, layer.norms_on[1][0])

    fn = train if kind == 'train' else lambda x: tuple(layer.serve(x, res, ids, weights).values())
    torch._dynamo.reset()
    traced = torch.compile(fn, backend='aot_eager', fullgraph=True)
    if kind == 'train':
        leaf, other = x.clone().requires_grad_(), x.clone().requires_grad_()
        assert torch.equal(*(torch.autograd.grad(f(t), t, res)[0] for f, t in ((traced, leaf), (fn, other))))
    else:
        for a, b in zip(traced(x), fn(x)):
            assert torch.equal(a, b)
    torch._dynamo.reset()


# ---- the norm's gradient inside what torch lays around a graph ------------------------------------------------------------


def leaves(dev):
    g = torch.Generator().manual_seed(11)
    x, res = (torch.randn(20, 136, generator=g).to(bf16).to(dev).requires_grad_() for _ in range(2))
    w, b = ((k + 0.1 * torch.randn(136, generator=g)).to(bf16).to(dev).requires_grad_() for k in (1, 0))
    return x, w, b, res


def norm(x, w, b, res):
    return layer_norm(x, w, b)


def norm_with_residual(x, w, b, res):
    y, h = layer_norm(x, w, b, EPS, res)
    return y + h


STEPS = [norm, norm_with_residual]


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
def test_hooks_checkpoints_and_anomaly_mode(dev, fn):
    want = gradients(fn, dev)
    packed = []

    def around(fn, ins):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: (packed.append(t.shape), t.cpu())[1], lambda t: t.to(dev)):
            return fn(*ins)

    same(gradients(fn, dev, around), want)
    assert len(packed) == 3
    same(gradients(fn, dev, lambda fn, ins: checkpoint(fn, *ins, use_reentrant=False)), want)
    with torch.autograd.detect_anomaly(check_nan=True):
        same(gradients(fn, dev), want)

    class Mine(Exception):
        pass

    def pack(t):
        raise Mine('while packing')

    with pytest.raises(Mine, match='while packing'):
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            fn(*leaves(dev))
    same(gradients(fn, dev), want)  # and nothing is left behind
    ins = leaves(dev)
    out = fn(*ins)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, ins, torch.ones((2, ) + out.shape, dtype=bf16, device=dev), is_grads_batched=True, allow_unused=True)
    x = leaves(dev)[0]
    grad, = torch.autograd.grad(fn(x, *leaves(dev)[1:]).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(grad.float().sum(), x)


def spread(t):
    """The same values in another layout."""
    wide = t.new_zeros(t.shape + (3, ))
    wide[..., 1] = t
    return wide[..., 1]


CHANGES = {
    'another device': lambda t: t.cpu(),
    'another type': lambda t: t.double(),
    'a narrower type': lambda t: t.half(),
    'fewer elements': lambda t: t[:1],
    'another shape': lambda t: t.reshape(-1, 1),
    'another layout': spread,
}


@pytest.mark.parametrize('native', [True, False])
@pytest.mark.parametrize('change', list(CHANGES))
@pytest.mark.parametrize('which', range(3))
@pytest.mark.parametrize('fn', STEPS)
def test_what_a_hook_gives_back_is_looked_at(dev, fn, which, change, native, monkeypatch):
    """The kernels are told nothing but addresses: a saved tensor that is another one raises before anything is enqueued, one that lies
    differently is the same."""
    if not native:
        monkeypatch.setattr(_fast, 'layer_norm', lambda *a: None)
    want = gradients(fn, dev)
    count = [0]

    def around(fn, ins):

        def pack(t):
            count[0] += 1
            return count[0] - 1, t

        with torch.autograd.graph.saved_tensors_hooks(pack, lambda packed: CHANGES[change](packed[1]) if packed[0] == which else packed[1]):
            return fn(*ins)

    if change == 'another layout':
        same(gradients(fn, dev, around), want)
        return
    with pytest.raises(RuntimeError, match='came back from its hook'):
        gradients(fn, dev, around)
    assert count[0] == 3


def test_gradients_that_are_broadcast_or_strided(dev):
    """A gradient of stride 0, of a sum; one whose columns are apart; a residual that is x itself."""
    g = torch.Generator().manual_seed(5)
    base, dy = torch.randn(6, 72, generator=g).to(dev), torch.randn(72, 6, generator=g).to(dev).t()
    w, b = torch.randn(72, generator=g).to(dev), torch.randn(72, generator=g).to(dev)
    for given in (torch.ones((), device=dev).expand(6, 72), torch.randn(72, generator=g).to(dev).expand(6, 72), dy):
        by = []
        for grad in (given, given.contiguous()):
            x = base.clone().requires_grad_()
            by.append(torch.autograd.grad(layer_norm(x, w, b), x, grad)[0])
        assert torch.equal(*by)
    x = base.clone().requires_grad_()
    y, h = layer_norm(x, w, b, EPS, x)
    got, = torch.autograd.grad(y, x, dy)
    (want, _, _), (bound, _, _) = norm_orc.layer_norm_grad(dy.cpu(), None, h.detach().cpu(), w.cpu(), EPS)
    inside(got, 2 * want, 2 * bound + 2 * orc.FP32 * want.abs(), 'twice the gradient of the sum')


def made(dev):
    """name -> (call of one tensor, that tensor)"""
    z = lambda *size, dtype=f32: torch.zeros(size, dtype=dtype, device=dev)
    x, w = z(4, 128) + 1, z(128) + 1
    ids, q, s = z(4, 1, dtype=i32), z(8, 64, dtype=u8), z(8, 4, dtype=u8)
    f8s = lambda n, k: (z(2, n, k, dtype=u8).view(f8), z(2, -(-n // 128), k // 128))
    up, down = f8s(256, 128), f8s(128, 128)
    return {
        'norm x': (lambda t: layer_norm(t, w, w), x),
        'norm weight': (lambda t: layer_norm(x, t, w), w),
        'norm bias': (lambda t: layer_norm(x, w, t), w),
        'norm residual': (lambda t: layer_norm(x, w, w, EPS, t)[0], x),
        'quantiser': (lambda t: per_group_quant_mxfp4(t)[1], x),
        'few rows': (lambda t: mxfp4_weight_gemm(t, q, s), x.to(bf16)),
        'experts x': (lambda t: few_token_experts(t, ids, x[:, :1].contiguous(), up, down), x.to(bf16)),
        'experts weights': (lambda t: few_token_experts(x.to(bf16), ids, t, up, down), z(4, 1)),
        'experts scales': (lambda t: few_token_experts(x.to(bf16), ids, x[:, :1].contiguous(), (up[0], t), down), z(2, 2, 1)),
    }


@pytest.mark.parametrize('name', list(made('cpu')))
def test_a_tangent_is_refused(dev, name):
    call, x = made(dev)[name]
    for leaf in (x, x.clone().requires_grad_()):
        with forward_ad.dual_level():
            with pytest.raises(NotImplementedError, match='forward-mode'):
                call(forward_ad.make_dual(leaf, torch.ones_like(x)))
    with pytest.raises(NotImplementedError, match='forward-mode'):
        torch.func.jvp(call, (x, ), (torch.ones_like(x), ))
    with forward_ad.dual_level():  # a level alone changes nothing
        assert torch.equal(call(x), call(x))


# ---- the ends of what is allowed ----------------------------------------------------------------------------------------


@pytest.mark.parametrize('kind', ['f8', 'f4'])
@pytest.mark.parametrize('T,E,topk', [(64, 1024, 16), (16, 1024, 16), (16, 40, 2), (16, 16, 16), (5, 1024, 16), (2, 1, 16), (1, 1024, 1)])
def test_the_largest_tables_of_routing(dev, T, E, topk, kind):
    print(f'case experts T={T} E={E} topk={topk} {kind}', flush=True)
    g = torch.Generator().manual_seed(T + E)
    H = I = 128
    x, weights = torch.randn(T, H, generator=g).to(bf16), torch.rand(T, topk, generator=g)
    if kind == 'f4':
        up, down = codes((E, 2 * I), H, g), codes((E, H), I, g)
        w13, w2 = orc.values(*up), orc.values(*down)
    else:
        up, down = (((torch.randn(E, n, 128, generator=g)).to(f8), 0.02 * (1 + torch.rand(E, n // 128, 1, generator=g))) for n in (256, 128))
        w13, w2 = orc.e4m3_values(*up), orc.e4m3_values(*down)
    on = lambda pair: tuple(t.to(dev) for t in pair)
    spread_out = torch.stack([torch.randperm(E, generator=g)[:topk] if topk <= E else torch.zeros(topk, dtype=torch.int64) for _ in range(T)])
    for ids in (spread_out, torch.full((T, topk), E - 1)):
        out = few_token_experts(x.to(dev), ids.to(dev), weights.to(dev), on(up), on(down))
        inside(out, *orc.experts(x, ids, weights, w13, w2), f'{T} tokens')


@pytest.mark.parametrize('kind', ['f8', 'f4'])
@pytest.mark.parametrize('T,dtype', [(1, f16), (6, bf16), (40, bf16), (40, f16)])
def test_long_rows(dev, T, dtype, kind):
    """Columns of x that two waves share, and halves of a workgroup's columns that an expert does not have."""
    g = torch.Generator().manual_seed(T)
    E, topk, H, I = 3, 2, 4224, 128 if kind == 'f8' else 96
    x, weights, ids = torch.randn(T, H, generator=g).to(dtype), torch.rand(T, topk, generator=g), torch.randint(0, E, (T, topk), generator=g)
    if kind == 'f4':
        up, down = codes((E, 2 * I), H, g, 118), codes((E, H), I, g, 118)
        w13, w2 = orc.values(*up), orc.values(*down)
    else:
        up, down = ((torch.randn(E, n, k, generator=g).to(f8), 0.01 * (1 + torch.rand(E, n // 128, k // 128, generator=g))) for n, k in ((2 * I, H), (H, I)))
        w13, w2 = orc.e4m3_values(*up), orc.e4m3_values(*down)
    on = lambda pair: tuple(t.to(dev) for t in pair)
    inside(few_token_experts(x.to(dev), ids.to(dev), weights.to(dev), on(up), on(down)), *orc.experts(x, ids, weights, w13, w2), f'{T} tokens')


def test_rows_and_ids_that_are_broadcast_and_weights_of_nobody(dev):
    g = torch.Generator().manual_seed(7)
    up, down = (tuple(t.to(dev) for t in codes((4, n), k, g)) for n, k in ((192, 160), (160, 96)))
    x, ids, weights = torch.randn(1, 160, generator=g).to(bf16).to(dev), torch.tensor([[3, 1]], device=dev), torch.rand(9, 2, generator=g).to(dev)
    wide = few_token_experts(x.expand(9, 160), ids.expand(9, 2), weights, up, down)
    assert torch.equal(wide, few_token_experts(x.repeat(9, 1), ids.repeat(9, 1), weights, up, down))
    flat = torch.zeros(up[1].numel() + 1, dtype=u8, device=dev)
    flat[1:] = up[1].flatten()
    assert torch.equal(wide, few_token_experts(x.repeat(9, 1), ids.repeat(9, 1), weights, (up[0], flat[1:].view(up[1].shape)), down))  # scales off their words
    ids, weights = torch.tensor([[3, -1], [7, 1], [-1, -1]], device=dev), weights[:3].clone()
    want = few_token_experts(x.repeat(3, 1), ids, weights, up, down)
    weights[0, 1], weights[1, 0], weights[2, 0] = float('nan'), float('inf'), float('nan')  # of slots that go nowhere
    got = few_token_experts(x.repeat(3, 1), ids, weights, up, down)
    assert torch.equal(got, want) and float(got[2].abs().max()) == 0.0


@pytest.mark.parametrize('columns', [128, 256])
def test_scales_off_their_words(dev, columns):
    """Contiguous tensors that start anywhere: the same product."""
    g = torch.Generator().manual_seed(columns)
    (a, a_s), (b, b_s) = (tuple(t.to(dev) for t in codes((n, ), columns, g)) for n in (70, 90))
    x = torch.randn(5, columns, generator=g).to(f16).to(dev)

    def moved(t, n):
        flat = torch.zeros(t.numel() + n, dtype=u8, device=dev)
        flat[n:] = t.flatten()
        return flat[n:].view(t.shape)

    want, few = mxfp4_gemm(a, b, a_s, b_s, f32), mxfp4_weight_gemm(x, b, b_s)
    for n in (1, 2, 3):
        assert torch.equal(mxfp4_gemm(moved(a, n), moved(b, n), moved(a_s, n), moved(b_s, n), f32), want)
        assert torch.equal(mxfp4_weight_gemm(x, b, moved(b_s, n)), few)


# few rows against many columns, blocks of rows that still fill no card, small and large tiles; whole words of scales and others
WAYS = [(9, 4130, 544), (16, 5000, 768), (32, 9000, 96), (20, 4200, 1280), (40, 4200, 544), (64, 5000, 1024), (70, 200, 1056), (130, 900, 640), (300, 1000, 640), (257, 1030, 1056),
        (1500, 1600, 640), (1411, 1633, 288), (1500, 1601, 1056)]


@pytest.mark.parametrize('M,N,K', WAYS)
def test_products_of_every_size(dev, M, N, K):
    """One row and one column have a first scale that is no number: their results alone are none, also where a row's scales end inside a word."""
    print(f'case {M}x{N}x{K}', flush=True)
    g = torch.Generator().manual_seed(M + N + K)
    (a, a_s), (b, b_s) = codes((M, ), K, g), codes((N, ), K, g)
    a_s[M // 2, 0] = b_s[N // 3, 0] = 255
    got = mxfp4_gemm(*(t.to(dev) for t in (a, b, a_s, b_s)), f32).cpu()
    nan = torch.zeros(M, N, dtype=torch.bool)
    nan[M // 2], nan[:, N // 3] = True, True
    assert torch.equal(got.isnan(), nan)
    a_s[M // 2, 0] = b_s[N // 3, 0] = 122
    want, mag = orc.gemm(a, a_s, b, b_s)
    inside(got[~nan], want[~nan], product_bound(K, mag)[~nan], f'{M}x{N}x{K}')


@pytest.mark.parametrize('M,N,K', [(3, 4200, 1024), (7, 4200, 544), (16, 4200, 256), (9, 9000, 1056), (16, 8210, 768), (40, 5000, 1024), (64, 4100, 160)])
def test_few_rows_of_every_size(dev, M, N, K):
    print(f'case {M}x{N}x{K}', flush=True)
    g = torch.Generator().manual_seed(M + N + K)
    x, (q, s) = torch.randn(M, K, generator=g).to(bf16), codes((N, ), K, g)
    w, rows = orc.values(q, s), x.double()
    inside(mxfp4_weight_gemm(*(t.to(dev) for t in (x, q, s))), rows @ w.t(), (K + 16) * 2 * orc.FP32 * (rows.abs() @ w.abs().t()), f'{M}x{N}x{K}')


def test_the_widest_rows(dev):
    K = 1 << 22
    g = torch.Generator().manual_seed(9)
    x = torch.randn(2, K, generator=g).to(bf16)
    q, s = per_group_quant_mxfp4(x.to(dev))
    want = orc.quant(x)
    assert torch.equal(q.cpu(), want[0]) and torch.equal(s.cpu(), want[1])
    w = codes((17, ), K, g)
    got, mag = orc.gemm(*want, *w)
    inside(mxfp4_gemm(q, w[0].to(dev), s, w[1].to(dev), f32), got, product_bound(K, mag), 'few rows')
    numbers = orc.values(*w)
    # columns are split over eight waves, so a sum has at most an eighth of them and a step of the unit adds 32: far below K additions
    inside(mxfp4_weight_gemm(x.to(dev), *(t.to(dev) for t in w)), x.double() @ numbers.t(), (K / 32 + 16) * 2 * orc.FP32 * (x.double().abs() @ numbers.abs().t()), 'few rows of 16 bits')


def test_norms_and_codes_whose_offsets_pass_32_bits(dev):
    T, H = 304000, 7168
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(T, H, device=dev, generator=g, dtype=bf16)
    assert x.numel() > 2**31
    w, b = (torch.randn(H, device=dev, generator=g).to(bf16) for _ in range(2))
    ends = [slice(lo, lo + 300) for lo in (0, T - 300)]
    y, h = layer_norm(x, w, b, EPS, x)
    for at in ends:
        part = x[at].clone()
        y1, h1 = layer_norm(part, w, b, EPS, part)
        assert torch.equal(y[at], y1) and torch.equal(h[at], h1)
    del y, h
    q, s = per_group_quant_mxfp4(x)
    for at in ends:
        q1, s1 = per_group_quant_mxfp4(x[at].clone())
        assert torch.equal(q[at], q1) and torch.equal(s[at], s1)
    del q, s
    x.requires_grad_()
    dx, = torch.autograd.grad(layer_norm(x, w, b), x, x.detach())
    for at in ends:
        part = x.detach()[at].clone().requires_grad_()
        assert torch.equal(dx[at], torch.autograd.grad(layer_norm(part, w, b), part, part.detach())[0])


@pytest.mark.parametrize('M,N,K', [(304000, 7168, 32), (304000, 40, 32768), (40, 304000, 32768), (70, 304000, 32736)])
def test_products_whose_offsets_pass_32_bits(dev, M, N, K):
    print(f'case {M}x{N}x{K}', flush=True)
    assert max(M * N // 2, max(M, N) * K // 2) > 2**30
    g = torch.Generator(device=dev).manual_seed(2)
    (a, a_s), (b, b_s) = ((torch.randint(0, 256, (n, K // 2), dtype=u8, device=dev, generator=g), torch.randint(120, 124, (n, K // 32), dtype=u8, device=dev, generator=g)) for n in (M, N))
    c = mxfp4_gemm(a, b, a_s, b_s, bf16)
    first, last = lambda t: t[:40].cpu(), lambda t: t[-40:].cpu()
    for rows in (first, last):
        for columns in (first, last):
            want, mag = orc.gemm(rows(a), rows(a_s), columns(b), columns(b_s))
            inside(columns(rows(c).t()).t(), want, product_bound(K, mag), f'{M}x{N}x{K}')


def test_weights_whose_offsets_pass_32_bits(dev):
    N, K, E = 480000, 18432, 600
    g = torch.Generator(device=dev).manual_seed(3)
    q = torch.randint(0, 256, (N, K // 2), dtype=u8, device=dev, generator=g)
    s = torch.randint(120, 124, (N, K // 32), dtype=u8, device=dev, generator=g)
    assert q.numel() > 2**32
    x = torch.randn(9, K, device=dev, generator=g).to(bf16)
    y = mxfp4_weight_gemm(x, q, s)
    for at in (slice(0, 20000), slice(N - 20000, N)):  # as many as make the tiles as wide
        assert torch.equal(y[:, at], mxfp4_weight_gemm(x, q[at].clone(), s[at].clone()))
    del q, s
    H, I = 2048, 2048
    up, down = (torch.randint(0, 0x7f, (E, n, k), dtype=u8, device=dev, generator=g).view(f8) for n, k in ((2 * I, H), (H, I)))
    assert up.numel() > 2**32
    up_s, down_s = (0.001 * torch.rand(E, n // 128, k // 128, device=dev, generator=g) for n, k in ((2 * I, H), (H, I)))
    ids = torch.tensor([[0, E - 1, 300, 511], [512, E - 2, E - 1, -1]], device=dev)
    weights = torch.rand(2, 4, device=dev, generator=g)
    named = [0, 300, 511, 512, E - 2, E - 1]
    renamed = torch.tensor([[0, 5, 1, 2], [3, 4, 5, -1]], device=dev)
    small = [t.view(u8)[named].view(t.dtype) if t.dtype == f8 else t[named] for t in (up, up_s, down, down_s)]
    fill = [torch.cat([t.view(u8), t.view(u8)[:2]]).view(f8) if t.dtype == f8 else torch.cat([t, t[:2]]) for t in small]  # as many experts as slots: the same split of the work
    got = few_token_experts(x[:2, :H], ids, weights, (up, up_s), (down, down_s))
    assert torch.equal(got, few_token_experts(x[:2, :H], renamed, weights, (fill[0], fill[1]), (fill[2], fill[3])))
