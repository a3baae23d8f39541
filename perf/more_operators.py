"""More steps of a decoder layer, on what its layers meet in use.

Five kinds of work:

    norm            layer_norm: residual addition and layer norm in front of a projection
    norm_train      layer_norm forward and backward, with the gradients of weight and bias
    linear          per_group_quant_mxfp4 of the activations and mxfp4_gemm with weights kept in the same form
    weight_linear   mxfp4_weight_gemm: a few 16-bit rows times weights of 4-bit floating point
    experts         few_token_experts: gate/up, silu, down and the weighted sum of a layer of experts for a few tokens

``own`` False computes each from elementary torch operations.  ``draw`` takes sizes from the whole range of the same kinds.
"""
import math
import random

import torch

own = False

GROUP = 32   # columns that share a scale in 4-bit floating point
BLOCK = 128  # rows and columns that share a scale of e4m3 weights
EPS = 1e-5
DTYPES = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}
BYTES = {'bf16': 2, 'f16': 2, 'f32': 4}


def listed():
    return [
        # the norm in front of a projection for one token of a running sequence: latency
        dict(name='norm_1x7168', kind='norm', t=1, h=7168, dtype='bf16', residual=True, bias=True, w32=False),
        # a training step of the norm with its residual stream: bandwidth, and the sums over all rows
        dict(name='norm_train_4096x7168', kind='norm_train', t=4096, h=7168, dtype='bf16', residual=True, bias=True, w32=False),
        # a width that is a multiple of no vector, 32 bits, no residual: the first norm of an odd model
        dict(name='norm_train_1237x2050_f32', kind='norm_train', t=1237, h=2050, dtype='f32', residual=False, bias=True, w32=True),
        # a decode step of 16 sequences against the narrow projection
        dict(name='linear_16x2112x7168', kind='linear', m=16, n=2112, k=7168, dtype='bf16'),
        # a prompt against the wide projection: the matrix units
        dict(name='linear_4096x7168x18432', kind='linear', m=4096, n=7168, k=18432, dtype='bf16'),
        # sizes that fill no tile and no wide load: 33 groups a row
        dict(name='linear_1000x1000x1056_f16', kind='linear', m=1000, n=1000, k=1056, dtype='f16'),
        # one token against the narrow projection: latency
        dict(name='weight_1x2112x7168', kind='weight_linear', m=1, n=2112, k=7168, dtype='bf16'),
        # a decode step of 16 sequences against the wide projection: the weights' bytes
        dict(name='weight_16x7168x18432', kind='weight_linear', m=16, n=7168, k=18432, dtype='bf16'),
        # one token through its eight experts of 32, e4m3 weights
        dict(name='experts_1_e32_f8', kind='experts', t=1, e=32, total=32, topk=8, h=7168, i=2048, weights='f8', dtype='bf16'),
        # a decode step of 16 sequences, nearly every expert used
        dict(name='experts_16_e32_f8', kind='experts', t=16, e=32, total=32, topk=8, h=7168, i=2048, weights='f8', dtype='bf16'),
        # the same with weights of 4-bit floating point
        dict(name='experts_16_e32_f4', kind='experts', t=16, e=32, total=32, topk=8, h=7168, i=2048, weights='f4', dtype='bf16'),
        # a few sequences, a third of the slots on another GPU, sizes that fill no tile
        dict(name='experts_5_e8_f4_f16', kind='experts', t=5, e=8, total=12, topk=2, h=1056, i=544, weights='f4', dtype='f16'),
    ]


def _log_int(rng, lo, hi, multiple=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(multiple, lo, min(hi, int(round(v / multiple)) * multiple))


def draw(rng):
    most = max(work(c)['bytes'] for c in listed())
    flops = max(work(c)['flops'] for c in listed())
    while True:
        kind = rng.choice(['norm', 'norm_train', 'linear', 'linear', 'weight_linear', 'experts', 'experts'])
        if kind in ('norm', 'norm_train'):
            c = dict(kind=kind, t=_log_int(rng, 1, 8192), h=_log_int(rng, 64, 8192, rng.choice([1, 8, 64])),
                     dtype=rng.choice(['bf16', 'bf16', 'f16', 'f32']), residual=rng.random() < 0.7, bias=rng.random() < 0.7, w32=rng.random() < 0.3)
        elif kind == 'linear':
            c = dict(kind=kind, m=_log_int(rng, 1, 4096), n=_log_int(rng, 64, 36864, rng.choice([1, 16, 64])),
                     k=_log_int(rng, 128, 18432, rng.choice([GROUP, 128])), dtype=rng.choice(['bf16', 'bf16', 'f16', 'f32']))
        elif kind == 'weight_linear':
            c = dict(kind=kind, m=_log_int(rng, 1, 64), n=_log_int(rng, 64, 36864, rng.choice([1, 16, 64])),
                     k=_log_int(rng, 128, 18432, rng.choice([GROUP, 128])), dtype=rng.choice(['bf16', 'bf16', 'f16']))
        else:
            e, weights = rng.choice([4, 8, 16, 32, 64]), rng.choice(['f8', 'f4'])
            unit = BLOCK if weights == 'f8' else rng.choice([GROUP, 128])
            c = dict(kind=kind, t=_log_int(rng, 1, 64), e=e, total=e * rng.choice([1, 1, 2]), topk=rng.randint(1, min(8, e)), h=_log_int(rng, 256, 7168, unit),
                     i=_log_int(rng, 128, 4096, unit), weights=weights, dtype=rng.choice(['bf16', 'bf16', 'f16']))
            # a plain form multiplies the tokens with every expert's weights
            if 3 * c['e'] * c['h'] * c['i'] > 32 * 3 * 7168 * 2048:
                continue
        w = work(c)
        if w['bytes'] <= most and w['flops'] <= flops:
            return c


# --- inputs -------------------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _stream(t, h, dtype, g):
    """Rows of a residual stream: a few channels are much larger than the others, and rows are off zero."""
    x = torch.randn(t, h, device='cuda', generator=g)
    gain = torch.where(torch.rand(h, device='cuda', generator=g) < 0.01, 20.0, 1.0)
    return (x * gain + 0.3 * torch.randn(t, 1, device='cuda', generator=g)).to(DTYPES[dtype])


def _f4_weights(size, k, g):
    """Codes of every value; scales that give products with N(0, 1) rows a size of about one, over an octave to each side."""
    q = torch.randint(0, 256, size + (k // 2, ), dtype=torch.uint8, device='cuda', generator=g)
    middle = 127 - round(math.log2(2.9 * math.sqrt(k)))
    s = torch.randint(middle - 1, middle + 2, size + (k // GROUP, ), dtype=torch.uint8, device='cuda', generator=g)
    return q, s


def _f8_weights(e, n, k, g):
    q = torch.randn(e, n, k, device='cuda', generator=g).mul_(100.0).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
    s = (0.5 + torch.rand(e, -(-n // BLOCK), k // BLOCK, device='cuda', generator=g)) / (100.0 * math.sqrt(k))
    return q, s


def _routing(case, g):
    """topk distinct experts of `total` for every token, some of them liked more; the first `e` are here, the others -1."""
    t, e, total, topk = case['t'], case['e'], case['total'], case['topk']
    liking = torch.rand(t, total, device='cuda', generator=g) + 0.3 * torch.rand(total, device='cuda', generator=g)
    ids = liking.topk(topk, dim=1).indices
    ids = torch.where(ids < e, ids, torch.full_like(ids, -1)).to(torch.int32)
    return ids, torch.sigmoid(torch.randn(t, topk, device='cuda', generator=g))


def prepare(case, seed):
    g, kind = _gen(seed), case['kind']
    st = dict(case=case)
    if kind in ('norm', 'norm_train'):
        t, h, dt = case['t'], case['h'], case['dtype']
        wt = torch.float32 if case['w32'] else DTYPES[dt]
        st['x'] = _stream(t, h, dt, g)
        st['res'] = _stream(t, h, dt, g) if case['residual'] else None
        st['w'] = (1.0 + 0.1 * torch.randn(h, device='cuda', generator=g)).to(wt)
        st['b'] = (0.1 * torch.randn(h, device='cuda', generator=g)).to(wt) if case['bias'] else None
        if kind == 'norm_train':
            st['dy'] = torch.randn(t, h, device='cuda', generator=g).to(DTYPES[dt])
            st['dsum'] = torch.randn(t, h, device='cuda', generator=g).to(DTYPES[dt]) if case['residual'] else None
            for name in ('x', 'res', 'w', 'b'):
                if st[name] is not None:
                    st[name].requires_grad_()
        return st
    if kind in ('linear', 'weight_linear'):
        st['x'] = torch.randn(case['m'], case['k'], device='cuda', generator=g).to(DTYPES[case['dtype']])
        st['q'], st['s'] = _f4_weights((case['n'], ), case['k'], g)
        return st
    e, h, i = case['e'], case['h'], case['i']
    st['x'] = torch.randn(case['t'], h, device='cuda', generator=g).to(DTYPES[case['dtype']])
    st['ids'], st['weights'] = _routing(case, g)
    if case['weights'] == 'f8':
        st['up'], st['down'] = _f8_weights(e, 2 * i, h, g), _f8_weights(e, h, i, g)
    else:
        st['up'], st['down'] = _f4_weights((e, 2 * i), h, g), _f4_weights((e, h), i, g)
    return st


# --- the plain forms ------------------------------------------------------------------------------------------------


def _plain_norm(st):
    x, res, w = st['x'].detach(), st['res'], st['w'].detach().float()
    h = x if res is None else (x.float() + res.detach().float()).to(x.dtype)
    hf = h.float()
    centred = hf - hf.mean(dim=1, keepdim=True)
    r = torch.rsqrt((centred * centred).mean(dim=1, keepdim=True) + EPS)
    n = centred * r
    y = n * w
    if st['b'] is not None:
        y = y + st['b'].detach().float()
    return h, n, r, w, y.to(x.dtype)


def _plain_norm_only(st):
    h, _, _, _, y = _plain_norm(st)
    return (y, ) if st['res'] is None else (y, h)


def _plain_norm_train(st):
    h, n, r, w, y = _plain_norm(st)
    dy = st['dy'].float()
    wdy = w * dy
    dh = r * (wdy - wdy.mean(dim=1, keepdim=True) - n * (wdy * n).mean(dim=1, keepdim=True))
    dw = ((dy * n).sum(dim=0).to(st['w'].dtype), )
    if st['b'] is not None:
        dw = dw + (dy.sum(dim=0).to(st['b'].dtype), )
    if st['res'] is None:
        return (y, dh.to(h.dtype)) + dw
    dh = (dh + st['dsum'].float()).to(h.dtype)
    return (y, h, dh, dh) + dw


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _f4_values(q, s):
    """The numbers that codes and scales stand for, in 32 bits."""
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=q.device)
    v = table[torch.stack([q & 15, q >> 4], dim=-1).flatten(-2).int()]
    scale = torch.ldexp(torch.ones((), device=q.device), s.int() - 127)
    return (v.view(v.shape[:-1] + (-1, GROUP)) * scale[..., None]).flatten(-2)


def _f4_rounded(x):
    """The numbers of the nearest 4-bit codes: the scale of a group is the power of two two octaves below its largest value's."""
    v = x.float().view(x.shape[0], -1, GROUP)
    exponent = torch.frexp(v.abs().amax(dim=2, keepdim=True)).exponent - 3
    up = torch.ldexp(v.abs(), -exponent)
    step = torch.where(up < 2, 0.5, torch.where(up < 4, 1.0, 2.0))
    near = (torch.round(up / step) * step).clamp_max(6.0)  # halves go to the even multiple, which is the even code
    return torch.ldexp(torch.where(v < 0, -near, near), exponent).view(x.shape)


def _plain_linear(st):
    return (_f4_rounded(st['x']) @ _f4_values(st['q'], st['s']).t()).to(st['x'].dtype)


def _plain_weight_linear(st):
    return (st['x'].float() @ _f4_values(st['q'], st['s']).t()).to(st['x'].dtype)


def _f8_values(q, s):
    return q.float() * s.repeat_interleave(BLOCK, dim=1)[:, :q.shape[1]].repeat_interleave(BLOCK, dim=2)


def _plain_experts(st):
    c, ids = st['case'], st['ids']
    values = _f8_values if c['weights'] == 'f8' else _f4_values
    t, topk, e = c['t'], c['topk'], c['e']
    here = ids >= 0
    zero = torch.zeros((), device=ids.device)
    if t * topk < e:
        # fewer slots than experts: the weights of each slot's expert, and one row
        pick = ids.clamp_min(0).flatten().long()
        up = values(st['up'][0][pick], st['up'][1][pick]) if c['weights'] == 'f4' else values(st['up'][0].view(torch.uint8)[pick].view(torch.float8_e4m3fn), st['up'][1][pick])
        down = values(st['down'][0][pick], st['down'][1][pick]) if c['weights'] == 'f4' else values(st['down'][0].view(torch.uint8)[pick].view(torch.float8_e4m3fn), st['down'][1][pick])
        rows = st['x'].float().repeat_interleave(topk, dim=0)[:, :, None].contiguous()
        by = torch.where(here, st['weights'], zero).flatten()[:, None]
    else:
        # every expert with all tokens, and how much of it a token takes
        up, down = values(*st['up']), values(*st['down'])
        rows = st['x'].float().t().expand(e, c['h'], t).contiguous()
        chosen = ids[None] == torch.arange(e, device=ids.device)[:, None, None]
        by = torch.where(chosen, st['weights'], zero).sum(dim=2)
    gate = torch.bmm(up, rows)
    act = gate[:, :c['i']] * torch.sigmoid(gate[:, :c['i']]) * gate[:, c['i']:]
    y = torch.bmm(down, act) * by[:, None, :]
    out = y[:, :, 0].view(t, topk, c['h']).sum(dim=1) if t * topk < e else y.sum(dim=0).t()
    return out.to(st['x'].dtype).contiguous()


# --- the framework's calls --------------------------------------------------------------------------------------------


def _own(st):
    from dlblas_amd.kernels import few_token_experts as fx
    from dlblas_amd.kernels import layer_norm as ln
    from dlblas_amd.kernels import mxfp4_gemm as mx
    c, kind = st['case'], st['case']['kind']
    if kind == 'norm':
        out = ln.layer_norm(st['x'], st['w'], st['b'], EPS, st['res'])
        return (out, ) if st['res'] is None else out
    if kind == 'norm_train':
        leaves = [st[name] for name in ('x', 'res', 'w', 'b') if st[name] is not None]
        if st['res'] is None:
            y = ln.layer_norm(st['x'], st['w'], st['b'], EPS)
            return (y, ) + torch.autograd.grad([y], leaves, [st['dy']])
        y, h = ln.layer_norm(st['x'], st['w'], st['b'], EPS, st['res'])
        return (y, h) + torch.autograd.grad([y, h], leaves, [st['dy'], st['dsum']])
    if kind == 'linear':
        q, s = mx.per_group_quant_mxfp4(st['x'])
        return mx.mxfp4_gemm(q, st['q'], s, st['s'], st['x'].dtype)
    if kind == 'weight_linear':
        return mx.mxfp4_weight_gemm(st['x'], st['q'], st['s'])
    return fx.few_token_experts(st['x'], st['ids'], st['weights'], st['up'], st['down'])


_PLAIN = dict(norm=_plain_norm_only, norm_train=_plain_norm_train, linear=_plain_linear, weight_linear=_plain_weight_linear, experts=_plain_experts)


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _PLAIN[state['case']['kind']](state)


# --- what a pass cannot do without -----------------------------------------------------------------------------------


def work(case):
    kind, b = case['kind'], BYTES[case['dtype']]
    if kind in ('norm', 'norm_train'):
        n, wb = case['t'] * case['h'], case['h'] * (4 if case['w32'] else b) * (2 if case['bias'] else 1)
        if kind == 'norm':
            return dict(bytes=n * (4 if case['residual'] else 2) * b + wb, flops=9.0 * n)
        # in: x, dy and with a residual that and the gradient of the sum; out: y, dx and the sum (its two gradients are one)
        return dict(bytes=n * (7 if case['residual'] else 4) * b + 2 * wb, flops=20.0 * n)
    f4 = 0.5 + 1 / GROUP  # bytes of a number with its share of a scale
    if kind in ('linear', 'weight_linear'):
        m, n, k = case['m'], case['n'], case['k']
        return dict(bytes=n * k * f4 + m * (n + k) * b, flops=2.0 * m * n * k)
    t, e, h, i = case['t'], case['e'], case['h'], case['i']
    chance = case['topk'] / case['total']
    used = e * (1 - (1 - chance)**t)  # experts that have a token, on average
    per = f4 if case['weights'] == 'f4' else 1 + 4 / (BLOCK * BLOCK)
    return dict(bytes=used * 3 * h * i * per + 2 * t * h * b + t * case['topk'] * 8, flops=6.0 * t * e * chance * h * i)


# --- the definitions in 64 bits ----------------------------------------------------------------------------------------


def _exact_norm(case, st):
    x = st['x'].detach().double()
    h = x if st['res'] is None else (x + st['res'].detach().double()).to(st['x'].dtype).double()
    w = st['w'].detach().double()
    inv = 1.0 / torch.sqrt(h.var(1, correction=0) + EPS)
    unit = (h - h.mean(1)[:, None]) * inv[:, None]
    y = unit * w if st['b'] is None else torch.addcmul(st['b'].detach().double(), unit, w)
    if case['kind'] == 'norm':
        return (y, ) if st['res'] is None else (y, h)
    dy = st['dy'].double()
    # the gradient before the centring, and then without its parts along the row of ones and along the normed row
    t = dy * w
    t = t - t.mean(1)[:, None]
    dh = inv[:, None] * (t - unit * (t * unit).mean(1)[:, None])
    if st['res'] is not None:
        dh = dh + st['dsum'].double()
    rows = (y, dh) if st['res'] is None else (y, h, dh, dh)
    sums = ((dy * unit).sum(0), ) if st['b'] is None else ((dy * unit).sum(0), dy.sum(0))
    return rows + sums


def _exact_f4(q, s):
    """One bit of sign, two of exponent, one of significand, times the scale."""
    out = torch.empty(q.shape[:-1] + (2 * q.shape[-1], ), dtype=torch.float64, device=q.device)
    for half in (0, 1):
        code = q.remainder(16) if half == 0 else q.div(16, rounding_mode='floor')
        sign, magnitude = code.div(8, rounding_mode='floor').double(), code.remainder(8).double()
        octave = torch.div(magnitude, 2, rounding_mode='floor')
        tail = magnitude - 2 * octave
        value = torch.where(octave == 0, tail / 2, torch.exp2(octave - 1) * (1 + tail / 2))
        out[..., half::2] = value * (1 - 2 * sign)
    return out * torch.exp2(s.double() - 127).repeat_interleave(GROUP, dim=-1)


def _exact_rounded(x):
    """Nearest of all values to x over its group's scale, found among the borders between them."""
    values = torch.tensor(_E2M1, dtype=torch.float64, device=x.device)
    borders = (values[1:] + values[:-1]) / 2
    v = x.double().reshape(-1, GROUP)
    scale = torch.exp2(torch.floor(torch.log2(v.abs().max(1, keepdim=True).values)) - 2)
    a = v.abs() / scale
    low, high = torch.bucketize(a, borders, right=False), torch.bucketize(a, borders, right=True)
    index = torch.where(low % 2 == 0, low, high)  # on a border the code that is even
    return (values[index] * torch.sign(v) * scale).reshape(x.shape)


def _exact_experts(case, st):
    x, ids, i = st['x'].double(), st['ids'], case['i']
    out = torch.zeros(case['t'], case['h'], dtype=torch.float64, device=x.device)
    for j in range(case['e']):
        tokens, slots = torch.nonzero(ids == j, as_tuple=True)
        if tokens.numel() == 0:
            continue
        parts = []
        for q, s in (st['up'], st['down']):
            if case['weights'] == 'f4':
                parts.append(_exact_f4(q[j], s[j]))
            else:
                wide = s[j].double().repeat_interleave(BLOCK, dim=0)[:q.shape[1]].repeat_interleave(BLOCK, dim=1)
                parts.append(q[j].double() * wide)
        both = x[tokens] @ parts[0].t()
        gate, up = both[:, :i], both[:, i:]
        out.index_add_(0, tokens, ((gate / (1 + torch.exp(-gate)) * up) @ parts[1].t()) * st['weights'].double()[tokens, slots, None])
    return out


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case['kind'] in ('norm', 'norm_train'):
            return _exact_norm(case, st)
        if case['kind'] == 'experts':
            return _exact_experts(case, st)
        x = _exact_rounded(st['x']) if case['kind'] == 'linear' else st['x'].double()
        return x @ _exact_f4(st['q'], st['s']).t()
