"""The steps around the products of a decoder block, on what its layers meet in use.

Seven kinds of work:

    norm_quant      rms_norm_quant: residual addition, RMS norm and the 1 x 128 quantiser in front of an FP8 product
    norm_train      rms_norm forward and backward: the same norm in a 16- or 32-bit training step
    permute         moe_permute: tokens sorted by expert, with the tables the grouped products read
    unpermute       moe_unpermute: the experts' rows back in token order, weighted
    permute_train   both with their gradients, the experts themselves left out
    w4              w4_gemm: a few rows times a matrix of 4-bit weights with group scales
    w4_experts      w4_gemm_grouped: the same for the row ranges of experts

``own`` False computes each from elementary torch operations.  ``draw`` takes sizes from the whole range of the same kinds.
"""
import math
import random

import torch

own = False

BLOCK = 128
FP8_MAX = 448.0
DTYPES = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32, 'f8': torch.float8_e4m3fn}
BYTES = {'bf16': 2, 'f16': 2, 'f32': 4, 'f8': 1}
EPS, QUANT_EPS = 1e-6, 1e-10
LARGEST_WEIGHTS = 32 * 4096 * 7168  # the largest listed matrices; a drawn case stays below them and below the listed bytes


def listed():
    return [
        # the norm in front of a projection for one token of a running sequence: latency
        dict(name='norm_quant_1x7168', kind='norm_quant', t=1, h=7168, dtype='bf16', residual=True),
        # the same for a prefill batch: bandwidth
        dict(name='norm_quant_8192x7168', kind='norm_quant', t=8192, h=7168, dtype='bf16', residual=True),
        # a training step of the norm with its residual stream
        dict(name='norm_train_4096x7168', kind='norm_train', t=4096, h=7168, dtype='bf16', residual=True),
        # a width that is a multiple of no vector, 32 bits, no residual: the first norm of an odd model
        dict(name='norm_train_1237x2050_f32', kind='norm_train', t=1237, h=2050, dtype='f32', residual=False),
        # a decode step of 16 sequences, every expert on this GPU
        dict(name='permute_16_e32', kind='permute', t=16, h=7168, e=32, total=32, topk=8, align=1, dtype='bf16'),
        # a prefill batch of quantised tokens with 32 of 256 experts here, in the 128-row blocks of the grouped products
        dict(name='permute_8192_e32_f8', kind='permute', t=8192, h=7168, e=32, total=256, topk=8, align=128, dtype='f8'),
        # an odd number of tokens back from 32 local experts, a third of the slots elsewhere
        dict(name='unpermute_1001_e32', kind='unpermute', t=1001, h=4096, e=32, total=48, topk=6, align=1, dtype='bf16'),
        # a training step of the sort and its way back
        dict(name='permute_train_4096_e32', kind='permute_train', t=4096, h=7168, e=32, total=32, topk=8, align=128, dtype='bf16'),
        # one token against the narrow projection: latency
        dict(name='w4_1x2112x7168', kind='w4', m=1, n=2112, k=7168, group=128, zeros=False, dtype='bf16'),
        # a decode step of 16 sequences against a wide projection: the weights' bytes
        dict(name='w4_16x7168x18432', kind='w4', m=16, n=7168, k=18432, group=128, zeros=False, dtype='bf16'),
        # gate/up projection of 32 local experts in a decode step of 16 sequences with eight experts each
        dict(name='w4_experts_128_4096x7168', kind='w4_experts', t=16, e=32, topk=8, n=4096, k=7168, group=128, zeros=False, dtype='bf16'),
        # a few sequences, sizes that fill no tile, small groups with zero points
        dict(name='w4_experts_10_1000x1056_f16', kind='w4_experts', t=5, e=8, topk=2, n=1000, k=1056, group=32, zeros=True, dtype='f16'),
    ]


def _log_int(rng, lo, hi, multiple=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / multiple)) * multiple))


def draw(rng):
    while True:
        kind = rng.choice(['norm_quant', 'norm_train', 'permute', 'unpermute', 'permute_train', 'w4', 'w4', 'w4_experts'])
        if kind == 'norm_quant':
            c = dict(kind=kind, t=_log_int(rng, 1, 8192), h=_log_int(rng, 128, 8192, BLOCK), dtype=rng.choice(['bf16', 'f16', 'f32']),
                     residual=rng.random() < 0.7)
        elif kind == 'norm_train':
            c = dict(kind=kind, t=_log_int(rng, 1, 8192), h=_log_int(rng, 64, 8192, rng.choice([1, 8, 64])),
                     dtype=rng.choice(['bf16', 'bf16', 'f16', 'f32']), residual=rng.random() < 0.7)
        elif kind in ('permute', 'unpermute', 'permute_train'):
            e = rng.choice([2, 8, 16, 32, 64, 160, 256])
            total = e * rng.choice([1, 1, 2, 8])
            dtype = rng.choice(['bf16', 'bf16', 'f16', 'f32', 'f8'] if kind == 'permute' else ['bf16', 'bf16', 'f16', 'f32'])
            c = dict(kind=kind, t=_log_int(rng, 1, 8192), h=_log_int(rng, 64, 7168, BLOCK if dtype == 'f8' else rng.choice([1, 8, 64])), e=e,
                     total=total, topk=min(total, rng.randint(1, 8)), align=rng.choice([1, 1, 16, 128]), dtype=dtype)
        else:
            group = rng.choice([32, 64, 128, 128])
            c = dict(kind=kind, n=_log_int(rng, 64, 36864 if kind == 'w4' else 7168, rng.choice([1, 16, 64])), k=_log_int(rng, 128, 18432, group),
                     group=group, zeros=rng.random() < 0.5, dtype=rng.choice(['bf16', 'bf16', 'f16']))
            if kind == 'w4':
                c['m'] = _log_int(rng, 1, 64)
            else:
                c['e'] = rng.choice([4, 8, 16, 32])
                c['t'], c['topk'] = _log_int(rng, 1, 64), rng.randint(1, min(8, c['e']))
        if kind in ('w4', 'w4_experts'):
            # the rows of a plain form are filled up to the longest expert's
            rows = c['m'] if kind == 'w4' else c['t']
            if c['n'] * c['k'] * c.get('e', 1) <= LARGEST_WEIGHTS and c['n'] * c['k'] * c.get('e', 1) * rows <= 16 * LARGEST_WEIGHTS:
                return c
        elif work(c)['bytes'] <= max(work(d)['bytes'] for d in listed()):
            return c


# --- inputs -------------------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _stream(t, h, dtype, g):
    """Rows of a residual stream: a few channels are much larger than the others."""
    x = torch.randn(t, h, device='cuda', generator=g)
    gain = torch.where(torch.rand(h, device='cuda', generator=g) < 0.01, 20.0, 1.0)
    return (x * gain).to(DTYPES[dtype])


def _norm_weight(h, dtype, g):
    return (1.0 + 0.1 * torch.randn(h, device='cuda', generator=g)).to(DTYPES[dtype])


def _rows_n(case):
    """Rows that a program reserves for the sorted order: a fifth and four deviations more than the mean of the slots that stay
    here, and what the spans of the experts are rounded up by.  Slots that find no room are dropped."""
    slots, align = case['t'] * case['topk'], case['align']
    mean = slots * case['e'] / case['total']
    room = slots if case['e'] == case['total'] else min(slots, int(1.2 * mean + 4 * math.sqrt(mean)) + 1)
    return -(-(room + min(case['e'], slots) * (align - 1)) // align) * align


def _routing(case, g):
    """topk distinct experts of `total` for every token, some of them liked more; the first `e` are here, the others -1."""
    t, e, total, topk = case['t'], case['e'], case['total'], case['topk']
    liking = torch.rand(t, total, device='cuda', generator=g) + 0.3 * torch.rand(total, device='cuda', generator=g)
    ids = liking.topk(topk, dim=1).indices
    ids = torch.where(ids < e, ids, torch.full_like(ids, -1)).to(torch.int32)
    return ids, torch.sigmoid(torch.randn(t, topk, device='cuda', generator=g))


def _w4_weights(e, n, k, group, zeros, dtype, g):
    """Codes of every value, scales that give the products of N(0, 1) rows a size of about one."""
    q = torch.randint(0, 256, (e, n, k // 2), dtype=torch.uint8, device='cuda', generator=g)
    s = ((0.5 + torch.rand(e, n, k // group, device='cuda', generator=g)) / (4.6 * math.sqrt(k))).to(DTYPES[dtype])
    z = torch.randint(4, 12, (e, n, k // group), dtype=torch.uint8, device='cuda', generator=g) if zeros else None
    return q, s, z


def prepare(case, seed):
    g, kind = _gen(seed), case['kind']
    st = dict(case=case)
    if kind in ('norm_quant', 'norm_train'):
        t, h, dt = case['t'], case['h'], case['dtype']
        st['x'] = _stream(t, h, dt, g)
        st['res'] = _stream(t, h, dt, g) if case['residual'] else None
        st['w'] = _norm_weight(h, dt, g)
        if kind == 'norm_train':
            st['dy'] = torch.randn(t, h, device='cuda', generator=g).to(DTYPES[dt])
            st['dsum'] = torch.randn(t, h, device='cuda', generator=g).to(DTYPES[dt]) if case['residual'] else None
            for name in ('x', 'res', 'w'):
                if st[name] is not None:
                    st[name].requires_grad_()
        return st
    if kind in ('permute', 'unpermute', 'permute_train'):
        st['ids'], st['weights'] = _routing(case, g)
        st['rows_n'] = _rows_n(case)
        t, h, dt = case['t'], case['h'], case['dtype']
        x = torch.randn(t, h, device='cuda', generator=g)
        if dt == 'f8':
            st['x'] = x.mul_(100.0).clamp_(-FP8_MAX, FP8_MAX).to(DTYPES['f8'])
            st['x_s'] = torch.rand(t, h // BLOCK, device='cuda', generator=g) * 0.01
            return st
        st['x'] = x.to(DTYPES[dt])
        if kind == 'unpermute':
            st['rows'] = torch.randn(st['rows_n'], h, device='cuda', generator=g).to(DTYPES[dt])
            st['row_index'] = _sorted_rows(st['ids'], case['e'], case['align'], st['rows_n'])[0]
        if kind == 'permute_train':
            st['dout'] = torch.randn(t, h, device='cuda', generator=g).to(DTYPES[dt])
            st['x'].requires_grad_()
            st['weights'].requires_grad_()
        return st
    if kind == 'w4':
        q, s, z = _w4_weights(1, case['n'], case['k'], case['group'], case['zeros'], case['dtype'], g)
        st.update(q=q[0], s=s[0], z=None if z is None else z[0])
        st['x'] = torch.randn(case['m'], case['k'], device='cuda', generator=g).to(DTYPES[case['dtype']])
        return st
    # every token's distinct experts, drawn on the host: the counts are a serving program's own
    rng = random.Random(seed)
    counts = [0] * case['e']
    for _ in range(case['t']):
        for j in rng.sample(range(case['e']), case['topk']):
            counts[j] += 1
    ends = [sum(counts[:j + 1]) for j in range(case['e'])]
    st['q'], st['s'], st['z'] = _w4_weights(case['e'], case['n'], case['k'], case['group'], case['zeros'], case['dtype'], g)
    st['end'] = torch.tensor(ends, dtype=torch.int32, device='cuda')
    st['start'] = torch.tensor([b - c for b, c in zip(ends, counts)], dtype=torch.int32, device='cuda')
    st['most'] = max(counts)
    st['x'] = torch.randn(sum(counts), case['k'], device='cuda', generator=g).to(DTYPES[case['dtype']])
    return st


# --- the plain forms ------------------------------------------------------------------------------------------------


def _plain_norm(st):
    x, res, w = st['x'].detach(), st['res'], st['w'].detach().float()
    h = x if res is None else (x.float() + res.detach().float()).to(x.dtype)
    hf = h.float()
    r = torch.rsqrt((hf * hf).mean(dim=1, keepdim=True) + EPS)
    return h, hf, r, w, hf * r * w


def _plain_norm_quant(st):
    h, _, _, _, y = _plain_norm(st)
    blocks = y.view(y.shape[0], -1, BLOCK)
    s = blocks.abs().amax(dim=2, keepdim=True).clamp_min(QUANT_EPS) / FP8_MAX
    q = (blocks / s).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn).view(y.shape)
    return (q, s.squeeze(2)) if st['res'] is None else (q, s.squeeze(2), h)


def _plain_norm_train(st):
    h, hf, r, w, y = _plain_norm(st)
    dy = st['dy'].float()
    wdy = w * dy
    dot = (wdy * hf).sum(dim=1, keepdim=True)
    dh = r * wdy - hf * (r * r * r * dot / hf.shape[1])
    dw = (dy * hf * r).sum(dim=0).to(st['w'].dtype)
    if st['res'] is None:
        return y.to(h.dtype), dh.to(h.dtype), dw
    dh = (dh + st['dsum'].float()).to(h.dtype)
    return y.to(h.dtype), h, dh, dh, dw


def _sorted_rows(ids, e, align, rows_n):
    """row_index, source slot and expert of the rows, first and last row of every expert."""
    flat = ids.flatten().long()
    n, dev = flat.numel(), ids.device
    key = torch.where((flat >= 0) & (flat < e), flat, torch.full_like(flat, e))
    counts = torch.zeros(e + 1, dtype=torch.int64, device=dev).index_add_(0, key, torch.ones_like(key))
    spans = (counts[:e] + align - 1) // align * align
    first = torch.cat([spans.new_zeros(1), spans.cumsum(0)])
    order = torch.argsort(key, stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(n, device=dev)
    before = counts.cumsum(0) - counts
    row = first[key] + place - before[key]
    row = torch.where((key < e) & (row < rows_n), row, torch.full_like(row, -1))
    source = torch.full((rows_n + 1, ), -1, dtype=torch.int32, device=dev)
    source[torch.where(row >= 0, row, torch.full_like(row, rows_n))] = torch.arange(n, dtype=torch.int32, device=dev)
    source = source[:rows_n]
    expert = (torch.arange(rows_n, device=dev)[:, None] >= first[None, 1:]).sum(dim=1).to(torch.int32)
    expert = torch.where(expert < e, expert, torch.full_like(expert, -1))
    start = first[:e].clamp_max(rows_n)
    end = (first[:e] + counts[:e]).clamp_max(rows_n)
    return row.view(ids.shape).to(torch.int32), source, expert, start.to(torch.int32), end.to(torch.int32)


def _rows_of(x, source, topk):
    """Row r: the token of slot source[r], zeros where that is none."""
    rows = x[(source.clamp_min(0) // topk).long()]
    return torch.where((source >= 0)[:, None], rows, torch.zeros((), dtype=x.dtype, device=x.device))


def _plain_permute(st):
    c = st['case']
    tables = _sorted_rows(st['ids'], c['e'], c['align'], st['rows_n'])
    if c['dtype'] == 'f8':
        rows = _rows_of(st['x'].view(torch.uint8), tables[1], c['topk']).view(torch.float8_e4m3fn)
        return (rows, _rows_of(st['x_s'], tables[1], c['topk'])) + tables
    return (_rows_of(st['x'].detach(), tables[1], c['topk']), ) + tables


def _weighted(rows, row_index, weights):
    """sum over the slots, in 32 bits, one slot of all tokens at a time."""
    picked = rows[row_index.clamp_min(0).long()].float()
    picked = torch.where((row_index >= 0)[..., None], picked, torch.zeros((), device=rows.device))
    if weights is not None:
        picked = picked * weights[..., None]
    return picked.sum(dim=1)


def _plain_unpermute(st):
    return _weighted(st['rows'], st['row_index'], st['weights']).to(st['rows'].dtype)


def _plain_permute_train(st):
    c, x, weights, dout = st['case'], st['x'].detach(), st['weights'].detach(), st['dout']
    row_index, source = _sorted_rows(st['ids'], c['e'], c['align'], st['rows_n'])[:2]
    rows = _rows_of(x, source, c['topk'])
    out = _weighted(rows, row_index, weights).to(x.dtype)
    there = (source >= 0)[:, None]
    slot = source.clamp_min(0).long()
    dtok = dout[slot // c['topk']].float()
    zero = torch.zeros((), device=x.device)
    drows = torch.where(there, dtok * weights.flatten()[slot][:, None], zero).to(x.dtype)
    dots = torch.where(there[:, 0], (dtok * rows.float()).sum(dim=1), zero)
    dw = torch.where(row_index >= 0, dots[row_index.clamp_min(0).long()], zero)
    dx = _weighted(drows, row_index, None).to(x.dtype)
    return out, dx, dw


def _dequantised(q, s, z, group):
    codes = torch.stack([q & 15, q >> 4], dim=-1).flatten(-2).float()
    codes = codes.view(codes.shape[:-1] + (-1, group))
    codes = codes - (8.0 if z is None else z.float()[..., None])
    return (codes * s.float()[..., None]).flatten(-2)


def _plain_w4(st):
    w = _dequantised(st['q'], st['s'], st['z'], st['case']['group'])
    return (st['x'].float() @ w.t()).to(st['x'].dtype)


def _plain_w4_experts(st):
    x, most = st['x'], st['most']
    w = _dequantised(st['q'], st['s'], st['z'], st['case']['group'])
    # the experts' rows side by side, each filled up to the longest; the product with the rows behind the others
    at = st['start'][:, None].long() + torch.arange(most, device=x.device)
    there = at < st['end'][:, None]
    side = torch.where(there[..., None], x[at.clamp_max(x.shape[0] - 1)].float(), torch.zeros((), device=x.device))
    y = torch.bmm(w, side.transpose(1, 2).contiguous()).transpose(1, 2)
    r = torch.arange(x.shape[0], device=x.device)
    expert = (r[:, None] >= st['end'][None].long()).sum(dim=1)
    return y[expert, r - st['start'].long()[expert]].to(x.dtype)


# --- the framework's calls --------------------------------------------------------------------------------------------


def _own(st):
    from dlblas_amd.kernels import moe_permute as mp
    from dlblas_amd.kernels import rms_norm as rn
    from dlblas_amd.kernels import w4_gemm as w4
    c, kind = st['case'], st['case']['kind']
    if kind == 'norm_quant':
        return rn.rms_norm_quant(st['x'], st['w'], EPS, st['res'])
    if kind == 'norm_train':
        if st['res'] is None:
            y = rn.rms_norm(st['x'], st['w'], EPS)
            return (y, ) + torch.autograd.grad([y], [st['x'], st['w']], [st['dy']])
        y, h = rn.rms_norm(st['x'], st['w'], EPS, st['res'])
        return (y, h) + torch.autograd.grad([y, h], [st['x'], st['res'], st['w']], [st['dy'], st['dsum']])
    if kind == 'permute':
        x = (st['x'], st['x_s']) if c['dtype'] == 'f8' else st['x']
        rows, p = mp.moe_permute(x, st['ids'], c['e'], alignment=c['align'], num_rows=st['rows_n'])
        return (tuple(rows) if c['dtype'] == 'f8' else (rows, )) + (p.row_index, p.source, p.m_indices, p.row_start, p.row_end)
    if kind == 'unpermute':
        return mp.moe_unpermute(st['rows'], st['row_index'], st['weights'])
    if kind == 'permute_train':
        rows, p = mp.moe_permute(st['x'], st['ids'], c['e'], alignment=c['align'], num_rows=st['rows_n'])
        out = mp.moe_unpermute(rows, p, st['weights'])
        return (out, ) + torch.autograd.grad([out], [st['x'], st['weights']], [st['dout']])
    if kind == 'w4':
        return w4.w4_gemm(st['x'], st['q'], st['s'], st['z'])
    return w4.w4_gemm_grouped(st['x'], st['q'], st['s'], st['start'], st['end'], st['z'])


_PLAIN = dict(norm_quant=_plain_norm_quant, norm_train=_plain_norm_train, permute=_plain_permute, unpermute=_plain_unpermute,
              permute_train=_plain_permute_train, w4=_plain_w4, w4_experts=_plain_w4_experts)


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _PLAIN[state['case']['kind']](state)


# --- what a pass cannot do without -----------------------------------------------------------------------------------


def work(case):
    kind, b = case['kind'], BYTES[case['dtype']]
    if kind == 'norm_quant':
        n = case['t'] * case['h']
        return dict(bytes=n * ((3 if case['residual'] else 1) * b + 1 + 4 / BLOCK) + case['h'] * b, flops=8.0 * n)
    if kind == 'norm_train':
        # in: x, dy and with a residual that and the gradient of the sum; out: y, dx and the sum (its two gradients are one)
        n = case['t'] * case['h']
        return dict(bytes=n * (7 if case['residual'] else 4) * b + 2 * case['h'] * b, flops=16.0 * n)
    if kind in ('permute', 'unpermute', 'permute_train'):
        t, h, slots = case['t'], case['h'], case['t'] * case['topk']
        rows = slots * case['e'] / case['total']  # those with a slot, on average; all of them are written
        out_rows = _rows_n(case)
        tables = slots * 8 + out_rows * 8
        if kind == 'permute':
            per = h * b + (4 * h / BLOCK if case['dtype'] == 'f8' else 0)
            return dict(bytes=(t + out_rows) * per + tables, flops=0.0)
        if kind == 'unpermute':
            return dict(bytes=(t + rows) * h * b + slots * 8, flops=2.0 * rows * h)
        # the rows and their gradients exist, because the experts work on them: each is written once and read again; the rows
        # once more for the gradients of the weights
        return dict(bytes=(4 * t + 2 * out_rows + 3 * rows) * h * b + tables + 4 * slots, flops=6.0 * rows * h)
    e, n, k = case.get('e', 1), case['n'], case['k']
    m = case['m'] if kind == 'w4' else case['t'] * case['topk']
    used = e if kind == 'w4' else e * (1 - (1 - case['topk'] / e)**case['t'])  # experts that have a row, on average
    weights = n * k / 2 + n * (k // case['group']) * (b + (1 if case['zeros'] else 0))
    return dict(bytes=used * weights + m * (n + k) * b, flops=2.0 * m * n * k)


# --- the definitions in 64 bits ----------------------------------------------------------------------------------------


def _e4m3(v):
    """Nearest e4m3 value, ties to even, of |v| <= 448: steps of an eighth of the power of two below, at least 2^-9."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 4).clamp_min(-9))
    return torch.round(v / step) * step


def _exact_norm(case, st):
    x = st['x'].detach().double()
    h = x if st['res'] is None else (x + st['res'].detach().double()).to(st['x'].dtype).double()
    w = st['w'].detach().double()
    n = h.shape[1]
    inv = 1.0 / torch.sqrt(h.square().sum(1) / n + EPS)
    unit = h * inv[:, None]
    if case['kind'] == 'norm_quant':
        y = (unit * w).reshape(h.shape[0], n // BLOCK, BLOCK)
        s = torch.maximum(y.abs().max(2).values, torch.tensor(QUANT_EPS, dtype=torch.float64, device=y.device)) / FP8_MAX
        q = _e4m3((y / s[..., None]).clamp(-FP8_MAX, FP8_MAX)).reshape(h.shape)
        return (q, s) if st['res'] is None else (q, s, h)
    dy = st['dy'].double()
    along = (unit * dy * w).mean(1)
    dh = inv[:, None] * (dy * w - unit * along[:, None])
    dw = (dy * unit).sum(0)
    if st['res'] is None:
        return unit * w, dh, dw
    dh = dh + st['dsum'].double()
    return unit * w, h, dh, dh, dw


def _exact_places(ids, e, align, rows_n):
    """Row of every slot by counting: the slots of its expert before it, behind the spans of the experts before."""
    flat = ids.flatten().long()
    mine = flat[:, None] == torch.arange(e, device=ids.device)
    upto = mine.to(torch.int32).cumsum(0)
    total = upto[-1].long()
    spans = -(-total // align) * align
    first = spans.cumsum(0) - spans
    row = ((upto - 1) + first).masked_fill(~mine, -1).max(dim=1).values
    return torch.where(row < rows_n, row, torch.full_like(row, -1))


def _exact_permute(case, st):
    t, topk, n = case['t'], case['topk'], st['rows_n']
    row = _exact_places(st['ids'], case['e'], case['align'], n)
    slots = torch.nonzero(row >= 0).flatten()
    x = st['x'].detach().double()
    if case['kind'] == 'permute':
        rows = torch.zeros(n, x.shape[1], dtype=torch.float64, device=x.device)
        rows[row[slots]] = x[slots // topk]
        tables = (None, ) * 5
        if case['dtype'] != 'f8':
            return (rows, ) + tables
        scales = torch.zeros(n, x.shape[1] // BLOCK, dtype=torch.float64, device=x.device)
        scales[row[slots]] = st['x_s'].double()[slots // topk]
        return (rows, scales) + tables
    w = torch.zeros(t * topk, dtype=torch.float64, device=x.device)
    w[slots] = st['weights'].detach().double().flatten()[slots]
    w = w.view(t, topk)
    if case['kind'] == 'unpermute':
        out = torch.zeros(t, case['h'], dtype=torch.float64, device=x.device)
        out.index_add_(0, slots // topk, st['rows'].double()[row[slots]] * w.flatten()[slots, None])
        return out
    # the experts left out, a token's rows are the token itself; the gradient of a row is held in the rows' type
    dout = st['dout'].double()
    here = (row >= 0).view(t, topk)
    out = x * w.sum(1)[:, None]
    dw = torch.where(here, (x * dout).sum(1)[:, None], torch.zeros((), dtype=torch.float64, device=x.device))
    dx = torch.zeros_like(x)
    for j in range(topk):
        dx += (dout * w[:, j, None]).to(st['x'].dtype).double()
    return out, dx, dw


def _exact_w4(case, st):
    # the row ranges come back to the host, and each expert is a product of its own
    x, group = st['x'].double(), case['group']
    one = case['kind'] == 'w4'
    ranges = [(0, x.shape[0])] if one else list(zip(st['start'].tolist(), st['end'].tolist()))
    out = torch.zeros(x.shape[0], case['n'], dtype=torch.float64, device=x.device)
    for j, (a, b) in enumerate(ranges):
        if a == b:
            continue
        q, s, z = ((None if v is None else v if one else v[j]) for v in (st['q'], st['s'], st['z']))
        w = torch.empty(case['n'], case['k'], dtype=torch.float64, device=x.device)
        w[:, 0::2], w[:, 1::2] = q.remainder(16).double(), q.div(16, rounding_mode='floor').double()
        w -= 8 if z is None else z.double().repeat_interleave(group, dim=1)
        w *= s.double().repeat_interleave(group, dim=1)
        out[a:b] = x[a:b] @ w.t()
    return out


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case['kind'].startswith('norm'):
            return _exact_norm(case, st)
        return _exact_permute(case, st) if 'permute' in case['kind'] else _exact_w4(case, st)
