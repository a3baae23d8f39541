"""Definitions in 64 bits of the steps around the products of a decoder block: RMS norm with residual, quantiser and gradients, tokens
sorted by expert and back, products with 4-bit weights.  CPU, plain loops where order is what is being defined."""
import torch


def norm_input(x, residual):
    """What the norm reads: x, or x + residual rounded to their type (one fp32 addition, one rounding)."""
    return x if residual is None else (x.float() + residual.float()).to(x.dtype)


def rms_norm(h, weight, eps):
    h, w = h.double(), weight.double()
    return h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * w


def quant_1x128(y, quant_eps=1e-10):
    """(scales, y / scale) before the rounding to e4m3."""
    g = y.reshape(y.shape[:-1] + (-1, 128))
    s = g.abs().amax(-1, keepdim=True).clamp_min(quant_eps) / 448.0
    return s.squeeze(-1), (g / s).reshape(y.shape)


def rms_norm_grad(dy, dsum, h, weight, eps):
    """(dx, dw) and the sums of magnitudes that bound the rounding of an fp32 evaluation of each."""
    dy, h, w = dy.double(), h.double(), weight.double()
    H = h.shape[-1]
    r = 1.0 / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    along = r**2 * (w * dy * h).sum(-1, keepdim=True) / H
    along_mag = r**2 * (w * dy * h).abs().sum(-1, keepdim=True) / H
    dx = r * (w * dy - h * along)
    mag = r * ((w * dy).abs() + h.abs() * (along.abs() + along_mag))
    if dsum is not None:
        dx = dx + dsum.double()
        mag = mag + dsum.double().abs()
    each = (dy * h * r).reshape(-1, H)
    return dx, each.sum(0), mag, each.abs().sum(0)


def sort_tables(ids, num_experts, alignment, num_rows):
    """(row_index, source, m_indices, row_start, row_end) as lists, slot after slot."""
    T, topk = ids.shape
    flat = [int(v) for v in ids.flatten()]
    by_expert = [[i for i, e in enumerate(flat) if e == x] for x in range(num_experts)]
    row_index, source, m_indices = [-1] * (T * topk), [-1] * num_rows, [-1] * num_rows
    row_start, row_end, first = [], [], 0
    for e, slots in enumerate(by_expert):
        span = -(-len(slots) // alignment) * alignment
        row_start.append(min(first, num_rows))
        row_end.append(min(first + len(slots), num_rows))
        for k in range(span):
            if first + k < num_rows:
                m_indices[first + k] = e
        for k, i in enumerate(slots):
            if first + k < num_rows:
                row_index[i], source[first + k] = first + k, i
        first += span
    as_int = lambda v: torch.tensor(v, dtype=torch.int32)
    return as_int(row_index).reshape(T, topk), as_int(source), as_int(m_indices), as_int(row_start), as_int(row_end)


def permute(x, source, topk):
    rows = torch.zeros((source.numel(), ) + x.shape[1:], dtype=x.dtype)
    for r, i in enumerate(source.tolist()):
        if i >= 0:
            rows[r] = x[i // topk]
    return rows


def unpermute(rows, row_index, weights):
    """(out, sum of the magnitudes of its terms)."""
    T, topk = row_index.shape
    out = torch.zeros(T, rows.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(out)
    for t in range(T):
        for j in range(topk):
            r = int(row_index[t, j])
            if 0 <= r < rows.shape[0]:
                term = rows[r].double() * (1.0 if weights is None else float(weights[t, j]))
                out[t] += term
                mag[t] += term.abs()
    return out, mag


def w4_codes(w_q):
    """[..., K / 2] bytes -> [..., K] codes."""
    return torch.stack([w_q & 15, w_q >> 4], -1).flatten(-2)


def w4_weights(w_q, w_s, w_z):
    codes = w4_codes(w_q).double()
    group = codes.shape[-1] // w_s.shape[-1]
    zero = torch.full(w_s.shape, 8.0, dtype=torch.float64) if w_z is None else w_z.double()
    return (codes - zero.repeat_interleave(group, -1)) * w_s.double().repeat_interleave(group, -1)


def w4_gemm(x, w_q, w_s, w_z):
    """(y, error bound of the kernel's fp32 evaluation before its rounding): the sums of a group are of terms up to 31 |x| twice, cut
    off and rounded to at most 24 * 2^-24 of their magnitudes; the groups' sums are then added with two fp32 roundings each, in any order."""
    w = w4_weights(w_q, w_s, w_z)
    group = w.shape[-1] // w_s.shape[-1]
    x = x.double()
    groups = w_s.shape[-1]
    x_abs = x.abs().reshape(x.shape[0], groups, group).sum(-1)
    s_abs = w_s.double().abs()
    bound = 24 * 2.0**-24 * 62 * (x_abs @ s_abs.t())
    bound = bound + (groups + 8) * 2.0**-24 * 15 * (x_abs @ s_abs.t())
    return x @ w.t(), bound
