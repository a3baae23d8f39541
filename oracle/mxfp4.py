"""Definitions in 64 bits of microscaled 4-bit floating point, its products, and a layer of experts.  CPU."""
import torch

GROUP = 32
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
FP32 = 2.0**-24


def quant(x):
    """(codes [..., K / 2], scales [..., K / 32]) as uint8."""
    K = x.shape[-1]
    v = x.double().reshape(-1, GROUP)
    amax = v.abs().amax(1)
    finite = v.isfinite().all(1)
    safe = torch.where(finite & (amax > 0), amax, torch.ones_like(amax))
    e = torch.where(amax > 0, torch.frexp(safe).exponent - 1 - 2, torch.full_like(amax, -127, dtype=torch.int32)).clamp_min(-127)
    s = torch.where(finite, e + 127, torch.full_like(e, 255))
    a = torch.where(finite[:, None], v.abs(), torch.zeros(())) * torch.exp2(-e.double())[:, None]
    values = torch.tensor(E2M1, dtype=torch.float64)
    off = (a[..., None] - values).abs()
    near = off.amin(-1, keepdim=True) == off
    even = torch.arange(8) % 2 == 0
    code = torch.where((near & even).any(-1), (near & even).int().argmax(-1), near.int().argmax(-1))  # of two as near the even one
    code = code + 8 * ((torch.signbit(v)) & finite[:, None]).int()
    code = code.reshape(x.shape[:-1] + (K // 2, 2))
    q = (code[..., 0] + 16 * code[..., 1]).to(torch.uint8)
    return q, s.reshape(x.shape[:-1] + (K // GROUP, )).to(torch.uint8)


def values(q, s):
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64)
    v = table[torch.stack([q & 15, q >> 4], -1).flatten(-2).long()]
    scale = torch.where(s == 255, torch.full(s.shape, float('nan'), dtype=torch.float64), torch.exp2(s.double() - 127))
    return v * scale.repeat_interleave(GROUP, -1)


def gemm(a, a_s, b, b_s):
    """(product, sum of the magnitudes of its terms)."""
    x, w = values(a, a_s), values(b, b_s)
    return x @ w.t(), x.abs() @ w.abs().t()


def e4m3_values(q, s):
    """[E, N, K] numbers of e4m3 weights with a scale per 128 x 128."""
    wide = s.double().repeat_interleave(128, 1)[:, :q.shape[1]].repeat_interleave(128, 2)
    return q.double() * wide


def experts(x, ids, weights, w13, w2):
    """(out, bound of an evaluation in fp32), from the numbers of the weights [E, 2 I, H], [E, H, I].

    A sum of n terms is off by at most (n + 8) 2^-23 of its magnitudes (the unit cuts off where it does not round).  silu(g) u: g and u as far off as that,
    |silu'| <= 1.1, the exponential off by 2^-23 of itself, silu then by as much of itself, and four roundings, which make 3 2^-23."""
    T, H = x.shape
    I = w13.shape[1] // 2
    x, out, bound = x.double(), torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    for t in range(T):
        for e, w in zip(ids[t].tolist(), weights[t].double().tolist()):
            if not 0 <= e < w13.shape[0]:
                continue
            both, mag = w13[e] @ x[t], w13[e].abs() @ x[t].abs()
            off = (H + 8) * 2 * FP32 * mag
            (g, u), (g_off, u_off) = both.split(I), off.split(I)
            silu = g / (1 + torch.exp(-g))
            act = silu * u
            act_off = 1.1 * g_off * (u.abs() + u_off) + silu.abs() * u_off + act.abs() * 3 * 2 * FP32
            out[t] += w * (w2[e] @ act)
            terms = abs(w) * (w2[e].abs() @ act.abs())
            bound[t] += abs(w) * (w2[e].abs() @ act_off) + (I + 40) * 2 * FP32 * terms
    return out, bound
