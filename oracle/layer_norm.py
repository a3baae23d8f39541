"""Definitions in 64 bits of the layer norm and its gradients, and how far an fp32 evaluation may be from them.  CPU.

The bounds count roundings of 2^-24.  A lane adds at most 32 terms, the wave 6 times, the workgroup 16 sums, so a sum over a row is off by
at most 56 of them of the sum of its terms' magnitudes; with the division a mean is off by 58."""
import torch

from .decoder import norm_input  # noqa: F401  (h = x + residual rounded, as for the RMS norm)

FP32 = 2.0**-24


def parts(h, eps):
    """(mean, r, n, bound of n): n = (h - mean) r.  The mean is off by d = 58 FP32 mean|h|, h - mean by that and a rounding of the
    difference; the mean square of the centred row by d^2 and 62 roundings of itself, and the root halves that."""
    h = h.double()
    mean = h.mean(-1, keepdim=True)
    var = (h - mean).square().mean(-1, keepdim=True)
    r = 1.0 / (var + eps).sqrt()
    n = (h - mean) * r
    d = 58 * FP32 * h.abs().mean(-1, keepdim=True)
    off = r * (d + FP32 * (h - mean).abs()) + n.abs() * (d * d * r * r / 2 + 40 * FP32)
    return mean, r, n, off


def layer_norm(h, weight, bias, eps):
    """(y, bound before the rounding at the store)."""
    _, _, n, off = parts(h, eps)
    w = weight.double()
    y = n * w
    if bias is not None:
        y = y + bias.double()
    return y, w.abs() * off + 2 * FP32 * ((n * w).abs() + y.abs())


def layer_norm_grad(dy, dsum, h, weight, eps):
    """(dx, dw, db) and the bounds of the three before their rounding; `adds` additions of a share make those of dw and db."""
    H = h.shape[-1]
    dy, w = dy.double(), weight.double()
    _, r, n, off = parts(h, eps)
    t = w * dy
    mean_t, mean_tn = t.mean(-1, keepdim=True), (t * n).mean(-1, keepdim=True)
    abs_t, abs_tn = t.abs().mean(-1, keepdim=True), (t * n).abs().mean(-1, keepdim=True)
    dx = r * (t - mean_t - n * mean_tn)
    off_tn = (t.abs() * off).mean(-1, keepdim=True) + 62 * FP32 * abs_tn
    bound = r * (62 * FP32 * abs_t + 4 * FP32 * t.abs() + off * mean_tn.abs() + n.abs() * off_tn + 4 * FP32 * n.abs() * abs_tn) + 40 * FP32 * (dx.abs() + r * (t.abs() + abs_t))
    d2 = (58 * FP32 * h.double().abs().mean(-1, keepdim=True) * r)**2 / 2
    bound = bound + d2 * r * (t.abs() + abs_t + n.abs() * abs_tn)
    if dsum is not None:
        dx = dx + dsum.double()
        bound = bound + FP32 * (dsum.double().abs() + dx.abs())
    rows = lambda v: v.reshape(-1, H).sum(0)
    return (dx, rows(dy * n), rows(dy)), (bound, (rows(dy.abs() * off), rows((dy * n).abs())), rows(dy.abs()))
