"""Plain 64-bit forms of the 4-bit cache's operators (numpy / torch on the CPU), and the bounds that their kernels are held to."""
import math

import numpy as np
import torch


def quantize(x: torch.Tensor):
    """Rows [..., hs] in FP32 -> (values in float64, scales in float64 [..., hs / 32]), by the definition: d = f16(m / -8), c = clamp(rint(x / d) + 8, 0, 15)."""
    x = x.float().cpu().numpy()
    g = x.reshape(*x.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        m = np.take_along_axis(g, np.argmax(np.abs(np.nan_to_num(g, nan=0.0, posinf=np.inf, neginf=-np.inf)), -1)[..., None], -1)
        d = np.clip(m * np.float32(-0.125), -65504, 65504).astype(np.float16).astype(np.float32)
        c = np.where(d == 0, 0, np.clip(np.rint(g / np.where(d == 0, 1, d)), -8, 7))
    bad = ~np.isfinite(g).all(-1, keepdims=True)
    d = np.where(bad, np.nan, d)
    v = c.astype(np.float64) * d.astype(np.float64)
    return torch.from_numpy(np.where(bad, np.nan, v).reshape(x.shape)), torch.from_numpy(d[..., 0].astype(np.float64))


def turn(x, weight, eps, cos, sin, positions, layout):
    """Norm and rotation of rows [n, heads, hs] in float64."""
    x = x.double().cpu()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double().cpu()
    if cos is None:
        return x
    c, s = cos.double().cpu()[positions.long().cpu()][:, None], sin.double().cpu()[positions.long().cpu()][:, None]
    h = x.shape[-1] // 2
    y = torch.empty_like(x)
    if layout == "half":
        a, b = x[..., :h], x[..., h:]
        y[..., :h], y[..., h:] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., 0::2], x[..., 1::2]
        y[..., 0::2], y[..., 1::2] = a * c - b * s, a * s + b * c
    return y


def attention(q, k, v, d, positions, slots, scale, window):
    """q [n, H, hs]; k, v [slots, context, G, hs] and their scales d (two of [slots, context, G, hs / 32]), all float64 on the CPU -> (out, bound) where bound is how far a kernel may
    be off in FP32.

    The bound: a query keeps 22 bits of its largest entry's magnitude and meets codes of at most 16 steps, so that a score's error is at most 2^-21 + hs 2^-24 (products and
    sums in FP32) of A = scale * max|q| * sum over groups of 32 * 16 |d|; a probability's relative error is twice that error (numerator and sum), plus 2^-20 for its exponential;
    its product with a value's scale keeps 16 bits (2^-16), and sums of n products in FP32 add n 2^-24 at most.  All relative to sum p |v|.  A value is (c - 8) d with c of up to 15,
    and the sums of p d c and of -8 p d go through the same accumulators: what they round, n / 16 + 16 times 2^-22 at most, is relative to 16 sum p |d|."""
    kd, vd = d
    n, H, hs = q.shape
    G = k.shape[2]
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for r in range(n):
        p, s = int(positions[r]), int(slots[r])
        lo = max(0, p - window + 1) if window else 0
        if p < 0:
            continue
        kk, vv, dk, dv = (t[s, lo:p + 1].transpose(0, 1) for t in (k, v, kd, vd))  # [G, positions, ...]
        x = q[r].view(G, H // G, hs)
        w = torch.softmax(x @ kk.transpose(1, 2) * scale, -1)
        A = scale * x.abs().amax(-1, keepdim=True) * dk.abs().sum(-1).amax(-1)[:, None, None] * 32 * 16
        out[r] = (w @ vv).view(H, hs)
        off = (w @ vv.abs()) * (2 * A * (2.0 ** -21 + hs * 2.0 ** -24) + 2.0 ** -16 + 2.0 ** -20 + (p + 1 - lo) * 2.0 ** -24)
        bound[r] = (off + (w @ dv.abs()).repeat_interleave(32, -1) * 16 * ((p + 1 - lo) / 16 + 16) * 2.0 ** -22).view(H, hs)
    return out, bound


def chunk_bound(q, k, v, positions, slots, scale, window, want, dtype):
    """How far the tensor-core form may be off ``want`` = attention(...)[0].  Its operands are FP16 (half a step: 2^-11 of each): queries and keys put at most 2^-10 of
    A = scale * sum |q| |k| on a score (and hs 2^-22 for sums in FP32), a probability's relative error is twice that (numerator and sum), plus 2^-11 for its rounding and 2^-11 for the
    value's, n 2^-22 for the sums, 2^-20 for exponentials: all relative to sum p |v|.  A probability below FP16's range (the largest is at least 2^-8 of the row's scale): 2^-25 each.
    At last the result's own half step."""
    n, H, hs = q.shape
    G = k.shape[2]
    bound = torch.zeros_like(want)
    for r in range(n):
        p, s = int(positions[r]), int(slots[r])
        lo = max(0, p - window + 1) if window else 0
        if p < 0:
            continue
        kk, vv = k[s, lo:p + 1].transpose(0, 1), v[s, lo:p + 1].transpose(0, 1).abs()  # [G, positions, hs]
        x, m = q[r].view(G, H // G, hs), p + 1 - lo
        w = torch.softmax(x @ kk.transpose(1, 2) * scale, -1)
        A = (x.abs() @ kk.abs().transpose(1, 2)).amax(-1, keepdim=True) * abs(scale)
        off = (w @ vv) * (2 * A * (2.0 ** -10 + hs * 2.0 ** -22) + 2 * 2.0 ** -11 + m * 2.0 ** -22 + 2.0 ** -20) + m * 2.0 ** -25 * vv.flatten(1).amax(-1)[:, None, None]
        bound[r] = off.view(H, hs)
    return bound + want.abs() * half_step(dtype) + 2.0 ** -25


def log_probs(x, targets, top):
    """(logprobs, entropy, ids, values) in float64 of rows x."""
    x = x.double().cpu()
    lp = torch.log_softmax(x, -1)
    p = lp.exp()
    entropy = -(torch.where(p > 0, p * lp, torch.zeros_like(p))).sum(-1)
    ids = torch.argsort(-x, dim=-1, stable=True)[:, :top]
    t = targets.long().cpu()
    ok = (t >= 0) & (t < x.shape[1])
    chosen = torch.where(ok, lp.gather(1, t.clamp(0, x.shape[1] - 1)[:, None])[:, 0], torch.zeros(len(t), dtype=torch.float64))
    return chosen, entropy, ids.int(), lp.gather(1, ids)


def tables(context, hs, base=10000.0):
    a = torch.arange(context, dtype=torch.float64)[:, None] * base ** (-torch.arange(0, hs, 2, dtype=torch.float64) / hs)
    return a.cos().float(), a.sin().float()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rsqrt(hs):
    return 1.0 / math.sqrt(hs)
