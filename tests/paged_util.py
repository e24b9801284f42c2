"""Plain 64-bit forms of the operators on pages and of the verification of drafts (torch on the CPU), and the bounds that their kernels are held to."""
import math

import torch

import kv4_util as U


def turn(x, weight, eps, cos, sin, positions, layout):
    """Norm and rotation of the first 2 * cos.shape[1] entries of rows [n, heads, hs], in float64."""
    x = U.turn(x, weight, eps, None, None, positions, layout)
    if cos is None:
        return x
    r = 2 * cos.shape[1]
    return torch.cat((U.turn(x[..., :r], None, eps, cos, sin, positions, layout), x[..., r:]), -1)


def rounding(want, off, dtype):
    """Half a step of a result that may be off by ``off`` before it is rounded; FP16 results below its normal range: half of 2^-24."""
    return off + (want.abs() + off) * U.half_step(dtype) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126)


def attention(q, keys, values, positions, sequences, tables, scale=None, window=0, dtype=torch.float64, probability=0.0):
    """(out, bound) in float64: a row at a time, over the positions that have a page.

    The bound.  Products of two 16-bit numbers are exact; a score's sum of hs of them, which the tensor core may cut rather than round, is off by at most hs 2^-22 of A = |scale| sum |q| |k|, its scaling and
    the subtraction of the reference by 4 of 2^-24 of that.  A probability's relative error is twice that (numerator and sum), 2^-20 for its exponential, 2^-17 for the two numbers that hold
    it (BF16; FP16's 2^-22 is less).  FP16 loses what is below 2^-25 of a row whose largest is at least 2^7: 2^-32 a position.  Sums of m products, 16 an instruction, two instructions each:
    (m / 8 + 32) 2^-22.  With 16-bit results a probability is one number, half a step off (``probability``), while their sum has it as it was: that much more of sum p |v|.  Then the
    result's own half step."""
    n, H, hs = q.shape
    pages, G, page, _ = keys.shape
    scale = 1.0 / math.sqrt(hs) if scale is None else scale
    q, keys, values = (t.double().cpu() for t in (q, keys, values))
    positions, tables = positions.tolist(), tables.tolist()
    sequences = [0] * n if sequences is None else sequences.tolist()
    out, bound = torch.zeros(n, H, hs, dtype=torch.float64), torch.zeros(n, H, hs, dtype=torch.float64)
    for r in range(n):
        p, s = positions[r], sequences[r]
        if s < 0 or s >= len(tables) or p < 0 or p >= len(tables[s]) * page:
            continue
        at = [j for j in range(max(0, p - window + 1) if window else 0, p + 1) if 0 <= tables[s][j // page] < pages]
        if not at:
            continue
        where = torch.tensor([tables[s][j // page] for j in at]), torch.tensor([j % page for j in at])
        k, v = (t[where[0], :, where[1]].transpose(0, 1) for t in (keys, values))  # [G, m, hs]
        x = q[r].view(G, H // G, hs)
        w = torch.softmax(x @ k.transpose(1, 2) * scale, -1)
        out[r] = (w @ v).view(H, hs)
        A = (x.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) * abs(scale)
        off = (w @ v.abs()) * (2 * A * (hs * 2.0 ** -22 + 4 * 2.0 ** -24) + 2.0 ** -20 + 2.0 ** -17 + probability + (len(at) / 8 + 32) * 2.0 ** -22)
        bound[r] = (off + len(at) * 2.0 ** -32 * v.abs().amax(1, keepdim=True)).reshape(H, hs)
    return out, rounding(out, bound, dtype) if dtype != torch.float64 else bound


def verify(logits, drafts, uniforms, draft_logits, temperature):
    """(tokens, accepted) by the definition, a sequence and a draft at a time, in float64 on the CPU."""
    S, K, V = logits.shape[0], logits.shape[1] - 1, logits.shape[2]
    logits, drafts = logits.double().cpu(), drafts.tolist()
    y = None if draft_logits is None or temperature == 0 else draft_logits.double().cpu()
    tokens, accepted = torch.full((S, K + 1), -1, dtype=torch.int32), torch.zeros(S, dtype=torch.int32)

    def row(x):
        if torch.isnan(x).any() or not math.isfinite(float(x.max())):
            return None
        e = torch.exp((x - x.max()) / temperature) if temperature else (torch.arange(V) == int((x == x.max()).nonzero()[0])).double()
        return e / e.sum()

    for s in range(S):
        n = 0
        while True:
            p = row(logits[s, n])
            d = drafts[s][n] if n < K and 0 <= drafts[s][n] < V else -1
            q = row(y[s, n]) if y is not None and d >= 0 else None
            if p is None or (d >= 0 and y is not None and q is None):
                w = None
                break
            if temperature == 0:
                w = p
                if d < 0 or float(p[d]) == 0:
                    break
            elif d < 0:
                w = p
                break
            elif not float(uniforms[s, n]) * (1.0 if q is None else float(q[d])) < float(p[d]):
                w = (p - q).clamp(min=0) if q is not None else p * (torch.arange(V) != d)
                w = w if float(w.sum()) > 0 else p
                break
            tokens[s, n] = d
            n += 1
        accepted[s] = n
        if w is not None:
            run = w.cumsum(0)
            past = (run > (float(uniforms[s, K]) if temperature else 0.5) * float(run[-1])) & (w > 0)
            tokens[s, n] = int((past if past.any() else w > 0).nonzero()[0 if past.any() else -1])
    return tokens, accepted
