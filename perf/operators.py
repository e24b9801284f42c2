"""Operators that serve long contexts and score tokens, as a list of measurable cases.

Kinds
  append     the rows of a QKV product go into a 4-bit key/value cache: norms of the query and key heads and the rotation on the way, the
             rotated queries come out.  The pass ends with a read of what was stored, as the values that the four bits stand for
  attention  query rows over a 4-bit cache: single steps of one or many sequences (``queries`` = 1) or the chunk of a prompt
  log_probs  logits rows and a token for each: its log probability, the row's entropy and the most likely alternatives

A cache holds groups of 32 neighbouring entries of a head: a scale d in 16 bits and codes c of 4 bits, value d * (c - 8).

``draw`` gives cases of the same ranges: heads of 32 to 256 with 1 to 16 query heads on a key head, 1 to 64 sequences, up to 131072 keys,
chunks of 2 to 512 tokens, vocabularies of 1000 to 151936, FP32, FP16 and BF16 rows.
"""
import functools
import importlib.util
import math
import os
import sys

import torch

own = False

GROUP = 32  # entries that share a scale
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _package():
    """The package's folder has a dot in its name: it is registered under the alias the framework documents."""
    name = "gpullama3_java_b200"
    if name not in sys.modules:
        root = os.path.join(os.getcwd(), "gpullama3.java_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(root, "__init__.py"), submodule_search_locations=[root])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


def _append(name, tokens, heads, kv_heads, head, dtype, norm, layout, seqs=1, start=0):
    return {"name": name, "kind": "append", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head": head, "dtype": dtype, "norm": norm, "layout": layout, "seqs": seqs,
            "start": start}


def _attention(name, heads, kv_heads, head, seqs, queries, keys, out, window=0, empty=False):
    return {"name": name, "kind": "attention", "heads": heads, "kv_heads": kv_heads, "head": head, "seqs": seqs, "queries": queries, "keys": keys, "out": out, "window": window,
            "empty": empty}


def _log_probs(name, rows, vocab, top, dtype, pad=0):
    return {"name": name, "kind": "log_probs", "rows": rows, "vocab": vocab, "top": top, "dtype": dtype, "pad": pad}


def listed():
    return [
        # the smallest call: one decode step's row of an 8B model, pairs of neighbours turned
        _append("append_step", 1, 32, 8, 128, "f32", False, "interleaved", start=700),
        # a prompt chunk of a model with normed heads, deep in its context
        _append("append_chunk", 512, 32, 8, 128, "f32", True, "half", start=3584),
        # a step of many conversations at once, heads of 96, rows of a 16-bit product
        _append("append_batch", 61, 24, 8, 96, "bf16", True, "half", seqs=61, start=37),
        # attention of one decode step early in a chat
        _attention("step_short", 32, 8, 128, 1, 1, 101, "f32"),
        # the same at the end of a very long document
        _attention("step_long", 32, 8, 128, 1, 1, 131071, "f32"),
        # a step of a batch of conversations of very different lengths, one of them without a key
        _attention("step_batch", 32, 8, 64, 48, 1, 4099, "f32", empty=True),
        # a chunk of a long prompt
        _attention("chunk_long", 32, 8, 128, 1, 512, 8192, "bf16"),
        # ragged chunks of several prompts through a sliding window
        _attention("chunk_window", 24, 8, 96, 3, 111, 1999, "bf16", window=500),
        # log probability of the token that a decode step chose
        _log_probs("logprob_step", 1, 128256, 5, "f32"),
        # a prompt chunk is scored: every row of it, with the usual most alternatives
        _log_probs("logprob_chunk", 512, 128256, 20, "f32"),
        # 16-bit logits of an odd vocabulary, rows cut out of padded ones, no alternatives wanted
        _log_probs("logprob_odd", 77, 50257, 0, "bf16", pad=47),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


HEADS = ((32, 8, 128), (32, 8, 64), (24, 8, 96), (16, 16, 64), (16, 2, 128), (8, 1, 256), (16, 1, 64), (12, 4, 32))


def draw(rng):
    kind = rng.choice(("append", "attention", "attention", "log_probs"))
    if kind == "log_probs":
        vocab = rng.choice((_spread(rng, 1000, 131072), 128256, 151936, 50257))
        rows = _spread(rng, 1, max(1, min(512, 512 * 128256 // vocab)))
        case = _log_probs("", rows, vocab, rng.choice((0, 1, 5, 20, 32)), rng.choice(tuple(TYPES)), rng.choice((0, 0, 1, 64)))
    else:
        heads, kv_heads, head = rng.choice(HEADS)
        if kind == "append":
            seqs = rng.choice((1, _spread(rng, 1, 64)))
            tokens = seqs if seqs > 1 else _spread(rng, 1, 512)
            case = _append("", tokens, heads, kv_heads, head, rng.choice(tuple(TYPES)), rng.random() < 0.5, rng.choice(("half", "interleaved")), seqs, _spread(rng, 1, 4000) - 1)
        elif rng.random() < 0.6:
            seqs = rng.choice((1, _spread(rng, 1, 64)))
            keys = _spread(rng, 1, 131072 // seqs if seqs > 1 else 131072)
            case = _attention("", heads, kv_heads, head, seqs, 1, keys, rng.choice(("f32", "bf16")), rng.choice((0, 0, 300)), seqs > 1 and rng.random() < 0.5)
        else:
            seqs = rng.choice((1, 1, 2, 5))
            queries = max(2, _spread(rng, 2, 512) // seqs)
            keys = max(queries, _spread(rng, queries, 8192) // seqs)
            case = _attention("", heads, kv_heads, head, seqs, queries, keys, "bf16" if queries * seqs > 32 else rng.choice(("f32", "bf16")), rng.choice((0, 0, 300)),
                              seqs > 1 and rng.random() < 0.5)
    del case["name"]
    return case


# ---- sizes ----------------------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Keys of every sequence: the longest has ``keys`` of them, the others from a share of that; ``empty``: the last has none."""
    n, most = case["seqs"], case["keys"]
    out = [max(1, most * (n - (5 * i) % n) // n) for i in range(n)]
    if case["empty"]:
        out[-1] = 0
    return out


def _positions(case):
    """Position of every query row: the last ones of its sequence; negative ones have no key."""
    return [length - case["queries"] + i for length in _lengths(case) for i in range(case["queries"])]


def _context(case):
    return case["start"] + (case["tokens"] if case["seqs"] == 1 else 1) if case["kind"] == "append" else case["keys"]


def work(case):
    if case["kind"] == "log_probs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + case["rows"] * (4 + 4 + 4 + 8 * case["top"]), "flops": 5 * n}
    H, G, hs = case["heads"], case["kv_heads"], case["head"]
    held = G * hs * 2 * (0.5 + 2 / GROUP)  # bytes of a position
    if case["kind"] == "append":
        n, size = case["tokens"], 4 if case["dtype"] == "f32" else 2
        values = n * G * hs * 2
        return {"bytes": n * (H + 2 * G) * hs * size + n * H * hs * 4 + n * held * 2 + values * 2, "flops": 10 * n * (H + 2 * G) * hs}
    window, seen, read = case["window"] or 1 << 30, 0, 0
    positions = _positions(case)
    for s, length in enumerate(_lengths(case)):
        mine = [p for p in positions[s * case["queries"]:(s + 1) * case["queries"]] if p >= 0]
        seen += sum(min(p + 1, window) for p in mine)
        read += min(length, window + len(mine) - 1) if mine else 0
    rows = len(positions)
    return {"bytes": read * held + rows * H * hs * (4 + (4 if case["out"] == "f32" else 2)), "flops": 4 * H * hs * seen}


# ---- inputs ---------------------------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape):
    return torch.randn(shape, device="cuda", generator=gen)


def _keys_values(case, gen, length):
    """Rows as a model leaves them: channels of very different strength in the keys."""
    G, hs = case["kv_heads"], case["head"]
    gain = torch.exp(0.7 * _normal(gen, G, hs))
    return _normal(gen, length, G, hs) * gain + 0.3 * _normal(gen, G, hs), _normal(gen, length, G, hs) * 0.4


def _inputs(case, seed):
    """What the case's call reads, apart from the cache: tensors by name, and for an attention the rows that fill the cache, sequence by sequence."""
    gen = _generator(seed)
    if case["kind"] == "log_probs":
        rows, vocab = case["rows"], case["vocab"]
        wide = _normal(gen, rows, vocab + case["pad"]) * 2.5
        few = torch.randint(0, vocab, (rows, 8), device="cuda", generator=gen)
        wide.scatter_add_(1, few, 6.0 + 2.0 * _normal(gen, rows, 8))  # a model is sure of a few tokens
        targets = few[:, 0].to(torch.int32)
        targets[::3] = torch.randint(0, vocab, (len(targets[::3]),), device="cuda", generator=gen, dtype=torch.int32)
        return {"logits": wide.to(TYPES[case["dtype"]])[:, :vocab], "targets": targets}
    H, G, hs = case["heads"], case["kv_heads"], case["head"]
    slots = torch.randperm(case["seqs"], device="cuda", generator=gen).to(torch.int32)
    if case["kind"] == "append":
        n = case["tokens"]
        qkv = (_normal(gen, n, (H + 2 * G) * hs) * 1.3).to(TYPES[case["dtype"]])
        step = torch.arange(n, device="cuda", dtype=torch.int32)
        angles = torch.arange(_context(case), device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, hs, 2, device="cuda", dtype=torch.float64) / hs)
        d = {"q": qkv[:, :H * hs].view(n, H, hs), "k": qkv[:, H * hs:(H + G) * hs].view(n, G, hs), "v": qkv[:, (H + G) * hs:].view(n, G, hs), "cos": angles.cos().float(),
             "sin": angles.sin().float(), "q_norm": None, "k_norm": None}
        if case["norm"]:
            d["q_norm"], d["k_norm"] = 1 + 0.2 * _normal(gen, hs), 1 + 0.2 * _normal(gen, hs)
        if case["seqs"] == 1:  # a chunk of one sequence
            return dict(d, slots=torch.zeros_like(step), positions=case["start"] + step)
        return dict(d, slots=slots, positions=(case["start"] - 13 * step).clamp(min=0))  # a step of each of many
    positions = torch.tensor(_positions(case), device="cuda", dtype=torch.int32)
    return {"q": _normal(gen, len(positions), H, hs) * 1.4, "positions": positions, "slots": slots.repeat_interleave(case["queries"]), "order": slots.tolist(),
            "rows": [_keys_values(case, gen, length) for length in _lengths(case)]}


EPS = 1e-6


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=dict(case))
    if case["kind"] == "log_probs":
        return state
    G, hs, context, seqs = case["kv_heads"], case["head"], _context(case), case["seqs"]
    if own:
        state["cache"] = _package().KV4Cache(seqs, context, G, hs)
    else:  # the same cache as plain tensors: two codes a byte and the scales, [keys, values][slot][head][position]
        state["cache"] = (torch.full((2, seqs, G, context, hs // 2), 0x88, device="cuda", dtype=torch.uint8),
                          torch.zeros((2, seqs, G, context, hs // GROUP), device="cuda", dtype=torch.float16))
    if case["kind"] == "attention":  # the sequences' past
        fill = state["cache"].append if own else functools.partial(_store, state["cache"])
        for slot, (k, v) in zip(state.pop("order"), state.pop("rows")):
            at = torch.arange(k.shape[0], device="cuda", dtype=torch.int32)
            fill(k, v, at, slots=torch.full_like(at, slot))
    return state


# ---- the plain forms ------------------------------------------------------------------------------------------------------------------
def _store(cache, k, v, positions, slots):
    codes, scales = cache
    x = torch.stack((k, v)).float().unflatten(-1, (-1, GROUP))
    first = x.abs().argmax(-1, keepdim=True)
    d = (x.gather(-1, first) / -8.0).clamp(-65504.0, 65504.0).half()
    c = torch.where(d == 0, torch.zeros_like(x), torch.round(x / d.float())).clamp(-8, 7) + 8
    c = c.to(torch.uint8).flatten(-2)
    codes[:, slots.long(), :, positions.long()] = (c[..., 0::2] | c[..., 1::2] << 4).transpose(0, 1)
    scales[:, slots.long(), :, positions.long()] = d.squeeze(-1).transpose(0, 1)


def _values(codes, scales):
    """codes [..., hs / 2], scales [..., hs / 32] -> [..., hs]"""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8.0
    return (c.unflatten(-1, (-1, GROUP)) * scales.float()[..., None]).flatten(-2)


def _turn(x, weight, cos, sin, positions, layout):
    x = x.float()
    if weight is not None:
        s = (1.0 / torch.sqrt((x.double() * x.double()).mean(-1, keepdim=True) + EPS)).float()
        x = weight * (s * x)
    cos, sin = cos[positions.long()][:, None], sin[positions.long()][:, None]
    a, b = x.chunk(2, -1) if layout == "half" else (x[..., 0::2], x[..., 1::2])
    a, b = a * cos - b * sin, a * sin + b * cos
    return torch.cat((a, b), -1) if layout == "half" else torch.stack((a, b), -1).flatten(-2)


def _append_plain(s, case):
    q = _turn(s["q"], s["q_norm"], s["cos"], s["sin"], s["positions"], case["layout"])
    k = _turn(s["k"], s["k_norm"], s["cos"], s["sin"], s["positions"], case["layout"])
    _store(s["cache"], k, s["v"], s["positions"], s["slots"])
    codes, scales = s["cache"]
    at = (slice(None), s["slots"].long(), slice(None), s["positions"].long())
    k, v = _values(codes[at], scales[at]).half().unbind(1)  # [n, 2, G, hs]
    return {"q": q, "k": k, "v": v}


def _attention_plain(s, case):
    H, G, hs, n, nq = case["heads"], case["kv_heads"], case["head"], case["seqs"], case["queries"]
    codes, scales = s["cache"]
    slots = s["slots"].view(n, nq)[:, 0].long()
    k, v = _values(codes[:, slots], scales[:, slots])  # [n, G, context, hs]
    q = s["q"].view(n, nq, G, H // G, hs).transpose(1, 2).reshape(n, G, -1, hs)
    x = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(hs))
    at = torch.arange(k.shape[2], device="cuda")
    pos = s["positions"].view(n, 1, nq, 1).expand(n, 1, nq, H // G).reshape(n, 1, -1, 1)
    seen = at <= pos
    if case["window"]:
        seen = seen & (at > pos - case["window"])
    x = x.masked_fill(~seen, float("-inf"))
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    z = e.sum(-1, keepdim=True)
    o = torch.where(z > 0, (e @ v) / z, torch.zeros_like(z))
    return o.view(n, G, nq, H // G, hs).transpose(1, 2).reshape(n * nq, H, hs).to(TYPES[case["out"]])


def _log_probs_plain(s, case):
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    y = x - m
    e = torch.exp(y)
    log_z = torch.log(e.sum(-1, dtype=torch.float64))
    entropy = log_z - (y * e).sum(-1, dtype=torch.float64) / e.sum(-1, dtype=torch.float64)
    chosen = y.gather(1, s["targets"].long()[:, None])[:, 0] - log_z
    values, ids = torch.sort(y, dim=-1, descending=True, stable=True)
    values, ids = values[:, :case["top"]], ids[:, :case["top"]]
    return {"logprobs": chosen.float(), "entropy": entropy.float(), "top_ids": ids.to(torch.int32), "top_logprobs": (values - log_z[:, None]).float()}


def run(state):
    case = state["case"]
    if case["kind"] == "append":
        if not own:
            return _append_plain(state, case)
        q = state["cache"].append(state["k"], state["v"], state["positions"], q=state["q"], slots=state["slots"], q_norm=state["q_norm"], k_norm=state["k_norm"], eps=EPS,
                                  cos=state["cos"], sin=state["sin"], layout=case["layout"])
        k, v = state["cache"].read(state["positions"], slots=state["slots"], dtype=torch.float16)
        return {"q": q, "k": k, "v": v}
    if case["kind"] == "attention":
        if not own:
            return _attention_plain(state, case)
        return state["cache"].attention(state["q"], state["positions"], slots=state["slots"], window=case["window"], max_len=case["keys"], chunk=case["queries"],
                                        dtype=TYPES[case["out"]])
    if not own:
        return _log_probs_plain(state, case)
    logprobs, entropy, ids, values = _package().log_probs(state["logits"], state["targets"], top=case["top"])
    return {"logprobs": logprobs, "entropy": entropy, "top_ids": ids, "top_logprobs": values}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------------
def _held(x):
    """What the cache gives back for rows x [..., hs]: the nearest of the sixteen multiples of the group's 16-bit scale."""
    g = x.double().reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    largest = g.abs() == g.abs().max(-1, keepdim=True).values
    step = ((g * (largest & (largest.cumsum(-1) == 1))).sum(-1, keepdim=True) / -8).to(torch.float16).double()
    n = torch.where(step == 0, torch.zeros_like(g), g / torch.where(step == 0, torch.ones_like(step), step)).round().clamp(-8, 7)
    return (n * step).reshape(x.shape)


def _exact_append(case, d):
    hs = case["head"]
    pair = (lambda i: (i, i + hs // 2)) if case["layout"] == "half" else (lambda i: (2 * i, 2 * i + 1))
    first, second = (torch.tensor([pair(i)[j] for i in range(hs // 2)], device="cuda") for j in (0, 1))
    angle = torch.complex(d["cos"].double(), d["sin"].double())[d["positions"].long()]

    def turned(x, weight):
        x = x.double()
        if weight is not None:
            x = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / hs + EPS) * weight.double()
        z = torch.complex(x[..., first], x[..., second]) * angle[:, None, :]
        y = torch.empty_like(x)
        y[..., first], y[..., second] = z.real, z.imag
        return y

    return {"q": turned(d["q"], d["q_norm"]), "k": _held(turned(d["k"], d["k_norm"])), "v": _held(d["v"])}


def _exact_attention(case, d):
    H, G, hs, nq = case["heads"], case["kv_heads"], case["head"], case["queries"]
    q, out = d["q"].double(), torch.zeros(len(d["positions"]), H, hs, device="cuda", dtype=torch.float64)
    for s, (k, v) in enumerate(d["rows"]):
        if k.shape[0] == 0:
            continue
        k, v = _held(k), _held(v)
        mine = slice(s * nq, (s + 1) * nq)
        gap = d["positions"][mine, None].long() - torch.arange(k.shape[0], device="cuda")
        hidden = (gap < 0) | (gap >= (case["window"] or 1 << 30))
        some = ~hidden.all(-1)
        for h in range(H):
            x = torch.einsum("id,jd->ij", q[mine, h], k[:, h * G // H]) / math.sqrt(hs)
            p = torch.softmax(x.masked_fill(hidden, -math.inf)[some], -1)
            o = torch.zeros(nq, hs, device="cuda", dtype=torch.float64)
            o[some] = p @ v[:, h * G // H]
            out[mine, h] = o
    return out


def _exact_log_probs(case, d):
    lp = torch.log_softmax(d["logits"].double(), -1)
    # by value, then by index: one key of both, since a row's order of equal values is part of the definition
    order = torch.argsort(-d["logits"].double(), dim=-1, stable=True)[:, :case["top"]]
    p = lp.exp()
    return {"logprobs": lp[torch.arange(len(lp), device="cuda"), d["targets"].long()], "entropy": -(p * lp).sum(-1), "top_ids": order.to(torch.int32), "top_logprobs": lp.gather(1, order)}


def exact(case, seed):
    return {"append": _exact_append, "attention": _exact_attention, "log_probs": _exact_log_probs}[case["kind"]](case, _inputs(case, seed))
