"""Operators that serve many conversations from one pool of memory and make drafted tokens exact, as a list of measurable cases.

Kinds
  append     the rows of a QKV product go into the pages of a 16-bit key/value cache: norms of the query and key heads and the rotation (of the whole head or its first
             part) on the way, the rotated queries come out.  The outputs are the queries and the whole pool
  attention  query rows over the pages: single steps of one or many conversations (``queries`` = 1), a few drafted tokens of each, or the chunk of a prompt
  verify     the target's logits of drafted tokens: how many of them stand, and the token behind them, from given uniform numbers.  ``draft``: with the draft's logits, else
             the drafts were looked up, not sampled

Position p of sequence s lies in page tables[s][p / page_size] of the pool, in row p % page_size.

``draw`` gives cases of the same ranges: heads of 32 to 256 with 1 to 16 query heads on a key head, 1 to 64 sequences, up to 131072 keys, pages of 1 to 256 positions, 1 to
16 drafted tokens, chunks of 17 to 512, vocabularies of 1000 to 151936, FP16 and BF16 caches, FP32, FP16 and BF16 rows.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

EPS = 1e-6
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


def _append(name, tokens, heads, kv_heads, head, rows, cache, page, norm, layout, rotated, seqs=1, start=0):
    return {"name": name, "kind": "append", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head": head, "rows": rows, "cache": cache, "page": page, "norm": norm,
            "layout": layout, "rotated": rotated, "seqs": seqs, "start": start}


def _attention(name, heads, kv_heads, head, seqs, queries, keys, cache, page, out, window=0, empty=False):
    return {"name": name, "kind": "attention", "heads": heads, "kv_heads": kv_heads, "head": head, "seqs": seqs, "queries": queries, "keys": keys, "cache": cache, "page": page,
            "out": out, "window": window, "empty": empty}


def _verify(name, seqs, drafts, vocab, dtype, draft, temperature, pad=0, ragged=False):
    return {"name": name, "kind": "verify", "seqs": seqs, "drafts": drafts, "vocab": vocab, "dtype": dtype, "draft": draft, "temperature": temperature, "pad": pad, "ragged": ragged}


def listed():
    return [
        # the smallest call: one decode step's row of an 8B model, pairs of neighbours turned
        _append("append_step", 1, 32, 8, 128, "bf16", "bf16", 16, False, "interleaved", 128, start=700),
        # a prompt chunk of a model with normed heads, deep in its context
        _append("append_chunk", 512, 32, 8, 128, "bf16", "bf16", 64, True, "half", 128, start=3584),
        # a step of many conversations at once, FP32 rows, the first 64 of 96 entries turned
        _append("append_batch", 61, 24, 8, 96, "f32", "f16", 32, False, "half", 64, seqs=61, start=1037),
        # attention of one decode step early in a chat
        _attention("step_short", 32, 8, 128, 1, 1, 101, "bf16", 16, "bf16"),
        # the same at the end of a very long document
        _attention("step_long", 32, 8, 128, 1, 1, 131071, "bf16", 64, "bf16"),
        # a step of a batch of conversations of very different lengths, one of them without a key
        _attention("step_batch", 32, 8, 64, 48, 1, 4099, "f16", 16, "f32", empty=True),
        # the drafted tokens of several conversations
        _attention("drafts_batch", 32, 8, 128, 16, 5, 8191, "bf16", 32, "bf16"),
        # a chunk of a long prompt
        _attention("chunk_long", 32, 8, 128, 1, 512, 8192, "bf16", 64, "bf16"),
        # ragged chunks of several prompts through a sliding window
        _attention("chunk_window", 24, 8, 96, 3, 111, 1999, "f16", 16, "f16", window=500),
        # one conversation's drafts, looked up in its own text
        _verify("verify_step", 1, 4, 128256, "f32", False, 1.0),
        # a batch of conversations, drafts sampled from a small model
        _verify("verify_batch", 32, 5, 128256, "f32", True, 0.7, ragged=True),
        # most likely tokens only, 16-bit logits of an odd vocabulary cut out of padded rows
        _verify("verify_greedy", 7, 3, 50257, "bf16", False, 0.0, pad=47, ragged=True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


HEADS = ((32, 8, 128), (32, 8, 64), (24, 8, 96), (16, 16, 64), (16, 2, 128), (8, 1, 256), (16, 1, 64), (12, 4, 32))
PAGES = (1, 8, 16, 32, 64, 256)


def draw(rng):
    kind = rng.choice(("append", "attention", "attention", "verify"))
    if kind == "verify":
        vocab = rng.choice((_spread(rng, 1000, 131072), 128256, 151936, 50257))
        drafts = rng.choice((0, 1, 2, 3, 4, 5, 8))
        seqs = max(1, min(64, _spread(rng, 1, 64), 32 * 11 * 128256 // (vocab * (2 * drafts + 1))))
        temperature = rng.choice((0.0, 0.7, 1.0, 1.3))
        case = _verify("", seqs, drafts, vocab, rng.choice(tuple(TYPES)), drafts > 0 and temperature > 0 and rng.random() < 0.5, temperature, rng.choice((0, 0, 1, 64)), rng.random() < 0.5)
    else:
        heads, kv_heads, head = rng.choice(HEADS)
        cache, page = rng.choice(("f16", "bf16")), rng.choice(PAGES)
        if kind == "append":
            seqs = rng.choice((1, _spread(rng, 1, 64)))
            tokens = seqs if seqs > 1 else _spread(rng, 1, 512)
            case = _append("", tokens, heads, kv_heads, head, rng.choice(tuple(TYPES)), cache, page, rng.random() < 0.5, rng.choice(("half", "interleaved")),
                           rng.choice((head, head, head // 2, head // 4)), seqs, _spread(rng, 1, 4000) - 1)
        elif rng.random() < 0.7:
            seqs, queries = rng.choice((1, _spread(rng, 1, 64))), rng.choice((1, 1, 2, 5, 8, 16))
            keys = max(queries, _spread(rng, 1, 131072 // seqs))
            case = _attention("", heads, kv_heads, head, seqs, queries, keys, cache, page, rng.choice(("f32", cache)), rng.choice((0, 0, 300)), seqs > 1 and rng.random() < 0.5)
        else:
            seqs = rng.choice((1, 1, 2, 5))
            queries = max(17, _spread(rng, 17, 512) // seqs)
            keys = max(queries, _spread(rng, queries, 8192) // seqs)
            case = _attention("", heads, kv_heads, head, seqs, queries, keys, cache, page, rng.choice(("f32", cache, cache)), rng.choice((0, 0, 300)), seqs > 1 and rng.random() < 0.5)
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


def _size(dtype):
    return 4 if dtype == "f32" else 2


def work(case):
    if case["kind"] == "verify":
        rows = case["seqs"] * (2 * case["drafts"] + 1 if case["draft"] else case["drafts"] + 1)  # (how many of them a pass can do without hangs on their values)
        n = rows * case["vocab"]
        return {"bytes": n * _size(case["dtype"]) + case["seqs"] * (12 * case["drafts"] + 12), "flops": 5 * n}
    H, G, hs = case["heads"], case["kv_heads"], case["head"]
    if case["kind"] == "append":
        n = case["tokens"]
        return {"bytes": n * ((H + 2 * G) * hs * (_size(case["rows"]) + 2) + 4 * case["rotated"] + 8), "flops": 10 * n * (H + 2 * G) * hs}
    window, seen, read = case["window"] or 1 << 30, 0, 0
    positions = _positions(case)
    for s, length in enumerate(_lengths(case)):
        mine = [p for p in positions[s * case["queries"]:(s + 1) * case["queries"]] if p >= 0]
        seen += sum(min(p + 1, window) for p in mine)
        read += min(length, window + len(mine) - 1) if mine else 0
    return {"bytes": read * G * hs * 4 + 4 * (read // case["page"]) + len(positions) * (H * hs * (2 + _size(case["out"])) + 8), "flops": 4 * H * hs * seen}


# ---- inputs ---------------------------------------------------------------------------------------------------------------------------
def _normal(gen, *shape):
    return torch.randn(shape, device="cuda", generator=gen)


def _pool(case, gen):
    """The pool's keys and values and every sequence's pages, in any order; some pages belong to nobody.  Rows as a model leaves them: channels of very different strength in the keys."""
    G, hs, page, seqs = case["kv_heads"], case["head"], case["page"], case["seqs"]
    width = -(-_context(case) // page)
    pages = seqs * width + 3
    tables = torch.randperm(pages, device="cuda", generator=gen)[:seqs * width].to(torch.int32).view(seqs, width)
    gain = torch.exp(0.7 * _normal(gen, G, 1, hs))
    shift = 0.3 * _normal(gen, G, 1, hs)
    dtype = TYPES[case["cache"]]
    return {"keys": torch.addcmul(shift, _normal(gen, pages, G, page, hs), gain).to(dtype), "values": (_normal(gen, pages, G, page, hs) * 0.4).to(dtype), "tables": tables}


def _verify_inputs(case, gen):
    S, K, V = case["seqs"], case["drafts"], case["vocab"]
    wide = _normal(gen, S, K + 1, V + case["pad"]) * 2.0
    few = torch.randint(0, V, (S, K + 1, 8), device="cuda", generator=gen)
    wide.scatter_add_(2, few, 9.0 + 2.0 * _normal(gen, S, K + 1, 8))  # a model is sure of a few tokens
    wide = wide.to(TYPES[case["dtype"]])
    near = wide[:, :K, :V].float() + 0.5 * _normal(gen, S, K, V)  # what a smaller model thinks
    race = -torch.log(torch.rand((S, K, V), device="cuda", generator=gen).clamp(min=1e-30))
    drafts = (near / max(case["temperature"], 0.5) - torch.log(race)).argmax(-1).to(torch.int32) if K else torch.zeros(S, 0, device="cuda", dtype=torch.int32)  # sampled from it
    if case["ragged"]:  # conversations with fewer drafts
        for s in range(S):
            drafts[s, K - s % (K + 1):] = -1
    draft = near.to(TYPES[case["dtype"]]) if case["draft"] else None
    return {"logits": wide[..., :V], "drafts": drafts, "uniforms": torch.rand((S, K + 1), device="cuda", generator=gen), "draft_logits": draft}


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "verify":
        return _verify_inputs(case, gen)
    H, G, hs = case["heads"], case["kv_heads"], case["head"]
    d = _pool(case, gen)
    if case["kind"] == "append":
        n, r = case["tokens"], case["rotated"]
        qkv = (_normal(gen, n, (H + 2 * G) * hs) * 1.3).to(TYPES[case["rows"]])
        step = torch.arange(n, device="cuda", dtype=torch.int32)
        angles = torch.arange(_context(case), device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)
        d.update(q=qkv[:, :H * hs].view(n, H, hs), k=qkv[:, H * hs:(H + G) * hs].view(n, G, hs), v=qkv[:, (H + G) * hs:].view(n, G, hs), cos=angles.cos().float(), sin=angles.sin().float(),
                 q_norm=None, k_norm=None)
        if case["norm"]:
            d["q_norm"], d["k_norm"] = 1 + 0.2 * _normal(gen, hs), 1 + 0.2 * _normal(gen, hs)
        if case["seqs"] == 1:  # a chunk of one sequence
            return dict(d, sequences=torch.zeros_like(step), positions=case["start"] + step)
        return dict(d, sequences=step, positions=(case["start"] - 13 * step).clamp(min=0))  # a step of each of many
    positions = torch.tensor(_positions(case), device="cuda", dtype=torch.int32)
    q = (_normal(gen, len(positions), H, hs) * 1.4).to(TYPES[case["cache"]])
    return dict(d, q=q, positions=positions, sequences=torch.arange(case["seqs"], device="cuda", dtype=torch.int32).repeat_interleave(case["queries"]))


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=dict(case))
    if own and case["kind"] != "verify":
        keys, values = state["keys"], state.pop("values")
        cache = _package().PagedKVCache(keys.shape[0], case["page"], case["kv_heads"], case["head"], dtype=keys.dtype)
        cache.keys.copy_(state.pop("keys"))
        cache.values.copy_(values)
        state["cache"] = cache
    return state


# ---- the plain forms ------------------------------------------------------------------------------------------------------------------
def _turn(x, weight, cos, sin, positions, layout):
    x = x.float()
    if weight is not None:
        x = weight * (x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS))
    cos, sin = cos[positions.long()][:, None], sin[positions.long()][:, None]
    x, rest = x[..., :2 * cos.shape[-1]], x[..., 2 * cos.shape[-1]:]
    a, b = x.chunk(2, -1) if layout == "half" else (x[..., 0::2], x[..., 1::2])
    a, b = a * cos - b * sin, a * sin + b * cos
    return torch.cat((a, b, rest) if layout == "half" else (torch.stack((a, b), -1).flatten(-2), rest), -1)


def _append_plain(s, case):
    q = _turn(s["q"], s["q_norm"], s["cos"], s["sin"], s["positions"], case["layout"])
    k = _turn(s["k"], s["k_norm"], s["cos"], s["sin"], s["positions"], case["layout"])
    at = s["positions"].long()
    page = s["tables"][s["sequences"].long(), at // case["page"]].long()
    s["keys"][page, :, at % case["page"]] = k.to(s["keys"].dtype)
    s["values"][page, :, at % case["page"]] = s["v"].float().to(s["values"].dtype)
    return {"q": q.to(s["keys"].dtype), "keys": s["keys"], "values": s["values"]}


def _attention_plain(s, case):
    H, G, hs, n, nq = case["heads"], case["kv_heads"], case["head"], case["seqs"], case["queries"]
    pages = s["tables"].long()
    k, v = (s[name][pages].transpose(1, 2).flatten(2, 3).float() for name in ("keys", "values"))  # [n, G, positions, hs]
    q = s["q"].float().view(n, nq, G, H // G, hs).transpose(1, 2).reshape(n, G, -1, hs)
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


def _softmax(x, temperature):
    x = (x.double() - x.double().amax(-1, keepdim=True)) / temperature
    e = torch.exp(x)
    return e / e.sum(-1, keepdim=True)


def _verify_plain(s, case):
    """In 64 bits throughout: a token is a whole number, and a uniform number may fall next to the border of two."""
    logits, drafts, uniforms, K = s["logits"], s["drafts"].long(), s["uniforms"].double(), case["drafts"]
    S, V = logits.shape[0], logits.shape[2]
    given, chosen = drafts >= 0, drafts.clamp(min=0)[..., None]
    if case["temperature"] == 0.0:
        best = torch.where(logits == logits.amax(-1, keepdim=True), torch.arange(V, device="cuda"), V).amin(-1)
        stands = given & (best[:, :K] == drafts)
    else:
        p = _softmax(logits, case["temperature"])
        q = _softmax(s["draft_logits"], case["temperature"]) if case["draft"] else None
        mine = p[:, :K].gather(2, chosen)[..., 0]
        stands = given & (uniforms[:, :K] * (q.gather(2, chosen)[..., 0] if q is not None else 1.0) < mine)
    accepted = stands.long().cumprod(1).sum(1)
    rows = torch.arange(S, device="cuda")
    if case["temperature"] == 0.0:
        token = best[rows, accepted]
    else:
        p = p[rows, accepted]
        w = p
        if K:
            last = accepted.clamp(max=K - 1)
            refused = (accepted < K) & given[rows, last]
            less = q[rows, last] if q is not None else torch.zeros_like(p).scatter(1, chosen[rows, last], 1.0)
            w = torch.where(refused[:, None], (p - less).clamp(min=0.0), p)
            w = torch.where(w.sum(1, keepdim=True) > 0, w, p)
        total = w.cumsum(1)
        past = total > uniforms[:, K:] * total[:, -1:]
        token = torch.where(past, torch.arange(V, device="cuda"), V).amin(1)
    at = torch.arange(K + 1, device="cuda")
    tokens = torch.cat((drafts, drafts.new_full((S, 1), -1)), 1)
    tokens = torch.where(at < accepted[:, None], tokens, torch.where(at == accepted[:, None], token[:, None], -1))
    return {"tokens": tokens.to(torch.int32), "accepted": accepted.to(torch.int32)}


def run(state):
    case = state["case"]
    if case["kind"] == "append":
        if not own:
            return _append_plain(state, case)
        cache = state["cache"]
        q = cache.append(state["k"], state["v"], state["positions"], state["tables"], sequences=state["sequences"], q=state["q"], q_norm=state["q_norm"], k_norm=state["k_norm"], eps=EPS,
                         cos=state["cos"], sin=state["sin"], layout=case["layout"])
        return {"q": q, "keys": cache.keys, "values": cache.values}
    if case["kind"] == "attention":
        if not own:
            return _attention_plain(state, case)
        return state["cache"].attention(state["q"], state["positions"], state["tables"], sequences=state["sequences"], window=case["window"], max_len=case["keys"], chunk=case["queries"],
                                        dtype=TYPES[case["out"]])
    if not own:
        return _verify_plain(state, case)
    tokens, accepted = _package().verify_drafts(state["logits"], state["drafts"], state["uniforms"], draft_logits=state["draft_logits"], temperature=case["temperature"])
    return {"tokens": tokens, "accepted": accepted}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------------
def _exact_append(case, d):
    hs, r = case["head"], case["rotated"]
    first = torch.arange(r // 2, device="cuda") * (1 if case["layout"] == "half" else 2)
    second = first + (r // 2 if case["layout"] == "half" else 1)
    angle = torch.complex(d["cos"].double(), d["sin"].double())[d["positions"].long()]

    def turned(x, weight):
        x = x.double()
        if weight is not None:
            x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / hs + EPS) * weight.double()
        z = torch.complex(x[..., first], x[..., second]) * angle[:, None, :]
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    keys, values, k = d["keys"].double(), d["values"].double(), turned(d["k"], d["k_norm"])
    tables = d["tables"].tolist()
    for row, (position, sequence) in enumerate(zip(d["positions"].tolist(), d["sequences"].tolist())):
        page, within = tables[sequence][position // case["page"]], position % case["page"]
        keys[page, :, within], values[page, :, within] = k[row], d["v"][row].double()
    return {"q": turned(d["q"], d["q_norm"]), "keys": keys, "values": values}


def _exact_attention(case, d):
    H, G, hs, nq = case["heads"], case["kv_heads"], case["head"], case["queries"]
    q, out = d["q"].double(), torch.zeros(len(d["positions"]), H, hs, device="cuda", dtype=torch.float64)
    for s, length in enumerate(_lengths(case)):
        if length == 0:
            continue
        at = torch.arange(length, device="cuda")
        page = d["tables"][s].long()[at // case["page"]]
        k, v = (d[name][page, :, at % case["page"]].double() for name in ("keys", "values"))  # [length, G, hs]
        mine = slice(s * nq, (s + 1) * nq)
        gap = d["positions"][mine, None].long() - at
        hidden = (gap < 0) | (gap >= (case["window"] or 1 << 30))
        some = ~hidden.all(-1)
        for h in range(H):
            x = torch.einsum("id,jd->ij", q[mine, h], k[:, h * G // H]) / math.sqrt(hs)
            p = torch.softmax(x.masked_fill(hidden, -math.inf)[some], -1)
            o = torch.zeros(nq, hs, device="cuda", dtype=torch.float64)
            o[some] = p @ v[:, h * G // H]
            out[mine, h] = o
    return out


def _exact_verify(case, d):
    """A conversation at a time, a draft at a time."""
    T, K = case["temperature"], case["drafts"]
    tokens = torch.full((case["seqs"], K + 1), -1, device="cuda", dtype=torch.int32)
    accepted = torch.zeros(case["seqs"], device="cuda", dtype=torch.int32)
    drafts, uniforms = d["drafts"].tolist(), d["uniforms"].double().tolist()
    for s in range(case["seqs"]):
        n, weights = 0, None
        while True:
            x = d["logits"][s, n].double()
            token = drafts[s][n] if n < K else -1
            if T == 0.0:
                best = int((x == x.max()).nonzero()[0])
                if token < 0 or token != best:
                    break
            else:
                p = torch.log_softmax(x / T, -1).exp()
                weights = p
                if token < 0:
                    break
                q = torch.log_softmax(d["draft_logits"][s, n].double() / T, -1).exp() if case["draft"] else None
                if not uniforms[s][n] * (1.0 if q is None else float(q[token])) < float(p[token]):
                    weights = p.clone()
                    if q is None:
                        weights[token] = 0.0
                    else:
                        weights -= torch.minimum(p, q)
                    if float(weights.sum()) <= 0.0:
                        weights = p
                    break
            tokens[s, n] = token
            n += 1
        if T > 0.0:
            border = weights.cumsum(0)
            best = int(torch.searchsorted(border, border[-1:] * uniforms[s][K], right=True))
        tokens[s, n], accepted[s] = best, n
    return {"tokens": tokens, "accepted": accepted}


def exact(case, seed):
    return {"append": _exact_append, "attention": _exact_attention, "verify": _exact_verify}[case["kind"]](case, _inputs(case, seed))
