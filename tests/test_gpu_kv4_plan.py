"""GGUF plans that keep their keys and values in 4 bits, and the scoring of tokens, through the plan's own entry points.

The reference runs in 64 bits.  Rounding in front of the cache (FP32 sums, FP16 operands on the tensor cores, int8 activations of Q8_0 plans) moves an entry that lies next to the border
of two codes to the other one, by a whole step; so every stored entry is held against the reference's (half a step off it at most, and what rounding in front of the cache adds), and the
reference goes on with what the plan stored.  What is left are the tolerances of the FP32 cache's tests: FP16 products 2^-8 of the largest logit, Q8_0 plans the int8 rounding of
activations, 3 %."""
import numpy as np
import pytest
import torch

import kv4_util as U
import pibidra_util as P
from test_gpu_pibidra import make_plan

pytestmark = pytest.mark.gpu
FP16_TOL, Q8_TOL = 2.0 ** -8, 0.03


class Reference:
    """A GGUF model in float64 with a 4-bit cache, token by token."""

    def __init__(self, pkg, model):
        self.m, self.c, self.q8 = model, model.configuration, False
        self.pkg, self.keys, self.values = pkg, [[] for _ in range(self.c.n_layers)], [[] for _ in range(self.c.n_layers)]

    def get(self, name):
        kind, dims, raw = self.m.tensors[name]
        raw = np.ascontiguousarray(raw)
        G = self.pkg.gguf.GGMLType
        if int(kind) == int(G.F32):
            t = raw.view(np.float32).astype(np.float64)
        elif int(kind) == int(G.F16):
            t = raw.view(np.float16).astype(np.float64)
        else:
            self.q8 = True
            b = raw.reshape(-1, 34)
            t = (b[:, 2:].view(np.int8).astype(np.float64) * np.ascontiguousarray(b[:, :2]).view(np.float16).astype(np.float64)).reshape(-1)
        return t if len(dims) == 1 else t.reshape(dims[1], dims[0])

    def times(self, x, name):
        w = self.get(name)
        if self.q8:  # Q8_0 multiplies activations in blocks of 32 int8 with an FP16 scale
            b = x.reshape(-1, 32)
            d = np.abs(b).max(-1, keepdims=True) / 127.0
            s = np.divide(b, d, out=np.zeros_like(b), where=d != 0)
            x = (np.trunc(s + np.copysign(0.5, s)) * d.astype(np.float16).astype(np.float64)).reshape(-1)
        return w @ x

    def rms(self, x, w):
        return w * (x / np.sqrt((x * x).mean(-1, keepdims=True) + self.c.rms_norm_eps))

    def held(self, x, stored, noise):
        """What the plan stored for x [1, G, hs]: the nearest step, or the end of the range, of every entry."""
        step = U.quantize(x)[1].abs().repeat_interleave(32, -1)
        top = x.abs().view(1, x.shape[1], -1, 32).amax(-1).repeat_interleave(32, -1)
        stored = torch.from_numpy(stored.astype(np.float64)).view_as(x)
        d = (stored - x).abs()
        cut = x.abs() > 7.4 * step
        assert (d <= step * 0.51 + noise * top)[~cut].all() and (d <= step * 1.01 + noise * top).all(), (d / top).max()
        return stored

    def forward(self, token, pos, stored, noise):
        """``stored``: the plan's rows of this position, [layer] -> (keys, values)."""
        c, hs = self.c, self.c.head_size
        H, G = c.n_heads, c.n_kv_heads
        arch = {0: "llama", 1: "qwen3", 2: "phi3"}[c.arch]
        x = self.get("token_embd.weight")[token]
        angle = pos * c.rope_theta ** (-np.arange(0, hs, 2) / hs)
        cos, sin = torch.from_numpy(np.cos(angle))[None], torch.from_numpy(np.sin(angle))[None]
        layout = "interleaved" if arch == "llama" else "half"
        zero = torch.zeros(1, dtype=torch.long)
        for i in range(c.n_layers):
            p = f"blk.{i}."
            a = self.rms(x, self.get(p + "attn_norm.weight"))
            if arch == "phi3":
                q, k, v = np.split(self.times(a, p + "attn_qkv.weight"), [H * hs, (H + G) * hs])
            else:
                q, k, v = (self.times(a, p + f"attn_{n}.weight") for n in "qkv")
            q, k, v = (torch.from_numpy(np.ascontiguousarray(t)).view(1, -1, hs) for t in (q, k, v))
            if arch == "qwen3":
                q, k = (torch.from_numpy(self.rms(t.numpy(), self.get(p + f"attn_{n}_norm.weight"))) for t, n in ((q, "q"), (k, "k")))
            q, k = (U.turn(t, None, 0.0, cos, sin, zero, layout) for t in (q, k))
            self.keys[i].append(self.held(k, stored[i][0], noise))
            self.values[i].append(self.held(v, stored[i][1], noise))
            K, V = torch.cat(self.keys[i]), torch.cat(self.values[i])
            o = torch.empty(H, hs, dtype=torch.float64)
            for h in range(H):
                g = h // (H // G)
                o[h] = torch.softmax(K[:, g] @ q[0, h] / np.sqrt(hs), 0) @ V[:, g]
            x = x + self.times(o.reshape(-1).numpy(), p + "attn_output.weight")
            a = self.rms(x, self.get(p + "ffn_norm.weight"))
            if arch == "phi3":
                gate, up = np.split(self.times(a, p + "ffn_up.weight"), 2)
            else:
                gate, up = self.times(a, p + "ffn_gate.weight"), self.times(a, p + "ffn_up.weight")
            x = x + self.times(gate / (1 + np.exp(-gate)) * up, p + "ffn_down.weight")
        a = self.rms(x, self.get("output_norm.weight"))
        return self.times(a, "output.weight" if "output.weight" in self.m.tensors else "token_embd.weight")


def off(got, want):
    return np.abs(np.asarray(got, dtype=np.float64) - want).max() / np.abs(want).max()


def caches(plan, c):
    """[layer] -> (keys, values), each [context, kv width], as the plan holds them."""
    return [[plan.read_buffer(name, c.context_length * c.kv_dim, layer=i).reshape(c.context_length, -1) for name in ("key_cache", "value_cache")] for i in range(c.n_layers)]


def row(held, pos):
    return [(k[pos], v[pos]) for k, v in held]


def tokens(vocab, n, seed=3):
    return np.random.default_rng(seed).integers(0, vocab, n).tolist()


@pytest.mark.parametrize("shape", ["tiny-llama", "tiny-qwen3", "tiny-phi3", "tiny-phi3-gqa"])
@pytest.mark.parametrize("quant", ["F16", "Q8_0"])
def test_decode_over_four_bits(pkg, make_model, shape, quant):
    m = make_model(shape, getattr(pkg.gguf.GGMLType, quant), 300)
    plan, ref = pkg.B200MasterPlan.initialize_plan(m), Reference(pkg, m)
    c = m.configuration
    try:
        before = plan.device_bytes
        assert plan.kv_info() == (plan.KV_F32, c.n_layers * 300 * c.kv_dim * 8)
        plan.forward_decode(1, 0)
        plan.set_kv_mode("q4")
        plan.set_kv_mode("q4")  # again: nothing happens
        mode, held = plan.kv_info()
        assert mode == plan.KV_Q4 and held == c.n_layers * c.n_kv_heads * 19 * 18 * c.head_size
        assert plan.device_bytes - before < held + (4 << 20) + 148 * 128 * (c.head_size + 2) * 4 - c.n_layers * 300 * c.kv_dim * 8
        toks = tokens(c.vocab_size, 145)  # past the position from which another graph takes over
        got = [plan.forward_decode(t, p) for p, t in enumerate(toks)]
        tol = FP16_TOL if quant == "F16" else Q8_TOL
        held = caches(plan, c)
        want = [ref.forward(t, p, row(held, p), tol) for p, t in enumerate(toks)]
        errors = [off(g[0], w) for g, w in zip(got, want)]
        assert max(errors) < tol, errors
        assert all(g[1] == int(np.argmax(g[0])) for g in got)
        assert all((t[145:] == 0).all() for layer in held for t in layer)
        plan.kv_reset()
        again = [plan.forward_decode(t, p)[0] for p, t in enumerate(toks[:5])]
        assert all(np.array_equal(a, g[0]) for a, g in zip(again, got))
        plan.kv_reset()
        ids, _ = plan.decode_sequence(toks[:20], 20, 0)
        assert ids.tolist() == [g[1] for g in got[:20]]
        plan.kv_reset()
        for p, t in enumerate(toks[:6]):
            plan.forward_prefill(t, p)
        assert np.array_equal(plan.forward_decode(toks[6], 6)[0], got[6][0])
        assert plan.forward_decode_sample(toks[7], 7, 0.0, 0.9, 0.5) == got[7][1]
    finally:
        plan.free()


@pytest.mark.parametrize("shape,batch,n", [("tiny-llama", 64, 150), ("tiny-qwen3", 32, 77), ("tiny-phi3-gqa", 128, 129)])
def test_prompts_on_the_tensor_cores(pkg, make_model, shape, batch, n):
    """FP16 plans: chunks through the GEMMs, the cache and the chunk attention (and, for short last chunks, the form of single rows), then steps."""
    m = make_model(shape, pkg.gguf.GGMLType.F16, 300)
    plan, ref = pkg.B200MasterPlan.initialize_plan(m, prefill_batch_size=batch), Reference(pkg, m)
    c = m.configuration
    try:
        plan.set_kv_mode("q4")
        if plan.prefill_info()[0] != plan.PREFILL_TENSOR_CORE:
            pytest.skip("the shape has no tensor-core prefill")
        toks = tokens(c.vocab_size, n + 4)
        for at in range(0, n, batch):
            plan.forward_batch_prefill(toks[at:min(at + batch, n)], at)
        got = [plan.forward_decode(t, p)[0] for p, t in enumerate(toks[n:], n)]
        held = caches(plan, c)
        want = [ref.forward(t, p, row(held, p), FP16_TOL) for p, t in enumerate(toks)][n:]
        errors = [off(g, w) for g, w in zip(got, want)]
        assert max(errors) < FP16_TOL, errors
        plan.kv_reset()
        plan.set_prefill_mode("exact")  # token by token here
        plan.forward_batch_prefill(toks[:batch], 0)
        rows, _, why = plan.exact_prefill_info()
        assert rows == 0 and why
    finally:
        plan.free()


def test_q8_prompts(pkg, make_model):
    """A Q8_0 plan's chunks: token by token over the 4-bit cache (the exact prefill writes FP32 rows), and on the tensor cores where that is asked for."""
    m = make_model("tiny-llama", pkg.gguf.GGMLType.Q8_0, 200)
    plan = pkg.B200MasterPlan.initialize_plan(m, prefill_batch_size=64)
    try:
        plan.set_kv_mode("q4")
        assert plan.exact_prefill_info()[0] == 0
        toks = tokens(m.configuration.vocab_size, 70)
        steps = None
        for mode in ("exact", "tensor_core"):
            plan.kv_reset()
            ref = Reference(pkg, m)
            plan.set_prefill_mode(mode)
            plan.forward_batch_prefill(toks[:60], 0)
            plan.forward_batch_prefill(toks[60:69], 60)
            got = plan.forward_decode(toks[69], 69)[0]
            held = caches(plan, m.configuration)
            want = [ref.forward(t, p, row(held, p), Q8_TOL) for p, t in enumerate(toks)][-1]
            assert off(got, want) < Q8_TOL
            if mode == "exact":
                steps = got
                plan.kv_reset()
                for p, t in enumerate(toks):
                    last = plan.forward_decode(t, p)[0]
                assert np.array_equal(last, steps)
    finally:
        plan.free()


def test_refusals(pkg, make_model):
    m = make_model("tiny-llama", pkg.gguf.GGMLType.Q8_0, 64)
    plan = pkg.B200MasterPlan.initialize_plan(m)
    try:
        first = plan.forward_decode(5, 0)[0]
        with pytest.raises(pkg.native.B200Error):
            plan.set_kv_mode(7)
        plan.set_kv_mode("f32")
        assert np.array_equal(plan.forward_decode(5, 0)[0], first)
        plan.set_kv_mode("q4")
        for f in (lambda: plan.set_kv_mode("f32"), lambda: plan.set_decode_mode("persistent"), lambda: plan._native.trace_decode(1, 0), lambda: plan.trace_persistent(1, 0)):
            with pytest.raises(pkg.native.UnsupportedOperation):
                f()
        assert plan.decode_info()[0] == plan.DECODE_GRAPH
        for f in (lambda: plan.forward_decode(1, 64), lambda: plan.score_tokens([1, 2], 63), lambda: plan.score_tokens([1, 512], 0), lambda: plan.score_tokens([1], -1),
                  lambda: plan.score_tokens([1], 2**31 - 1)):
            with pytest.raises(pkg.native.B200Error):
                f()
        for f in (lambda: plan.score_tokens([1, 2], 0, top=33), lambda: plan.score_tokens([1, 2], 0, targets=[1])):
            with pytest.raises(ValueError):
                f()
    finally:
        plan.free()
    S = pkg.synth
    cfg, rows = P.configs(S)["loop_mid"]
    plan = make_plan(pkg, cfg, S.pibidra_weights(cfg, 13, bias_rows=rows), batch=8)
    try:
        with pytest.raises(pkg.native.UnsupportedOperation):
            plan.set_kv_mode("q4")
        with pytest.raises(pkg.native.UnsupportedOperation):
            plan.kv_info()
    finally:
        plan.free()


# ---- scoring --------------------------------------------------------------------------------------------------------------------------
def check_scores(scores, logits, targets, top):
    lp, h, ids, values = scores
    wl, wh, wi, wv = U.log_probs(torch.from_numpy(np.stack(logits)), torch.tensor(targets), top)
    assert (np.abs(lp - wl.numpy()) <= 2.0 ** -18 + 2.0 ** -22 * np.abs(wl.numpy())).all() and (np.abs(h - wh.numpy()) <= 2.0 ** -18 * (2 * wh.numpy() + 1)).all()
    assert np.array_equal(ids, wi.numpy()) and (np.abs(values - wv.numpy()) <= 2.0 ** -18 + 2.0 ** -22 * np.abs(wv.numpy())).all()


@pytest.mark.parametrize("mode", ["f32", "q4"])
def test_scores_of_a_gguf_plan(pkg, make_model, mode):
    m = make_model("tiny-qwen3", pkg.gguf.GGMLType.Q8_0, 200)
    V = m.configuration.vocab_size
    plan = pkg.B200MasterPlan.initialize_plan(m)
    try:
        plan.set_kv_mode(mode)
        toks = tokens(V, 140)
        logits = [plan.forward_decode(t, p)[0] for p, t in enumerate(toks)]
        plan.kv_reset()
        check_scores(plan.score_tokens(toks, 0, top=5), logits, toks[1:] + [-1], 5)
        plan.kv_reset()
        targets = tokens(V, 140, 9)
        targets[3] = -1
        first = plan.score_tokens(toks[:100], 0, targets=targets[:100])
        rest = plan.score_tokens(toks[100:], 100, targets=targets[100:], top=32)
        check_scores([np.concatenate(x) for x in zip(first[:2], rest[:2])] + [np.zeros((140, 0), np.int32), np.zeros((140, 0), np.float32)], logits, targets, 0)
        check_scores(rest, logits[100:], targets[100:], 32)
        plan.kv_reset()
        ppl = pkg.engine.perplexity(plan, toks)
        assert ppl == pytest.approx(float(np.exp(-np.mean([U.log_probs(torch.from_numpy(x[None]), torch.tensor([t]), 0)[0][0] for x, t in zip(logits, toks[1:])]))), rel=1e-4)
        assert plan.score_tokens([], 0)[0].shape == (0,)
        with pytest.raises(ValueError):
            pkg.engine.perplexity(plan, [1])
    finally:
        plan.free()


@pytest.mark.parametrize("compute", ["float32", "bfloat16"])
def test_scores_of_a_layered_plan(pkg, compute):
    """In chunks of the plan's capacity, equal to the log probabilities of the rows that the plan gives back."""
    S = pkg.synth
    cfg, rows = P.configs(S)["loop_mid"]
    plan = make_plan(pkg, cfg, S.pibidra_weights(cfg, 13, bias_rows=rows), batch=7, compute=compute)
    try:
        toks = tokens(cfg["vocab"], 31)
        scores = plan.score_tokens(toks, 0, top=3)
        plan.kv_reset()
        logits = []
        for at in range(0, 31, 7):
            part = toks[at:at + 7]
            logits += list(plan.forward_batch_logits(part, at, rows=range(len(part)))[0])
        check_scores(scores, logits, toks[1:] + [-1], 3)
    finally:
        plan.free()
