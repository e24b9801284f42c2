"""Plans are complete when the call that makes them returns, whatever the program has under way on the default stream.

A plan's stream does not wait for the default (legacy) stream.  Here that one is never idle while plans are created and switched and run their first prompts: zeros that a plan's creation
left to it would arrive late and clear tokens, activations or weights."""
import threading

import numpy as np
import pytest
import torch

import zulesun_util as Z
from test_gpu_zulesun import make_plan, prefill_all

pytestmark = pytest.mark.gpu


class BusyDefaultStream:
    """Short waits on the default stream, two of them under way at any time."""

    def __enter__(self):
        self.stop = threading.Event()
        self.thread = threading.Thread(target=self.run)
        torch.cuda._sleep(30_000_000)  # cycles: 15 ms
        self.thread.start()

    def run(self):
        events = []
        while not self.stop.is_set():
            torch.cuda._sleep(30_000_000)
            events.append(torch.cuda.Event())
            events[-1].record()
            if len(events) > 1:
                events.pop(0).synchronize()

    def __exit__(self, *what):
        self.stop.set()
        self.thread.join()
        torch.cuda.synchronize()


def gguf_rows(pkg, model, mode, toks):
    """Logits behind a prompt of two chunks, the first thing that the plan does in that mode, and of the steps after it."""
    plan = pkg.B200MasterPlan.initialize_plan(model, prefill_batch_size=64)
    try:
        if mode == "q4":
            plan.set_kv_mode("q4")
        if mode != "as created":
            plan.set_prefill_mode("tensor_core")
        plan.forward_batch_prefill(toks[:60], 0)
        plan.forward_batch_prefill(toks[60:69], 60)
        return np.stack([plan.forward_decode(t, p)[0] for p, t in enumerate(toks[69:], 69)])
    finally:
        plan.free()


@pytest.mark.parametrize("quant,mode", [("Q8_0", "tensor cores"), ("Q8_0", "q4"), ("Q8_0", "as created"), ("F16", "as created"), ("F16", "q4")])
def test_gguf_plans(pkg, make_model, quant, mode):
    m = make_model("tiny-llama", getattr(pkg.gguf.GGMLType, quant), 200)
    toks = np.random.default_rng(3).integers(0, m.configuration.vocab_size, 72).tolist()
    want = gguf_rows(pkg, m, mode, toks)
    with BusyDefaultStream():
        got = [gguf_rows(pkg, m, mode, toks) for _ in range(2)]
    assert all(np.array_equal(g, want) for g in got)


@pytest.mark.parametrize("name", ["tiles_a", "mixed"])
def test_layered_plans(pkg, name):
    """With a per-layer token input, whose gate is padded to whole tiles, and a scan's."""
    cfg = Z.configs(pkg.synth)[name]
    w = pkg.synth.zulesun_weights(cfg, 21)
    toks = np.random.default_rng(12).integers(0, cfg["vocab"], 100).tolist()

    def rows():
        plan = make_plan(pkg, cfg, w, ctx=128, batch=50, compute="bfloat16")
        try:
            return prefill_all(plan, toks, 50)
        finally:
            plan.free()

    want = rows()
    with BusyDefaultStream():
        got = [rows() for _ in range(2)]
    assert all(np.array_equal(g, want) for g in got)
