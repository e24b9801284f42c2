"""Q8_0 plans over a 4-bit cache at contexts where a step's attention is cut over whole clusters: results in blocks of 32 quants, heads of 96 among them."""
import pytest

from test_gpu_kv4_plan import Q8_TOL, Reference, caches, off, row, tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,context", [("tiny-phi3", 2048), ("tiny-phi3", 4096), ("tiny-phi3", 8000), ("tiny-phi3-gqa", 4096), ("tiny-llama", 4096)])
def test_deep_steps_of_q8_plans(pkg, make_model, shape, context):
    """Steps in front of and behind the position from which the graph for the whole context takes over."""
    m = make_model(shape, pkg.gguf.GGMLType.Q8_0, context)
    plan, ref = pkg.B200MasterPlan.initialize_plan(m), Reference(pkg, m)
    c = m.configuration
    try:
        plan.set_kv_mode("q4")
        toks = tokens(c.vocab_size, 140)
        got = [plan.forward_decode(t, p)[0] for p, t in enumerate(toks)]
        held = caches(plan, c)
        want = [ref.forward(t, p, row(held, p), Q8_TOL) for p, t in enumerate(toks)]
        errors = [off(g, w) for g, w in zip(got, want)]
        assert max(errors) < Q8_TOL, errors
    finally:
        plan.free()
