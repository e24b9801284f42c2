"""Positions whose end passes 32 bits are refused like others behind the context."""
import numpy as np
import pytest

import pibidra_util as P
from test_gpu_pibidra import make_plan

pytestmark = pytest.mark.gpu
FAR = [2**31 - 1, 2**31 - 2, 2**31 - 64, 200]


def refused(pkg, *calls):
    for call in calls:
        with pytest.raises(pkg.native.B200Error):
            call()


@pytest.mark.parametrize("quant", ["Q8_0", "F16"])
def test_gguf_plans(pkg, make_model, quant):
    m = make_model("tiny-llama", getattr(pkg.gguf.GGMLType, quant), 200)
    plan = pkg.B200MasterPlan.initialize_plan(m, prefill_batch_size=64)
    try:
        want = plan.forward_decode(5, 0)[0]
        for at in FAR:
            refused(pkg, lambda: plan.forward_batch_prefill([1, 2], at), lambda: plan.decode_sequence([1, 2], 2, at), lambda: plan.decode_sequence([1], 64, at, True),
                    lambda: plan.score_tokens([1, 2], at), lambda: plan.forward_decode(1, at))
        plan.kv_reset()
        assert np.array_equal(plan.forward_decode(5, 0)[0], want)
    finally:
        plan.free()


def test_layered_plans(pkg):
    S = pkg.synth
    cfg, rows = P.configs(S)["loop_mid"]
    plan = make_plan(pkg, cfg, S.pibidra_weights(cfg, 13, bias_rows=rows), batch=8)
    try:
        for at in [*FAR[:3], 10**6]:
            refused(pkg, lambda: plan.forward_batch_logits([1, 2], at, rows=[0]), lambda: plan.forward_batch_prefill([1, 2], at), lambda: plan.score_tokens([1, 2], at))
    finally:
        plan.free()
