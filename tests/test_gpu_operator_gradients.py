"""The operators take no part in a graph of gradients, and say so."""
import pytest
import torch

from test_gpu_kv4 import filled, gen, ints, rand

pytestmark = pytest.mark.gpu


def test_tensors_that_require_gradients_are_refused(pkg):
    """No operator has a backward pass: a graph that ended in one would lose its gradients without a word."""
    cache, _, _, _ = filled(pkg, 1, 20, 2, 64, 1)
    k, q, pos, w = rand(gen(1), 3, 2, 64), rand(gen(2), 3, 4, 64), ints(0, 1, 2), torch.ones(64, device="cuda")
    x, t = rand(gen(3), 3, 50), ints(0, 1, 2)
    on = lambda y: y.clone().requires_grad_()  # noqa: E731
    calls = [lambda f: cache.append(f(k), k, pos), lambda f: cache.append(k, f(k), pos), lambda f: cache.append(k, k, pos, q=f(q)), lambda f: cache.append(k, k, pos, q=q, q_norm=f(w)),
             lambda f: cache.append(k, k, pos, k_norm=f(w)), lambda f: cache.attention(f(q), pos), lambda f: pkg.log_probs(f(x), t)]
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call(on)
        with torch.no_grad():
            call(on)
        with torch.inference_mode():
            call(on)
        call(lambda y: y)
