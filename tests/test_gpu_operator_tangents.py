"""The operators on torch tensors have no forward-mode derivatives either: a tensor that carries a tangent is refused, not answered without it."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def test_tangents_are_refused(pkg):
    ones = lambda *s, dtype=torch.bfloat16: torch.ones(s, device="cuda", dtype=dtype)  # noqa: E731
    k, q, x, norm, cos = ones(3, 2, 64), ones(3, 4, 64), ones(1, 2, 8, dtype=torch.float32), ones(64, dtype=torch.float32), ones(20, 32, dtype=torch.float32)
    pos, table, drafts, u = torch.arange(3, device="cuda", dtype=torch.int32), torch.zeros(1, 1, device="cuda", dtype=torch.int32), torch.zeros(1, 1, device="cuda", dtype=torch.int32), ones(1, 2, dtype=torch.float32) / 2
    cache, small = pkg.PagedKVCache(2, 16, 2, 64), pkg.KV4Cache(1, 16, 2, 64)
    with forward_ad.dual_level():
        on = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        bad = [lambda: cache.append(on(k), k, pos, table), lambda: cache.append(k, on(k), pos, table), lambda: cache.append(k, k, pos, table, q=on(q)), lambda: cache.append(k, k, pos, table, k_norm=on(norm)),
               lambda: cache.append(k, k, pos, table, cos=on(cos), sin=cos), lambda: cache.append(k, k, pos, table, cos=cos, sin=on(cos)), lambda: cache.attention(on(q), pos, table),
               lambda: cache.attention(on(q)[:2], pos[:2], table), lambda: cache.attention(q, pos, table, out=on(q.clone())), lambda: pkg.verify_drafts(on(x), drafts, u), lambda: pkg.verify_drafts(x, drafts, on(u)),
               lambda: pkg.verify_drafts(x, drafts, u, draft_logits=on(x[:, :1].clone())), lambda: small.append(on(k), k, pos), lambda: small.append(k, on(k), pos), lambda: small.attention(on(q.float()), pos),
               lambda: pkg.log_probs(on(x[0]), None)]
        for i, call in enumerate(bad):
            with pytest.raises(ValueError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                call()
        cache.append(on(k).detach(), k, pos, table)
        cache.attention(forward_ad.unpack_dual(on(q)).primal.detach(), pos, table)
        pkg.verify_drafts(on(x).detach(), drafts, u)
