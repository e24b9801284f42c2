"""The operators together: sequences of a small model decode with drafted tokens over shared pages, and come out as they do token by token."""
import pytest
import torch

import kv4_util as U

pytestmark = pytest.mark.gpu


class Model:
    """Two layers of attention over pages and a classifier, random weights."""

    def __init__(self, pkg, pages, page, seed=3, H=8, G=2, hs=64, V=400):
        g = torch.Generator(device="cuda").manual_seed(seed)
        w = lambda *s: torch.randn(s, device="cuda", generator=g) / s[0] ** 0.5  # noqa: E731
        self.H, self.G, self.hs, self.dim = H, G, hs, H * hs
        self.embed, self.head = torch.randn(V, self.dim, device="cuda", generator=g), 4 * w(self.dim, V)
        self.qkv, self.out = [w(self.dim, (H + 2 * G) * hs) for _ in range(2)], [w(self.dim, self.dim) for _ in range(2)]
        self.norms = [1 + 0.1 * torch.randn(hs, device="cuda", generator=g) for _ in range(4)]
        self.caches = [pkg.PagedKVCache(pages, page, G, hs, dtype=torch.float16) for _ in range(2)]
        self.cos, self.sin = (t.cuda() for t in U.tables(512, hs))

    def __call__(self, tokens, positions, sequences, tables, chunk):
        x, n, H, G = self.embed[tokens.long()], len(tokens), self.H, self.G
        for l, cache in enumerate(self.caches):
            y = x @ self.qkv[l] / x.square().mean(-1, keepdim=True).sqrt()
            q, k, v = y.view(n, H + 2 * G, self.hs).split((H, G, G), 1)
            q = cache.append(k, v, positions, tables, sequences=sequences, q=q, q_norm=self.norms[2 * l], k_norm=self.norms[2 * l + 1], cos=self.cos, sin=self.sin)
            x = x + cache.attention(q, positions, tables, sequences=sequences, chunk=chunk, dtype=torch.float32).view(n, -1) @ self.out[l]
        return x @ self.head / x.square().mean(-1, keepdim=True).sqrt()


def decode(pkg, prompts, steps, drafted, seed=5):
    """Greedy tokens of every prompt; with ``drafted`` > 0 that many are guessed a step, some rightly, and verified."""
    S, page = len(prompts), 16
    model = Model(pkg, S * 16, page)
    tables = torch.randperm(S * 16, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).int().view(S, 16)
    told = [list(p) for p in prompts]
    for s, p in enumerate(prompts):  # the prompt but its last token, as one chunk
        at = torch.arange(len(p) - 1, device="cuda", dtype=torch.int32)
        model(torch.tensor(p[:-1], device="cuda"), at, torch.full_like(at, s), tables, len(p) - 1)
    counts = []
    guess = torch.Generator().manual_seed(seed)
    truth = decode.truth
    while min(len(t) - len(p) for t, p in zip(told, prompts)) < steps:
        rows, pos = [], []
        drafts = torch.full((S, drafted), -1, dtype=torch.int32)
        for s in range(S):
            done = len(told[s]) - len(prompts[s])
            for i in range(drafted):  # what will be said, with a mistake now and then
                if done + i < steps:
                    drafts[s, i] = truth[s][done + i] if torch.rand((), generator=guess) < 0.8 else (truth[s][done + i] + 1) % 400
            rows += [told[s][-1]] + drafts[s].clamp(min=0).tolist()
            pos += [len(told[s]) - 1 + i for i in range(drafted + 1)]
        seq = torch.arange(S, device="cuda", dtype=torch.int32).repeat_interleave(drafted + 1)
        logits = model(torch.tensor(rows, device="cuda"), torch.tensor(pos, device="cuda", dtype=torch.int32), seq, tables, drafted + 1)
        tokens, accepted = pkg.verify_drafts(logits.view(S, drafted + 1, -1), drafts.cuda(), None, temperature=0.0)
        for s, (t, a) in enumerate(zip(tokens.tolist(), accepted.tolist())):
            told[s] += t[:a + 1]
            counts.append(a)
    return [t[len(p):len(p) + steps] for t, p in zip(told, prompts)], counts


def test_drafted_tokens_change_nothing(pkg):
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 400, (n,), generator=g).tolist() for n in (5, 40, 17, 100)]
    decode.truth = None
    decode.truth, none = decode(pkg, prompts, 30, 0)
    assert set(none) == {0} and len({tuple(t) for t in decode.truth}) == 4
    for drafted in (1, 3, 6):
        told, counts = decode(pkg, prompts, 30, drafted)
        assert told == decode.truth
        assert 0 < sum(counts) / len(counts) < drafted  # some stand and some do not (0.8 + .. + 0.8^6 = 2.95 of 6 would, but sequences that are done count as none until the last one is)
