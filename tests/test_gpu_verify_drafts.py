"""The verification of drafted tokens on the GPU: equal to its definition in 64 bits, token for token."""
import math

import pytest
import torch

import paged_util as P

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def case(g, S, K, V, dtype, with_draft, pad=0, spread=2.0):
    """A target's logits (parts of padded rows), drafts sampled from something near them, uniform numbers, that something's logits."""
    x = (torch.randn(S, K + 1, V + pad, device="cuda", generator=g) * spread).to(dtype)[..., :V]
    y = (x[:, :K].float() + 0.5 * torch.randn(S, K, V, device="cuda", generator=g)).to(dtype)
    race = -torch.log(-torch.log(torch.rand(S, K, V, device="cuda", generator=g).clamp(1e-30, 1 - 1e-7)))
    drafts = (y.float() + race).argmax(-1).int() if K else torch.zeros(S, 0, device="cuda", dtype=torch.int32)
    return x, drafts, torch.rand(S, K + 1, device="cuda", generator=g), y if with_draft else None


def check(pkg, x, drafts, u, y, temperature=1.0):
    tokens, accepted = pkg.verify_drafts(x, drafts, u, draft_logits=y, temperature=temperature)
    want = P.verify(x, drafts, u, y, temperature)
    assert torch.equal(accepted.cpu(), want[1]), (accepted.tolist(), want[1].tolist())
    assert torch.equal(tokens.cpu(), want[0]), (tokens.tolist(), want[0].tolist())
    return tokens, accepted


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("with_draft,temperature", [(True, 1.0), (False, 1.0), (True, 0.6), (False, 1.7), (False, 0.0)])
@pytest.mark.parametrize("S,K,V,pad", [(1, 0, 1, 0), (3, 1, 2, 0), (5, 4, 7, 1), (16, 3, 999, 0), (9, 2, 8192, 8), (4, 5, 8193, 0), (2, 8, 50257, 47), (3, 1, 128256, 0), (70, 2, 33, 3), (2, 64, 300, 0)])
def test_equals_its_definition(pkg, dtype, with_draft, temperature, S, K, V, pad):
    g = gen(S + K + V)
    for spread in (0.3, 2.0, 6.0):
        x, drafts, u, y = case(g, S, K, V, dtype, with_draft, pad, spread)
        tokens, accepted = check(pkg, x, drafts, u, y, temperature)
        again = pkg.verify_drafts(x, drafts, u, draft_logits=y, temperature=temperature)
        assert torch.equal(tokens, again[0]) and torch.equal(accepted, again[1])


def test_fewer_drafts(pkg):
    """Negative tokens and those outside the vocabulary end a sequence's drafts, whatever stands behind them."""
    g = gen(1)
    x, drafts, u, y = case(g, 12, 5, 100, F32, True)
    for s in range(12):
        drafts[s, s % 6:] = torch.tensor([-1, 100, -2**31, 2**31 - 1, -7, 3], device="cuda", dtype=torch.int32)[s % 6] if s % 6 < 5 else 0
        drafts[s, s % 6 + 1:] = drafts[s, 0]
    u[:, :5] = 0  # whatever is drafted stands
    for d in (y, None):
        tokens, accepted = check(pkg, x, drafts, u, d)
        assert accepted.tolist() == [s % 6 for s in range(12)]


def test_borders_of_decisions(pkg):
    """u q against p where FP32 sums cannot tell them apart: equal numbers do not stand, one step less does."""
    V, K = 4096, 3
    x = torch.zeros(4, K + 1, V, device="cuda")
    drafts = torch.full((4, K), 17, device="cuda", dtype=torch.int32)
    u = torch.full((4, K + 1), 1 / V, device="cuda")
    below = math.nextafter(1, 0) and float(torch.nextafter(torch.tensor(1 / V), torch.tensor(0.0)))
    u[1, 0] = u[2, :2] = u[3, :3] = below
    tokens, accepted = check(pkg, x, drafts, u, None)
    assert accepted.tolist() == [0, 1, 2, 3]
    y = torch.zeros(4, K, V, device="cuda")
    y[..., V // 2:] = float("-inf")  # q = 2 / V: u = 0.5 is the border
    u = torch.full((4, K + 1), 0.5, device="cuda")
    u[1, 0] = u[2, :2] = u[3, :3] = float(torch.nextafter(torch.tensor(0.5), torch.tensor(0.0)))
    tokens, accepted = check(pkg, x, drafts, u, y)
    assert accepted.tolist() == [0, 1, 2, 3] and all(int(t[a]) >= V // 2 for t, a in list(zip(tokens, accepted.tolist()))[:3])  # what the draft left over


@pytest.mark.parametrize("u", [0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24])
def test_borders_of_tokens(pkg, u):
    x = torch.full((1, 1, 40000), float("-inf"), device="cuda")
    x[0, 0, [5, 9000, 9001, 39999]] = 0.0
    drafts = torch.zeros(1, 0, device="cuda", dtype=torch.int32)
    tokens, _ = check(pkg, x, drafts, torch.tensor([[u]], device="cuda"), None)
    assert tokens.item() == {0.0: 5, 0.25: 9000, 0.5: 9001, 0.75: 39999}.get(u, 39999)
    for bad in (1.0, 2.0, float("nan")):  # outside [0, 1): the last that weighs anything
        assert pkg.verify_drafts(x, drafts, torch.tensor([[bad]], device="cuda"))[0].item() == 39999


def test_masked_logits(pkg):
    g = gen(3)
    x, drafts, u, y = case(g, 20, 3, 500, F32, True)
    x[torch.rand(x.shape, device="cuda", generator=g) < 0.9] = float("-inf")
    x[:10][x[:10] == float("-inf")] = torch.finfo(F32).min
    x[..., 7] = 0.5
    y[:, :, 250:] = float("-inf")
    check(pkg, x, drafts, u, y)
    check(pkg, x, drafts, u, None)
    check(pkg, x, drafts, None, None, 0.0)
    only = torch.full((2, 2, 50), float("-inf"), device="cuda")
    only[:, :, 3] = 1.0
    three = torch.full((2, 1), 3, device="cuda", dtype=torch.int32)
    tokens, accepted = check(pkg, only, three, torch.tensor([[0.9, 0.1], [1.0, 0.9]], device="cuda"), None)  # u = 1 does not stand, and there is nothing but the draft
    assert accepted.tolist() == [1, 0] and tokens.tolist() == [[3, 3], [3, -1]]


def test_draft_that_its_model_cannot_have_made(pkg):
    """q = 0 at the draft: u q < p stands; where p is 0 as well nothing does, and the same distributions leave p."""
    x = torch.zeros(2, 2, 64, device="cuda")
    y = torch.zeros(2, 1, 64, device="cuda")
    y[:, :, 5] = x[1, :, 5] = float("-inf")
    drafts = torch.full((2, 1), 5, device="cuda", dtype=torch.int32)
    tokens, accepted = check(pkg, x, drafts, torch.tensor([[0.9, 0.5], [0.9, 0.5]], device="cuda"), y)
    assert accepted.tolist() == [1, 0] and tokens[1, 0] != 5


@pytest.mark.parametrize("u", [0.0, 0.3, 1 - 2.0 ** -24])
@pytest.mark.parametrize("V", [300, 40000])
def test_entries_that_weigh_the_same_are_not_drawn(pkg, V, u):
    """Two logits exchanged: the same sums, and all that is left over lies on one token, wherever the border falls."""
    g = gen(V)
    for low, high in ((V - 1, 0), (0, V - 1), (V // 2, V // 3), (5, 6)):
        x = torch.randn(1, 2, V, device="cuda", generator=g)
        x[0, 0, low], x[0, 0, high] = 1.0, 6.0
        y = x[:, :1].clone()
        y[0, 0, low], y[0, 0, high] = 6.0, 1.0
        tokens, accepted = pkg.verify_drafts(x, torch.tensor([[low]], device="cuda", dtype=torch.int32), torch.tensor([[0.9, u]], device="cuda"), draft_logits=y)
        assert accepted.item() == 0 and tokens.tolist() == [[high, -1]]


@pytest.mark.parametrize("bad", ["nan", "inf", "empty"])
@pytest.mark.parametrize("temperature", [1.0, 0.0])
def test_rows_without_a_distribution(pkg, bad, temperature):
    """They end a sequence where they are reached, and only there."""
    def spoil(row):
        if bad == "empty":
            row.fill_(float("-inf"))
        else:
            row[..., 9100] = float(bad)

    x, drafts, u, y = case(gen(2), 6, 3, 9500, F32, True)
    if temperature == 0:
        drafts = x[:, :3].argmax(-1).int()
    u[:, :3] = 0
    drafts[4, 1] = -1
    u[5, 0] = 1.0
    if temperature == 0:
        drafts[5, 0] = (drafts[5, 0] + 1) % 9500
    for s, i in ((0, 0), (1, 2), (2, 3), (4, 2), (5, 1)):
        spoil(x[s, i])
    for d in (y, None):
        tokens, accepted = check(pkg, x, drafts, u, d, temperature)
        assert accepted.tolist()[:5] == [0, 2, 3, 3, 1] and tokens[0].tolist() == [-1] * 4 and tokens[1, 2] == tokens[2, 3] == -1 and tokens[3, 3] >= 0 and tokens[4, 1] >= 0
    if temperature:
        x, drafts, u, y = case(gen(2), 2, 3, 9500, F32, True)
        u[:, :3] = 0
        spoil(y[0, 1])
        tokens, accepted = check(pkg, x, drafts, u, y)
        assert accepted.tolist() == [1, 3] and tokens[0, 1] == -1


def test_ties_go_to_the_first(pkg):
    x = torch.zeros(1, 2, 20000, device="cuda")
    x[0, :, [9000, 123, 17000]] = 4.0
    tokens, accepted = check(pkg, x, torch.tensor([[123]], device="cuda", dtype=torch.int32), None, None, 0.0)
    assert tokens.tolist() == [[123, 123]]
    assert pkg.verify_drafts(x, torch.tensor([[9000]], device="cuda", dtype=torch.int32), None, temperature=0.0)[0].tolist() == [[123, -1]]


@pytest.mark.parametrize("with_draft", [True, False])
def test_tokens_are_distributed_as_the_targets(pkg, with_draft):
    """65536 sequences of one draft: the first token's frequencies within 5 standard deviations of p, whatever the draft is."""
    g, S, V = gen(7), 65536, 6
    x = torch.randn(1, 2, V, device="cuda", generator=g).expand(S, 2, V)
    y = torch.randn(1, 1, V, device="cuda", generator=g)
    q = torch.softmax(y[0, 0], -1)
    drafts = torch.multinomial(q.expand(S, V), 1, generator=g).int() if with_draft else torch.full((S, 1), 2, device="cuda", dtype=torch.int32)
    tokens, accepted = pkg.verify_drafts(x, drafts, torch.rand(S, 2, device="cuda", generator=g), draft_logits=y.expand(S, 1, V) if with_draft else None)
    p = torch.softmax(x[0, 0].double(), -1)
    freq = torch.bincount(tokens[:, 0].long(), minlength=V).double() / S
    assert ((freq - p).abs() <= 5 * torch.sqrt(p * (1 - p) / S)).all()
    second = tokens[accepted == 1][:, 1].long()
    p = torch.softmax(x[0, 1].double(), -1)
    assert len(second) > 1000 and ((torch.bincount(second, minlength=V).double() / len(second) - p).abs() <= 5 * torch.sqrt(p * (1 - p) / len(second))).all()


def test_captured_and_on_streams(pkg):
    g = gen(4)
    sets = [case(g, 3, 4, 9000, F32, True) for _ in range(3)]
    want = [pkg.verify_drafts(x, d, u, draft_logits=y) for x, d, u, y in sets]
    x, d, u, y = (t.clone() for t in sets[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.verify_drafts(x, d, u, draft_logits=y)
    for s, w in zip(sets, want):
        for mine, new in zip((x, d, u, y), s):
            mine.copy_(new)
        graph.replay()
        assert torch.equal(out[0], w[0]) and torch.equal(out[1], w[1])
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    torch.cuda.synchronize()
    for _ in range(10):
        for st, (x, d, u, y), w in zip(streams, sets, want):
            with torch.cuda.stream(st):
                got.append((pkg.verify_drafts(x, d, u, draft_logits=y), w))
    torch.cuda.synchronize()
    assert all(torch.equal(o[0], w[0]) and torch.equal(o[1], w[1]) for o, w in got)


def test_refusals(pkg):
    x, d, u, y = case(gen(1), 2, 3, 50, F32, True)
    bad = [lambda: pkg.verify_drafts(x[0], d, u), lambda: pkg.verify_drafts(x, d.long(), u), lambda: pkg.verify_drafts(x, d[:1], u), lambda: pkg.verify_drafts(x, d, u.double()), lambda: pkg.verify_drafts(x, d, u[:, :3]),
           lambda: pkg.verify_drafts(x, d, None), lambda: pkg.verify_drafts(x, d, u, draft_logits=y.half()), lambda: pkg.verify_drafts(x, d, u, draft_logits=y[:, :2]), lambda: pkg.verify_drafts(x.double(), d, u),
           lambda: pkg.verify_drafts(x.transpose(1, 2), d, u), lambda: pkg.verify_drafts(x[:, :0], d, u), lambda: pkg.verify_drafts(x, d.cpu(), u), lambda: pkg.verify_drafts(x, d, u.cpu()),
           lambda: pkg.verify_drafts(x.clone().requires_grad_(), d, u), lambda: pkg.verify_drafts(x, d, u, draft_logits=y.clone().requires_grad_())]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    for t in (-1.0, float("nan"), 1e-9, 1e9):
        with pytest.raises(pkg.native.B200Error):
            pkg.verify_drafts(x, d, u, temperature=t)
    with pytest.raises(pkg.native.UnsupportedOperation):
        pkg.verify_drafts(x[:, :1].expand(2, 66, 50), d[:, :1].expand(2, 65).contiguous(), torch.zeros(2, 66, device="cuda"))
    none = pkg.verify_drafts(x[:0], d[:0], u[:0])
    assert none[0].shape == (0, 4) and none[1].shape == (0,)
