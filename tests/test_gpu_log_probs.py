"""Log probabilities of given tokens, entropy and alternatives on the GPU against the plain 64-bit form."""
import math

import pytest
import torch

import kv4_util as U

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def check(pkg, x, targets, top):
    """exp of a difference y has a relative error of at most 2^-24 |y| 1.45 + 2^-21, terms with |y| > 30 do not count (e^-30 of the sum): 2^-18 of every term, so of the sum too
    (its additions in FP32 included); a log probability then is off by that and by the roundings of x - M and the difference (2^-23 of the values), an entropy by
    2^-18 (1 + the largest |y| that counts) in the worst case: both sums have that relative error."""
    lp, h, ids, values = pkg.log_probs(x, targets, top)
    wl, wh, wi, wv = U.log_probs(x, targets, top)
    assert lp.dtype == h.dtype == values.dtype == F32 and ids.dtype == torch.int32
    assert ((lp.double().cpu() - wl).abs() <= 2.0 ** -18 + 2.0 ** -22 * wl.abs()).all()
    assert ((h.double().cpu() - wh).abs() <= 2.0 ** -18 * (2 * wh + 1)).all()
    assert torch.equal(ids.cpu(), wi)
    assert ((values.double().cpu() - wv).abs() <= 2.0 ** -18 + 2.0 ** -22 * wv.abs()).all()


@pytest.mark.parametrize("rows,vocab,top,pad,skip", [(1, 1, 1, 0, 0), (3, 7, 7, 0, 0), (2, 33, 32, 0, 1), (5, 1000, 20, 3, 0), (2, 8191, 5, 0, 0), (2, 8193, 1, 0, 3), (1, 32064, 20, 0, 0),
                                                     (40, 50257, 5, 0, 0), (3, 128256, 32, 64, 7), (1, 151936, 20, 0, 0), (2, 300007, 8, 1, 1), (700, 2049, 3, 0, 0), (64, 128256, 0, 0, 0)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rows(pkg, rows, vocab, top, pad, skip, dtype):
    g = torch.Generator(device="cuda").manual_seed(vocab + rows)
    x = (torch.randn(rows, vocab + pad + skip, device="cuda", generator=g) * 3).to(dtype)[:, skip:skip + vocab]  # rows that begin anywhere
    targets = torch.randint(0, vocab, (rows,), device="cuda", generator=g).int()
    targets[0] = int(x[0].float().argmax())
    check(pkg, x, targets, top)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_orders_and_ties(pkg, dtype):
    """Rising, falling and constant rows (every batch, or none, brings better ones; equal ones go by index), few different values, and one block of large ones."""
    n = 40000
    up = torch.arange(n, device="cuda").float() / 1000
    x = torch.stack((up, up.flip(0), torch.zeros(n, device="cuda"), (torch.arange(n, device="cuda") * 7919 % 13).float(), torch.where((up > 20) & (up < 20.3), 5.0, -5.0),
                     torch.where(torch.arange(n, device="cuda") % 512 == 3, 4.0, 0.0), -0.0 * (torch.arange(n, device="cuda") % 2).float())).to(dtype)
    check(pkg, x, torch.arange(7, device="cuda").int() * 1000, 32)


def test_sure_rows_keep_their_small_numbers(pkg):
    """log p of the token that has nearly everything is -(the others' share), far below FP32's step at 1."""
    x = torch.full((3, 5000), -40.0, device="cuda")
    x[:, 77] = torch.tensor([0.0, -5.0, 3.0], device="cuda")
    lp, h, _, _ = pkg.log_probs(x, torch.tensor([77] * 3, device="cuda").int(), 1)
    y = -40.0 - torch.tensor([0.0, -5.0, 3.0], dtype=torch.float64)
    z = 4999 * torch.exp(y)  # (a softmax in 64 bits starts at 1 too and holds two digits of these)
    wl, wh = -torch.log1p(z), torch.log1p(z) - y * z / (1 + z)
    assert ((lp.double().cpu() / wl - 1).abs() < 2.0 ** -15).all() and ((h.double().cpu() / wh - 1).abs() < 2.0 ** -15).all()  # |y| up to 43: 2^-24 * 43 * 1.45 + sums


def test_masked_infinite_and_missing(pkg):
    inf, nan = math.inf, math.nan
    x = torch.randn(8, 9000, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    x[0, 100:] = -inf  # most are masked
    x[1] = -inf
    x[1, 5] = 2.0  # one is left: log p = 0, entropy 0
    x[2] = -inf  # none
    x[3, 8999] = nan
    x[4, 17] = inf
    x[5] = nan
    x[5, 3], x[5, 4444] = 1.0, 2.0
    t = torch.tensor([3, 5, 1, 4, 17, 3, -1, 9000], device="cuda").int()
    lp, h, ids, values = pkg.log_probs(x, t, 4)
    wl, wh, wi, wv = U.log_probs(x[[0, 1, 6, 7]], t[[0, 1, 6, 7]], 4)
    got = [a[[0, 1, 6, 7]].double().cpu() for a in (lp, h, values)]
    assert ((got[0] - wl).abs() <= 2.0 ** -17).all() and ((got[1] - wh).abs() <= 2.0 ** -14).all() and torch.equal(ids[[0, 1, 6, 7]].cpu(), wi)
    assert torch.equal(torch.isinf(got[2]), torch.isinf(wv)) and ((got[2] - wv).abs()[torch.isfinite(wv)] <= 2.0 ** -17).all()
    assert lp[6] == 0 and lp[7] == 0 and lp[1] == 0 and h[1] == 0
    assert ids[1].tolist() == [5, 0, 1, 2] and ids[2].tolist() == [0, 1, 2, 3]
    for r in (2, 3, 4, 5):
        assert torch.isnan(lp[r]) and torch.isnan(h[r]) and torch.isnan(values[r]).all()
    assert ids[4, 0] == 17 and ids[5].tolist() == [4444, 3, -1, -1] and (ids[3] >= 0).all()


def test_no_targets_no_rows_and_refusals(pkg):
    x = torch.randn(4, 100, device="cuda")
    lp, h, ids, values = pkg.log_probs(x, None)
    assert (lp == 0).all() and ids.shape == (4, 0) and values.shape == (4, 0) and (h > 0).all()
    assert pkg.log_probs(x[:0], None, 3)[2].shape == (0, 3)
    t = torch.zeros(4, device="cuda").int()
    for f in (lambda: pkg.log_probs(x, t, 33), lambda: pkg.log_probs(x, t, -1), lambda: pkg.log_probs(x[:, :5], t, 6), lambda: pkg.log_probs(x, t[:3]), lambda: pkg.log_probs(x, t.long()),
              lambda: pkg.log_probs(x, t.cpu()), lambda: pkg.log_probs(x.t(), t), lambda: pkg.log_probs(x.double(), t), lambda: pkg.log_probs(x[0], t), lambda: pkg.log_probs(x[:, :0], t)):
        with pytest.raises(ValueError):
            f()


def test_captured_and_on_two_streams(pkg):
    g = torch.Generator(device="cuda").manual_seed(5)
    x, t = torch.randn(6, 30000, device="cuda", generator=g), torch.arange(6, device="cuda").int()
    pkg.log_probs(x, t, 5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = pkg.log_probs(x, t, 5)
    for _ in range(3):
        x.copy_(torch.randn(6, 30000, device="cuda", generator=g))
        graph.replay()
        for a, b in zip(outs, pkg.log_probs(x, t, 5)):
            assert torch.equal(a, b)
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for s in streams:
        with torch.cuda.stream(s):
            got.append([pkg.log_probs(x, t, 5) for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for side in got for out in side for a, b in zip(out, got[0][0]))
