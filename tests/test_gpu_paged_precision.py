"""What the documentation says of FP32 results of paged attention: probabilities of 24 bits over BF16 pages, 22 over FP16, and sums that do not drift.  Inputs for which less shows.

The products' instructions add 16 positions each and may cut what they add, 2^-22 of their sum at most."""
import math

import pytest
import torch

from test_gpu_paged import BF16, F16, F32, gen, ints, paged

pytestmark = pytest.mark.gpu


def places(tables, n, page=16):
    at = torch.arange(n, device="cuda")
    return tables[0].long()[at // page], slice(None), at % page


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,hs,chunk", [(4, 32, 1), (4, 64, 1), (4, 128, 1), (12, 128, 1), (4, 256, 1), (4, 64, 4), (4, 128, 8), (4, 256, 4), (1, 96, 3)])
def test_probabilities_have_the_bits_they_should(pkg, dtype, heads, hs, chunk):
    """Three positions without a value whose score is the largest (each of a CTA's two warps meets one first), and 64 others whose probability p is (1 + 2^-9 + 2^-17) / 2 of its (FP16: (1 + 2^-11 + 2^-22) / 2): two
    numbers of BF16 hold it to 2^-17 of itself, 7.6e-6 (one of FP16 to 2^-12), and the results, c 64 p / (3 + 64 p), would be as far off, as the sum of the probabilities has them as they are.

    Bound, relative: 2^-24 (BF16 in three) or 2^-22 (FP16 in two) for p's parts; a tile's 32 positions are two instructions for each part, each cutting 2^-22 at most, 6 of them or 4; three tiles (five of 16 with heads of
    256) and the join: 8 roundings of 2^-24 of the results and 10 of the sum; p itself, 2^-21, counts by 3 / (3 + 64 p) < 2^-3.  2.7e-6, 2.4e-6."""
    n = 67
    cache, tables = paged(pkg, gen(1), [n], 16, 1, hs, dtype)
    k, v = torch.zeros(n, 1, hs, device="cuda"), (torch.arange(hs, device="cuda") % 16 + 16.0).expand(n, 1, hs).clone() / 16
    k[[0, 16, 32], 0, 0], v[[0, 16, 32]] = 1.0, 0.0
    cache.keys[places(tables, n)], cache.values[places(tables, n)] = k.to(dtype), v.to(dtype)
    q = torch.zeros(chunk, heads, hs, device="cuda", dtype=dtype)
    q[:, :, 0] = 1.0
    p = (1 + 2.0 ** -9 + 2.0 ** -17) / 2 if dtype == BF16 else (1 + 2.0 ** -11 + 2.0 ** -22) / 2
    got = cache.attention(q, ints(*[n - 1] * chunk), tables, scale=-math.log(p), chunk=chunk, dtype=F32).double().cpu()
    want = v[1, 0].double().cpu() * (64 * p / (3 + 64 * p))
    parts = 3 if dtype == BF16 else 2
    bound = (2.0 ** -24 if dtype == BF16 else 2.0 ** -22) + 2 * parts * 2.0 ** -22 + 18 * 2.0 ** -24 + 2.0 ** -24
    assert bound < 2.8e-6
    off = (got / want - 1).abs().max().item()
    assert off <= bound, off


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,chunk", [(4, 1), (4, 4), (4, 8)])
@pytest.mark.parametrize("shared", [True, False])
def test_long_sums_do_not_drift(pkg, dtype, heads, chunk, shared):
    """Values of one sign over 16384 positions of about the same probability: sums that the instructions cut, position by position, would drift one way (2^14 / 16 / 2 warps instructions for each of two or three
    parts, on average half of 2^-23 of half the sum: 3e-5, 4.6e-5).

    Bound, relative: the tiles' own sums, from zero, 6 instructions of 2^-22 at most, 1.4e-6; they are added as FP32 numbers are: 256 roundings of a warp, to nearest, each below 2^-24 of its sum, whose signs
    have no pattern: 6 standard deviations of 2^-24 / sqrt(3) sqrt(256), 3.3e-6; the probabilities' sum likewise, in 16 lanes of which each adds 1024: 6 of 2^-24 / sqrt(3) sqrt(1024 / 16), 1.7e-6; 2^-21 for the
    probabilities themselves, whose errors the division takes out, and the join."""
    g, n, hs = gen(2), 16384, 64
    cache, tables = paged(pkg, g, [n], 16, 1, hs, dtype)
    k = (torch.randn(n, 1, hs, device="cuda", generator=g) * 0.05).to(dtype)
    v = (torch.rand(n, 1, hs, device="cuda", generator=g) * 0.5 + 0.5).to(dtype)
    cache.keys[places(tables, n)], cache.values[places(tables, n)] = k, v
    q = torch.randn(chunk, heads, hs, device="cuda", generator=g).to(dtype)
    kw = {} if shared else {"max_len": 1}  # several CTAs share them, or one takes them all
    got = cache.attention(q, ints(*[n - 1] * chunk), tables, chunk=chunk, dtype=F32, **kw).double()
    w = torch.softmax(q.double().view(-1, hs) @ k[:, 0].double().T / 8, -1)
    want = (w @ v[:, 0].double()).view(chunk, heads, hs)
    bound = 6 * 2.0 ** -22 + 6 * 2.0 ** -24 / 3 ** 0.5 * (16 + 8) + 2.0 ** -21
    off = (got / want - 1).abs().max().item()
    assert off <= bound, off
