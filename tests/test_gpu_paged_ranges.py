"""The paged cache and its attention on the GPU where inputs are unusual: what padding holds, scores of any size, precision of long rows, overlapping results."""
import pytest
import torch

import paged_util as P
from test_gpu_paged import BF16, F16, F32, check, gen, ints, paged, probability, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,out", [(BF16, F32), (F16, F32), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("H,hs,slots,used", [(8, 64, 5, 3), (8, 128, 5, 3), (6, 32, 4, 1), (2, 256, 6, 5), (24, 96, 2, 1), (8, 64, 40, 17)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_padding_holds_does_not_matter(pkg, dtype, out, H, hs, slots, used, bad):
    """Draft slots that are not used (no sequence, or a position behind the table) and rows at negative positions: the other rows have the same bits whatever lies in their queries."""
    g = gen(hs + slots)
    cache, tables = paged(pkg, g, [320, 300, 310], 16, 2, hs, dtype)
    pos = torch.cat([torch.arange(n - used, n - used + slots, device="cuda") for n in (320, 300, 310)]).int()
    seq = torch.arange(3, device="cuda", dtype=torch.int32).repeat_interleave(slots)
    live = (torch.arange(slots, device="cuda") < used).repeat(3)
    kind = torch.arange(3 * slots, device="cuda") % 3
    seq[~live & (kind == 0)] = -1
    pos[~live & (kind == 1)] = 10**6
    pos[~live & (kind == 2)] = -1
    q = rand(g, 3 * slots, H, hs, dtype=dtype)
    q[~live] = 0
    want = check(cache, q, pos, tables, seq, out, chunk=slots)
    q[~live] = bad
    got = cache.attention(q, pos, tables, sequences=seq, dtype=out, chunk=slots)
    assert torch.equal(got[live], want[live]) and (got[~live & (kind == 2)] == 0).all()


@pytest.mark.parametrize("dtype,out", [(BF16, F32), (F16, F32), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("size", [1e5, 1.5e6, 9e6, 3e7, 7e7, 2e8, 9e8, 1.1e9, 7e9, 1.3e11, 2.9e13, 1e20, 1e30])
@pytest.mark.parametrize("chunk,hs", [(1, 64), (1, 256), (4, 64), (4, 128), (40, 64)])
def test_huge_scores(pkg, dtype, out, size, chunk, hs):
    """Scores (times log2(e)) of up to 1e30, whose rounding alone is many powers of two.  Equal ones share a row out evenly, and one that is larger by 2^-7 of itself, 2^-7 size > 780 powers of two,
    takes it alone.  The probabilities of equal scores are equal, so a mean's error is that of sums (m products of 16 an instruction, (m / 8 + 32) 2^-22), 2^-17 for the parts of a probability, its half
    step with 16-bit results, all of the mean of |v|, and the result's half step."""
    g, n = gen(hs + chunk), 500
    cache, tables = paged(pkg, g, [n], 16, 1, hs, dtype)
    at = torch.arange(n, device="cuda")
    where = tables[0].long()[at // 16], 0, at % 16
    pos = torch.arange(n - 40, n, device="cuda", dtype=torch.int32)
    q = torch.full((40, 4, hs), 8.0, device="cuda", dtype=dtype)
    scale = size * 0.6931471805599453 / (hs * 64.0)
    values = cache.values[where].double().cpu()
    off = (n / 8 + 32) * 2.0 ** -22 + 2.0 ** -17 + probability(cache, out)
    for factor in (1.0, 0.83, 0.71):  # references that round up and down
        cache.keys[where] = torch.full((n, hs), 8.0, device="cuda", dtype=dtype)
        got = cache.attention(q, pos, tables, scale=scale * factor, chunk=chunk, dtype=out).double().cpu()
        for i in range(40):
            v = values[:n - 39 + i]
            bound = P.rounding(v.mean(0), off * v.abs().mean(0), out)
            assert ((got[i] - v.mean(0)).abs() <= bound).all()
        best = int(torch.randint(0, n - 40, (), device="cuda", generator=g))
        cache.keys[tables[0, best // 16], 0, best % 16] = 8.0625
        got = cache.attention(q, pos, tables, scale=scale * factor, chunk=chunk, dtype=out).double().cpu()
        assert ((got - values[best]).abs() <= P.rounding(values[best], off * values[best].abs(), out)).all()
        grown = 8.0 + 0.0625 * (torch.arange(n, device="cuda") // 50)  # a maximum that grows every 50 positions, the last row's on 50 or fewer
        cache.keys[where] = grown[:, None].expand(n, hs).to(dtype)
        got = cache.attention(q, pos, tables, scale=scale * factor, chunk=chunk, dtype=out).double().cpu()
        for i in range(40):
            v = values[450:n - 39 + i]
            bound = P.rounding(v.mean(0), off * v.abs().mean(0), out)
            assert ((got[i] - v.mean(0)).abs() <= bound).all()


@pytest.mark.parametrize("chunk,hs", [(1, 64), (3, 64), (40, 64), (40, 128), (40, 32)])
def test_results_in_the_place_of_queries_or_beside_them(pkg, chunk, hs):
    """``out`` may be the queries themselves, or another part of the same wider rows; what overlaps otherwise is refused."""
    g = gen(chunk)
    cache, tables = paged(pkg, g, [90, 3000], 16, 2, hs, BF16)
    pos = torch.cat([torch.arange(50, 90, device="cuda"), torch.arange(2960, 3000, device="cuda")]).int()
    seq = torch.arange(2, device="cuda", dtype=torch.int32).repeat_interleave(40)
    wide = rand(g, 80, 3 * 8 * hs, dtype=BF16)
    q, beside, across = (wide[:, i:i + 8 * hs].view(80, 8, hs) for i in (8 * hs, 16 * hs, 12 * hs))
    want = cache.attention(q, pos, tables, sequences=seq, chunk=chunk)
    cache.attention(q, pos, tables, sequences=seq, chunk=chunk, out=beside)
    assert torch.equal(beside, want)
    with pytest.raises(pkg.native.B200Error, match="overlap"):
        cache.attention(q, pos, tables, sequences=seq, chunk=chunk, out=across)
    cache.attention(q, pos, tables, sequences=seq, chunk=chunk, out=q)
    assert torch.equal(q, want)
    k, v = wide[:, :2 * hs].view(80, 2, hs), wide[:, 2 * hs:4 * hs].view(80, 2, hs)
    turned = cache.append(k, v, pos, tables, sequences=seq, q=q, q_out=beside)
    assert turned.data_ptr() == beside.data_ptr() and torch.equal(beside, q)
    for bad in (across, wide[:, :8 * hs].view(80, 8, hs), cache.keys.view(-1)[:80 * 8 * hs].view(80, 8, hs)):
        with pytest.raises(pkg.native.B200Error, match="overlap"):
            cache.append(k, v, pos, tables, sequences=seq, q=q, q_out=bad)


def test_memory_that_is_taken_away_or_moves(pkg):
    """``keys`` and ``values`` are the caller's too: a call without their memory is refused, and one after they have moved uses them where they are."""
    g = gen(2)
    cache, tables = paged(pkg, g, [70], 16, 2, 64, BF16)
    q, pos, k = rand(g, 3, 8, 64, dtype=BF16), ints(67, 68, 69), rand(g, 3, 2, 64, dtype=BF16)
    cache.append(k, k, pos, tables)
    want, keys = cache.attention(q, pos, tables), cache.keys.clone()
    bytes_ = cache.keys.untyped_storage().nbytes()
    torch.cuda.synchronize()
    for t in (cache.keys, cache.values):
        kept = t.clone()
        t.untyped_storage().resize_(0)
        with pytest.raises(ValueError, match="taken away"):
            cache.attention(q, pos, tables)
        with pytest.raises(ValueError, match="taken away"):
            cache.append(k, k, pos, tables)
        filler = torch.empty(bytes_ // 2, device="cuda", dtype=BF16)  # another tenant of what was freed
        t.untyped_storage().resize_(bytes_)
        t.copy_(kept)
        del filler
    assert torch.equal(cache.attention(q, pos, tables), want) and torch.equal(cache.keys.view(torch.int16), keys.view(torch.int16))
    cache.keys.requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        cache.append(k, k, pos, tables)
    cache.keys.requires_grad_(False)
    cache.keys.transpose_(1, 2)
    with pytest.raises(ValueError, match="shape"):
        cache.attention(q, pos, tables)
    cache.keys.transpose_(1, 2)
    assert torch.equal(cache.attention(q, pos, tables), want)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("out", [F32, None])
@pytest.mark.parametrize("size", [3e6, 7e7, 1.1e9, 1.3e11, 1e25])
@pytest.mark.parametrize("chunk,hs", [(1, 64), (5, 128), (33, 64)])
def test_huge_scores_of_rows_that_are_shared(pkg, dtype, out, size, chunk, hs):
    """As above over 9000 positions, whose parts are joined: equal scores, a single larger one, and a maximum that grows every 1000 positions.  Sums: (m / 8 + 32) 2^-22 and the parts' join."""
    g, n, out = gen(hs + chunk), 9000, out or dtype
    cache, tables = paged(pkg, g, [n], 16, 1, hs, dtype)
    at = torch.arange(n, device="cuda")
    where = tables[0].long()[at // 16], 0, at % 16
    pos = torch.arange(n - chunk, n, device="cuda", dtype=torch.int32)
    q = torch.full((chunk, 4, hs), 8.0, device="cuda", dtype=dtype)
    values = cache.values[where].double().cpu()
    off = (n / 8 + 32) * 2.0 ** -22 + 2.0 ** -17 + probability(cache, out)
    for factor in (1.0, 0.83, 0.71):
        scale = factor * size * 0.6931471805599453 / (hs * 64.0)
        for keys, first in ((torch.full((n,), 8.0, device="cuda"), 0), (8.0 + 0.0625 * (at // 1000), 8000), (torch.where(at == 4321, 8.0625, 8.0), None)):
            cache.keys[where] = keys[:, None].expand(n, hs).to(dtype)
            got = cache.attention(q, pos, tables, scale=scale, chunk=chunk, dtype=out).double().cpu()
            for i in range(chunk):
                v = values[4321:4322] if first is None else values[first:n - chunk + 1 + i]
                assert ((got[i] - v.mean(0)).abs() <= P.rounding(v.mean(0), off * v.abs().mean(0), out)).all()
