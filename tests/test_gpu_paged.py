"""The paged 16-bit key/value cache and its attention on the GPU against their plain 64-bit forms."""
import ctypes as C

import pytest
import torch

import kv4_util as U
import paged_util as P

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=F32):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def ints(*v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


def paged(pkg, g, lengths, page, G, hs, dtype, gain=1.0):
    """(cache, tables): sequences of given lengths on pages in any order; whatever holds no position of theirs is NaN."""
    width = max(1, -(-max(lengths) // page))
    need = [-(-n // page) for n in lengths]
    cache = pkg.PagedKVCache(sum(need) + 3, page, G, hs, dtype=dtype)
    cache.keys.fill_(float("nan"))
    cache.values.fill_(float("nan"))
    order = torch.randperm(sum(need) + 3, device="cuda", generator=g).int()
    tables = torch.full((len(lengths), width), -1, device="cuda", dtype=torch.int32)
    used = 0
    for s, n in enumerate(lengths):
        tables[s, :need[s]] = order[used:used + need[s]]
        used += need[s]
        at = torch.arange(n, device="cuda")
        where = tables[s].long()[at // page], slice(None), at % page
        cache.keys[where] = rand(g, n, G, hs, dtype=dtype) * gain
        cache.values[where] = rand(g, n, G, hs, dtype=dtype) * 0.5
    return cache, tables


def probability(cache, dtype):
    """What the documentation says: with 16-bit results a probability is one number of the cache's type, half a step off."""
    return 0.0 if dtype == F32 else U.half_step(cache.keys.dtype)


def check(cache, q, positions, tables, sequences=None, dtype=None, **kw):
    got = cache.attention(q, positions, tables, sequences=sequences, dtype=dtype, **kw)
    want, bound = P.attention(q, cache.keys, cache.values, positions, sequences, tables, kw.get("scale"), kw.get("window", 0), got.dtype, probability(cache, got.dtype))
    written = positions.cpu() < tables.shape[1] * cache.page_size
    if sequences is not None:
        written &= (sequences.cpu() >= 0) & (sequences.cpu() < tables.shape[0])  # (padding's rows are not)
    off = (got.double().cpu() - want).abs()[written]
    assert (off <= bound[written]).all(), f"off by up to {float((off / bound[written]).max())} of the bound"
    return got


# ---- append -----------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("H,G,hs,turned", [(4, 2, 32, 32), (4, 2, 32, 8), (8, 8, 64, 64), (6, 2, 96, 96), (6, 2, 96, 24), (5, 1, 128, 128), (5, 1, 128, 32), (3, 3, 256, 256), (3, 3, 256, 2), (2, 1, 64, 38)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("norm,dtype,pad,cache_type", [(True, F32, 0, BF16), (False, F32, 1, F16), (True, BF16, 3, BF16), (False, F16, 8, F16), (True, F16, 0, BF16)])
def test_append_norms_rotates_and_stores(pkg, H, G, hs, turned, layout, norm, dtype, pad, cache_type):
    """Norm: 3 roundings (s, s x, w s x), rotation: products and sum, 3 of at most |a| + |b|: 8 half steps of FP32 at the largest entry; then the cache's half step."""
    g, n, page = gen(H * hs + pad + turned), 33, 8
    cache, tables = paged(pkg, g, [24, 9, 31], page, G, hs, cache_type)
    before = cache.keys.clone(), cache.values.clone()
    wide = rand(g, n, (H + 2 * G) * hs + pad, dtype=dtype) * 2  # parts of a padded row, unaligned where pad is odd
    q, k, v = (wide[:, a * hs + pad:b * hs + pad].view(n, b - a, hs) for a, b in ((0, H), (H, H + G), (H + G, H + 2 * G)))
    cos, sin = (t[:, :turned // 2].contiguous().cuda() for t in U.tables(40, hs))
    qn, kn = (1 + 0.3 * rand(g, hs), 1 + 0.3 * rand(g, hs)) if norm else (None, None)
    places = torch.randperm(3 * 24, generator=g, device="cuda")[:n].int()  # any order; those of sequence 1 behind its two pages have none
    seq, pos = places // 24, places % 24
    got = cache.append(k, v, pos, tables, sequences=seq, q=q, q_norm=qn, k_norm=kn, eps=1e-5, cos=cos, sin=sin, layout=layout)
    assert got.dtype == cache_type
    page_of = tables.cpu()[seq.cpu().long(), pos.cpu().long() // page].long()
    stored = page_of >= 0
    assert 0 < stored.sum() < n

    def close(got, x, weight):
        want = P.turn(x, weight, 1e-5, cos, sin, pos, layout)
        size = U.turn(x, weight, 1e-5, None, None, pos, layout).abs().amax(-1, keepdim=True)
        bound = P.rounding(want, 8 * 2.0 ** -24 * size, cache_type)
        return ((got.double().cpu() - want).abs() <= bound)

    assert close(got, q, qn).all()
    where = page_of[stored], slice(None), pos.cpu().long()[stored] % page
    keys, values = cache.keys.cpu(), cache.values.cpu()
    assert close(torch.where(stored[:, None, None], keys[page_of.clamp(min=0), :, pos.cpu().long() % page], 0), k, kn)[stored].all()
    assert torch.equal(values[where], v.to(cache_type).cpu()[stored])
    keys[where], values[where] = before[0].cpu()[where], before[1].cpu()[where]
    for now, was in ((keys, before[0]), (values, before[1])):  # and nothing else
        assert torch.equal(now.view(torch.int16), was.cpu().view(torch.int16))


def test_append_leaves_padding_alone(pkg):
    """Rows without a sequence, behind the table, behind the rotation's tables or at a negative position: neither stored nor their q_out written."""
    g = gen(5)
    cache, tables = paged(pkg, g, [16, 16], 8, 2, 64, BF16)
    before = cache.keys.clone()
    k = rand(g, 6, 2, 64)
    seq, pos = ints(0, -1, 2, 0, 1, 0), ints(-1, 3, 3, 16, -5, 13)
    cos, sin = (t.cuda() for t in U.tables(13, 64))
    out = torch.full((6, 2, 64), 7.0, device="cuda", dtype=BF16)
    cache.append(k, k, pos, tables, sequences=seq, q=k, cos=cos, sin=sin, q_out=out)
    assert (out == 7).all() and torch.equal(cache.keys.view(torch.int16), before.view(torch.int16))
    cache.append(k, k, pos, tables, sequences=seq, q=k, q_out=out)  # without a rotation the last one counts
    assert (out[:5] == 7).all() and torch.equal(out[5], k[5].bfloat16()) and torch.equal(cache.keys[tables[0, 1], :, 5], k[5].bfloat16())
    cache.append(k[:0], k[:0], pos[:0], tables)
    cache.append(k, k, pos, tables[:0], sequences=seq)
    cache.append(k, k, pos, tables[:, :0], sequences=seq)


def test_append_keeps_large_and_odd_numbers(pkg):
    cache, tables = paged(pkg, gen(1), [8], 8, 1, 32, F16)
    k = torch.zeros(4, 1, 32, device="cuda")
    k[0, 0, 0], k[1, 0, 1], k[2, 0, 2], k[3, 0, :] = 1e6, float("nan"), float("-inf"), 1e25
    cache.append(k, k, ints(0, 1, 2, 3), tables, k_norm=torch.ones(32, device="cuda"))
    v = cache.values[tables[0, 0], 0, :4].cpu()
    assert v[0, 0] == float("inf") and torch.isnan(v[1, 1]) and v[2, 2] == float("-inf")
    assert torch.allclose(cache.keys[tables[0, 0], 0, 3].float().cpu(), torch.ones(32), atol=1e-3)  # squares beyond FP32: the mean is taken in 64 bits


# ---- attention --------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("H,G,hs", [(4, 2, 32), (8, 8, 64), (16, 1, 64), (6, 2, 96), (32, 8, 128), (5, 1, 128), (8, 1, 256), (3, 3, 256), (40, 1, 64), (71, 1, 32)])
@pytest.mark.parametrize("dtype,page,window,out", [(BF16, 16, 0, F32), (F16, 1, 0, F32), (F16, 64, 20, F16), (BF16, 8, 1, BF16), (BF16, 256, 0, BF16)])
def test_single_rows(pkg, H, G, hs, dtype, page, window, out):
    g = gen(hs + page)
    cache, tables = paged(pkg, g, [1, 200, 16, 17, 67, 1], page, G, hs, dtype)
    pos, seq = ints(0, 199, 15, 16, 66, 3, -1, 150, 0, 5), ints(0, 1, 2, 3, 4, 4, 1, 1, 6, -1)
    q = rand(g, 10, H, hs, dtype=dtype)
    check(cache, q, pos, tables, seq, out, window=window)
    check(cache, q, pos, tables, seq, out, window=window, max_len=200)


@pytest.mark.parametrize("H,G,hs", [(4, 4, 32), (8, 2, 64), (24, 8, 96), (8, 2, 128), (16, 1, 128), (12, 1, 256), (40, 2, 64)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("queries,window", [(2, 0), (5, 0), (5, 3), (16, 30)])
def test_drafted_rows(pkg, H, G, hs, dtype, queries, window):
    """The last rows of sequences of many lengths, one of them shorter than its rows."""
    g, lengths = gen(H + hs), [queries, 70, 129, 31]
    cache, tables = paged(pkg, g, lengths, 16, G, hs, dtype)
    lengths[0] -= 1
    pos = torch.tensor([n - queries + i for n in lengths for i in range(queries)], device="cuda", dtype=torch.int32)
    seq = torch.arange(4, device="cuda", dtype=torch.int32).repeat_interleave(queries)
    check(cache, rand(g, 4 * queries, H, hs, dtype=dtype), pos, tables, seq, F32, window=window, chunk=queries, max_len=129)


@pytest.mark.parametrize("H,G,hs,page", [(8, 2, 64, 16), (24, 8, 96, 1), (16, 4, 128, 64), (4, 1, 128, 8), (16, 16, 64, 256), (8, 1, 256, 32), (4, 2, 32, 16)])
@pytest.mark.parametrize("dtype,out", [(F16, F16), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("window", [0, 70])
def test_chunks(pkg, H, G, hs, page, dtype, out, window):
    g = gen(hs + H)
    cache, tables = paged(pkg, g, [333, 77], page, G, hs, dtype)
    pos = torch.cat([torch.arange(333 - 150, 333, device="cuda"), torch.arange(77, device="cuda")]).int()
    seq = torch.tensor([0] * 150 + [1] * 77, device="cuda", dtype=torch.int32)
    check(cache, rand(g, 227, H, hs, dtype=dtype), pos, tables, seq, out, window=window, chunk=150, max_len=333)


@pytest.mark.parametrize("dtype,out", [(BF16, F32), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("chunk", [1, 7, 50, 10**9])
def test_rows_in_any_order(pkg, dtype, out, chunk):
    """What ``chunk`` and ``max_len`` say may be wrong: rows of many sequences, positions up and down, padding in between."""
    g = gen(chunk % 97)
    cache, tables = paged(pkg, g, [100, 40, 260], 16, 2, 64, dtype)
    seq = torch.randint(-1, 4, (90,), device="cuda", generator=g).int()
    pos = (torch.rand(90, device="cuda", generator=g) * ints(100, 40, 260, 10).float()[seq.clamp(min=0).long()]).int() - 2
    seq[40:60], pos[40:60] = 2, torch.arange(259, 239, -1, device="cuda")
    q = rand(g, 90, 8, 64, dtype=dtype)
    given = torch.full((90, 8, 64), 7.0, device="cuda", dtype=out)
    got = check(cache, q, pos, tables, seq, out, chunk=chunk, max_len=50)
    cache.attention(q, pos, tables, sequences=seq, chunk=chunk, out=given)
    pad = (seq < 0) | (seq > 2)
    assert (given[pad] == 7).all() and torch.equal(given[~pad], cache.attention(q, pos, tables, sequences=seq, chunk=chunk, dtype=out)[~pad])
    assert got.shape == given.shape


@pytest.mark.parametrize("G,mul,hs,page,queries", [(1, 8, 128, 64, 1), (8, 4, 128, 16, 1), (2, 5, 96, 32, 4), (1, 16, 64, 16, 3), (2, 4, 256, 64, 1), (3, 1, 32, 128, 1)])
def test_long_rows_are_split_and_joined(pkg, G, mul, hs, page, queries):
    g = gen(G)
    cache, tables = paged(pkg, g, [20011, 9000, 3], page, G, hs, BF16)
    pos = torch.tensor([n - queries + i for n in (20011, 9000, 3) for i in range(queries)], device="cuda", dtype=torch.int32)
    seq = torch.arange(3, device="cuda", dtype=torch.int32).repeat_interleave(queries)
    q = rand(g, 3 * queries, G * mul, hs, dtype=BF16)
    check(cache, q, pos, tables, seq, F32, chunk=queries)
    check(cache, q, pos, tables, seq, F32, chunk=queries, max_len=20011)
    check(cache, q, pos, tables, seq, F32, chunk=queries, max_len=8000)  # longer than it says
    check(cache, q, pos, tables, seq, F32, chunk=queries, window=12345)


@pytest.mark.parametrize("given", ["none", "little", "crooked"])
def test_workspaces(pkg, given):
    """Without a workspace, or with too little of it, a call does without; one that is not aligned is refused."""
    g, N = gen(3), pkg.native
    cache, tables = paged(pkg, g, [9000], 16, 2, 64, F16)
    q, pos = rand(g, 1, 8, 64, dtype=F16), ints(8999)
    out, work = torch.zeros(1, 8, 64, device="cuda"), torch.full((1000000,), 7.0, device="cuda")
    c, a, err = N.PagedCache(cache.keys.data_ptr(), cache.values.data_ptr(), cache.pages, 16, 2, 64, 1, 0), N.PagedAttention(), C.create_string_buffer(256)
    a.n, a.heads, a.q, a.out, a.q_stride, a.out_stride, a.positions, a.tables, a.table_stride, a.n_sequences, a.table_width, a.scale = 1, 8, q.data_ptr(), out.data_ptr(), 512, 512, pos.data_ptr(), \
        tables.data_ptr(), tables.shape[1], 1, tables.shape[1], 0.125
    need = N.lib().b200_paged_attention_workspace(C.byref(c), C.byref(a))
    assert 0 < need < 4000000
    a.workspace, a.workspace_bytes = {"none": (None, 0), "little": (work.data_ptr(), need - 1), "crooked": (work.data_ptr() + 4, need)}[given]
    rc = N.lib().b200_paged_attention(C.byref(c), C.byref(a), torch.cuda.current_stream().cuda_stream, err, 256)
    if given == "crooked":
        assert rc == -1
        return
    assert rc == 0
    want, bound = P.attention(q, cache.keys, cache.values, pos, None, tables, dtype=F32)
    assert ((out.double().cpu() - want).abs() <= bound).all() and (work == 7).all()


def test_pages_that_are_none_and_shared_ones(pkg):
    g = gen(9)
    cache, _ = paged(pkg, g, [64], 16, 2, 64, BF16)
    cache.keys.copy_(rand(g, *cache.keys.shape, dtype=BF16))
    cache.values.copy_(rand(g, *cache.keys.shape, dtype=BF16))
    tables = ints(0, -1, 2, 7, 0, 1, 2, 3, 2**31 - 1, 7, -2**31, -1).view(3, 4)
    pos, seq = ints(63, 30, 63, 15, 63, 17), ints(0, 0, 1, 1, 2, 2)
    for chunk in (1, 2, 6):
        got = check(cache, rand(g, 6, 4, 64, dtype=BF16), pos, tables, seq, F32, chunk=chunk)
        assert (got[4:] == 0).all()
    got = check(cache, rand(g, 2, 4, 64, dtype=BF16), ints(50, 63), tables, ints(0, 0), F32, chunk=2, window=3)  # the window holds only positions without a page
    assert (got == 0).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("chunk,hs,out", [(1, 128, F32), (6, 64, F32), (40, 64, F32), (40, 128, F32), (40, 64, None), (40, 96, None), (40, 128, None), (3, 128, None)])
def test_values_that_are_not_finite_reach_who_sees_them(pkg, dtype, bad, chunk, hs, out):
    g, out = gen(4), out or dtype
    cache, tables = paged(pkg, g, [90], 16, 2, hs, dtype)
    q = rand(g, 40, 8, hs, dtype=dtype)
    pos = torch.arange(50, 90, device="cuda", dtype=torch.int32)
    clean = cache.attention(q, pos, tables, chunk=chunk, window=20, dtype=out)
    cache.values[tables[0, 4], 1, 6, 5] = bad  # position 70: rows 70 .. 89 see it, in heads 4 .. 7, entry 5
    got = cache.attention(q, pos, tables, chunk=chunk, window=20, dtype=out)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[20:, 4:, 5] = True
    assert not torch.isfinite(got[hit]).any()
    want, bound = P.attention(q, cache.keys, torch.where(torch.isfinite(cache.values), cache.values, 0), pos, None, tables, window=20, dtype=out, probability=probability(cache, out))
    assert ((got.double().cpu() - want).abs() <= bound)[~hit.cpu()].all() and clean.isfinite().all()


def test_keys_that_are_not_finite(pkg):
    g = gen(4)
    cache, tables = paged(pkg, g, [90], 16, 2, 64, BF16)
    q, pos = rand(g, 40, 8, 64, dtype=BF16), torch.arange(50, 90, device="cuda", dtype=torch.int32)
    cache.keys[tables[0, 4], 1, 6, 5] = float("nan")
    for chunk in (1, 6, 40):  # the last on the tensor cores
        got = cache.attention(q, pos, tables, chunk=chunk)
        assert got[20:, 4:].isnan().all() and got[:20].isfinite().all() and got[:, :4].isfinite().all()


def test_values_near_the_types_end(pkg):
    """Sums of many large values leave FP32's range before they are divided: the result is their mean all the same."""
    cache, tables = paged(pkg, gen(1), [400], 16, 1, 64, BF16)
    cache.keys.zero_()
    cache.values.fill_(3e38)
    cache.values[:, :, :, 1] = -3e38
    top = float(torch.tensor(3e38).bfloat16())
    q, pos = torch.zeros(3, 4, 64, device="cuda", dtype=BF16), ints(0, 100, 399)
    for chunk in (1, 3):
        got = cache.attention(q, pos, tables, chunk=chunk, dtype=F32).cpu() / top
        assert torch.allclose(got[..., 0], torch.ones(3, 4), atol=1e-4) and torch.allclose(got[..., 1], -torch.ones(3, 4), atol=1e-4)
    q, pos = torch.zeros(40, 4, 64, device="cuda", dtype=BF16), torch.arange(360, 400, device="cuda", dtype=torch.int32)
    got = cache.attention(q, pos, tables, chunk=40).float().cpu() / top  # (on the tensor cores, then once more)
    assert torch.allclose(got[..., 0], torch.ones(40, 4), atol=2.0 ** -7) and torch.allclose(got[..., 1], -torch.ones(40, 4), atol=2.0 ** -7)


@pytest.mark.parametrize("gain,scale", [(30.0, None), (1.0, 0.0), (1.0, -0.3), (3.0, 1.0), (1e-3, None)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_scores_of_any_size(pkg, gain, scale, dtype):
    g = gen(11)
    cache, tables = paged(pkg, g, [300], 32, 2, 64, dtype, gain)
    pos = ints(0, 299, 5, 120)
    kw = {} if scale is None else {"scale": scale}
    check(cache, rand(g, 4, 8, 64, dtype=dtype), pos, tables, None, F32, **kw)
    check(cache, rand(g, 4, 8, 64, dtype=dtype), pos, tables, None, F32, chunk=4, **kw)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_long_tail_of_small_probabilities_counts(pkg, dtype):
    """One position 2^20 times as likely as 8000 others, whose values are large."""
    cache, tables = paged(pkg, gen(2), [8000], 64, 1, 64, dtype)
    cache.keys.zero_()
    cache.values.fill_(100.0)
    cache.keys[tables[0, 0], 0, 3, 0], cache.values[tables[0, 0], 0, 3] = 1.0, 0.0
    q = torch.zeros(2, 4, 64, device="cuda", dtype=dtype)
    q[:, :, 0] = 20.0
    scale = 0.6931471805599453
    got = cache.attention(q, ints(7999, 7998), tables, scale=scale, chunk=2, dtype=F32).double().cpu()
    want, bound = P.attention(q, cache.keys, cache.values, ints(7999, 7998), None, tables, scale=scale, dtype=F32)
    assert ((got - want).abs() <= bound).all() and ((got / want - 1).abs() < 0.01).all()


@pytest.mark.parametrize("pad,out", [(1, F32), (3, BF16), (8, F32), (4, F16)])
def test_rows_of_wider_ones(pkg, pad, out):
    g = gen(pad)
    dtype = BF16 if out == F32 else out
    cache, tables = paged(pkg, g, [70, 9], 16, 2, 64, dtype)
    seq, pos = ints(0, 1, 0, 0, 0), ints(69, 8, 3, 4, 5)
    q = rand(g, 5, 8 * 64 + pad, dtype=dtype)[:, pad:].view(5, 8, 64)
    wide = torch.full((5, 8 * 64 + 2 * pad), 7.0, device="cuda", dtype=out)
    place = wide[:, pad:-pad].view(5, 8, 64)
    wide_tables = torch.full((2, tables.shape[1] + 3), 10**9, device="cuda", dtype=torch.int32)
    wide_tables[:, 1:-2] = tables
    for chunk in (1, 3, 5):
        place.fill_(7.0)
        cache.attention(q, pos, wide_tables[:, 1:-2], sequences=seq, chunk=chunk, out=place)
        want, bound = P.attention(q, cache.keys, cache.values, pos, seq, tables, dtype=out, probability=probability(cache, out))
        assert ((place.double().cpu() - want).abs() <= bound).all()
        assert (wide[:, :pad] == 7).all() and (wide[:, -pad:] == 7).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,G,hs,page,lengths,chunk,window", [(8, 2, 64, 16, [3000, 777], 64, 0), (4, 1, 128, 64, [4100], 128, 0), (4, 1, 128, 32, [9000], 33, 0), (3, 1, 96, 16, [2500, 40, 700], 40, 1500),
                                                              (64, 1, 64, 8, [5000], 3, 0), (4, 1, 64, 64, [40000], 32, 0), (128, 1, 64, 16, [300], 5, 0), (16, 8, 96, 1, [1000, 900], 50, 333)])
def test_chunks_of_long_sequences(pkg, dtype, H, G, hs, page, lengths, chunk, window):
    """Few rows over many positions (shared by several CTAs) and many rows; sequences with holes and scores that grow."""
    g = gen(chunk)
    cache, tables = paged(pkg, g, lengths, page, G, hs, dtype)
    for n, t in zip(lengths, tables):
        at = torch.arange(n, device="cuda")
        cache.keys[t.long()[at // page], :, at % page] *= (0.2 + 3 * at / n)[:, None, None]  # a maximum that keeps growing
    if page > 1:
        tables[:, 1] = -1
    pos = torch.cat([torch.arange(n - min(chunk, n), n, device="cuda") for n in lengths]).int()
    seq = torch.cat([torch.full((min(chunk, n),), s, device="cuda") for s, n in enumerate(lengths)]).int()
    check(cache, rand(g, len(pos), H, hs, dtype=dtype), pos, tables, seq, dtype, chunk=chunk, window=window)
    check(cache, rand(g, len(pos), H, hs, dtype=dtype), pos, tables, seq, dtype, chunk=chunk, window=window, max_len=max(lengths), scale=-0.2)


@pytest.mark.parametrize("n,chunk,out", [(300, 1, F32), (1500, 1500, F32), (700, 3, F16)])
def test_more_rows_than_are_shared_out(pkg, n, chunk, out):
    """Many groups of rows take a CTA a unit, whatever their lengths are; results of another 16-bit type than the cache's."""
    g = gen(n)
    cache, tables = paged(pkg, g, [500, 40, 1400], 16, 1, 32, BF16)
    seq = torch.randint(-1, 3, (n,), device="cuda", generator=g).int() if chunk < n else torch.full((n,), 2, device="cuda", dtype=torch.int32)
    pos = (torch.rand(n, device="cuda", generator=g) * ints(500, 40, 1400).float()[seq.clamp(min=0).long()]).int() if chunk < n else torch.arange(n, device="cuda").int() - 100
    check(cache, rand(g, n, 2, 32, dtype=BF16), pos, tables, seq, out, chunk=chunk)


def test_offsets_beyond_32_bits(pkg):
    """A pool of 2 x 5.2 GB: entries behind 2^31 and bytes behind 2^32."""
    g, G, hs, page, pages = gen(12), 8, 128, 256, 10000
    cache = pkg.PagedKVCache(pages, page, G, hs, dtype=BF16)
    tables = ints(pages - 1, 3, pages - 2).view(1, 3)
    n = 600
    k, v, pos = rand(g, n, G, hs, dtype=BF16), rand(g, n, G, hs, dtype=BF16), torch.arange(n, device="cuda", dtype=torch.int32)
    cache.append(k, v, pos, tables)
    assert torch.equal(cache.keys[pages - 1].transpose(0, 1), k[:256]) and torch.equal(cache.values[pages - 2, :, :88].transpose(0, 1), v[512:])
    small, q = pkg.PagedKVCache(3, page, G, hs, dtype=BF16), rand(g, 64, 2 * G, hs, dtype=BF16)
    for name in ("keys", "values"):
        getattr(small, name).copy_(getattr(cache, name)[tables[0].long()])
    for chunk, out in ((1, F32), (64, BF16)):
        got = cache.attention(q, pos[-64:], tables, chunk=chunk, dtype=out)
        assert torch.equal(got, small.attention(q, pos[-64:], ints(0, 1, 2).view(1, 3), chunk=chunk, dtype=out))
    check(small, q, pos[-64:], ints(0, 1, 2).view(1, 3), None, F32)


def test_a_wait_that_runs_out_is_heard_of(pkg):
    """Rows of a block whose wait ran out are NaN, whether they are joined or not, and the next call is as it was."""
    g, N = gen(3), pkg.native
    for length, heads in ((300, 8), (5000, 4)):
        cache, tables = paged(pkg, g, [length], 16, heads // 4, 64, F16)
        q, pos = rand(g, 32, heads, 64, dtype=F16), torch.arange(length - 32, length, device="cuda", dtype=torch.int32)
        want = cache.attention(q, pos, tables, chunk=32)
        out = torch.zeros(32, heads, 64, device="cuda", dtype=F16)
        c, a, err = N.PagedCache(cache.keys.data_ptr(), cache.values.data_ptr(), cache.pages, 16, heads // 4, 64, 1, 0), N.PagedAttention(), C.create_string_buffer(256)
        a.n, a.heads, a.q, a.out, a.q_stride, a.out_stride, a.positions, a.tables, a.table_stride, a.n_sequences, a.table_width, a.scale, a.chunk, a.out_type = 32, heads, q.data_ptr(), out.data_ptr(), \
            heads * 64, heads * 64, pos.data_ptr(), tables.data_ptr(), tables.shape[1], 1, tables.shape[1], 0.125, 32, 1
        need = N.lib().b200_paged_attention_workspace(C.byref(c), C.byref(a))
        work = torch.zeros(need // 4 + 4, device="cuda")
        a.workspace, a.workspace_bytes = work.data_ptr(), need
        assert (need > 0) == (length == 5000)
        assert N.lib().b200_test_paged_give_up(C.byref(c), C.byref(a), torch.cuda.current_stream().cuda_stream, err, 256) == 0
        torch.cuda.synchronize()
        assert out.isnan().all()
        assert torch.equal(cache.attention(q, pos, tables, chunk=32), want)


# ---- streams, graphs, repeats ------------------------------------------------------------------------------------------------------------
def test_the_same_bits_again_captured_or_not(pkg):
    g = gen(6)
    cache, tables = paged(pkg, g, [5000, 70, 900], 16, 2, 128, BF16)
    pos, seq = ints(4990, 60, 880), ints(0, 1, 2)
    q, k = rand(g, 3, 8, 128, dtype=BF16), rand(g, 3, 2, 128, dtype=BF16)
    cos, sin = (t.cuda() for t in U.tables(5000, 128))
    graphs, outs = [], []
    for _ in range(2):  # two graphs: a workspace each
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            cache.attention(q, pos, tables, sequences=seq)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            turned = cache.append(k, k, pos, tables, sequences=seq, q=q, cos=cos, sin=sin)
            outs.append(cache.attention(turned, pos, tables, sequences=seq, chunk=1))
        graphs.append(graph)
    for step in range(3):
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        turned = cache.append(k, k, pos, tables, sequences=seq, q=q, cos=cos, sin=sin)
        want = cache.attention(turned, pos, tables, sequences=seq, chunk=1)
        assert all(torch.equal(o, want) for o in outs) and torch.equal(want, cache.attention(turned, pos, tables, sequences=seq, chunk=1))
        check(cache, turned, pos, tables, seq, BF16)
        pos += 1
        q.copy_(rand(g, 3, 8, 128, dtype=BF16))


def test_streams_beside_each_other(pkg):
    g = gen(8)
    cache, tables = paged(pkg, g, [9000, 8000], 16, 2, 64, F16)
    q = [rand(g, 1, 8, 64, dtype=F16) for _ in range(2)]
    where = [(ints(8999), ints(0)), (ints(7999), ints(1))]
    want = [cache.attention(x, p, tables, sequences=s) for x, (p, s) in zip(q, where)]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(cache.attention(q[i], where[i][0], tables, sequences=where[i][1]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for os, w in zip(outs, want) for o in os)


# ---- refusals ---------------------------------------------------------------------------------------------------------------------------
def test_refusals(pkg):
    cache, tables = paged(pkg, gen(1), [20], 16, 2, 64, BF16)
    k, q, pos = rand(gen(1), 3, 2, 64), rand(gen(2), 3, 4, 64, dtype=BF16), ints(0, 1, 2)
    w, cos = torch.ones(64, device="cuda"), torch.ones(20, 32, device="cuda")
    on = lambda y: y.clone().requires_grad_()  # noqa: E731
    bad = [lambda: cache.append(k.cpu(), k, pos, tables), lambda: cache.append(k, k.half(), pos, tables), lambda: cache.append(k.double(), k.double(), pos, tables), lambda: cache.append(k[:, :1], k, pos, tables),
           lambda: cache.append(k, k, pos.long(), tables), lambda: cache.append(k, k, pos[:2], tables), lambda: cache.append(k, k, pos, tables.long()), lambda: cache.append(k, k, pos, tables[0]),
           lambda: cache.append(k, k, pos, tables.cpu()), lambda: cache.append(k, k, pos, tables, sequences=pos[:2]), lambda: cache.append(k, k, pos, tables, cos=cos), lambda: cache.append(k, k, pos, tables, cos=cos, sin=cos[:10]),
           lambda: cache.append(k, k, pos, tables, cos=torch.ones(20, 33, device="cuda"), sin=torch.ones(20, 33, device="cuda")), lambda: cache.append(k, k, pos, tables, layout="other"), lambda: cache.append(k, k, pos, tables, q_norm=w),
           lambda: cache.append(k, k, pos, tables, k_norm=w[:3]), lambda: cache.append(k, k, pos, tables, q=k, q_out=k), lambda: cache.append(k.bfloat16(), k.bfloat16(), pos, tables, q=q, q_out=q), lambda: cache.append(k.transpose(1, 2), k, pos, tables), lambda: cache.append(on(k), k, pos, tables),
           lambda: cache.append(k, k, pos, tables, q=on(k)), lambda: cache.append(k, k, pos, tables, k_norm=on(w)), lambda: cache.attention(q.float(), pos, tables), lambda: cache.attention(q[:, :3], pos, tables),
           lambda: cache.attention(on(q), pos, tables), lambda: cache.attention(q, pos, tables, window=-1), lambda: cache.attention(q, pos, tables, dtype=torch.float64), lambda: cache.attention(q, pos, tables, out=q[:2]),
           lambda: cache.attention(q, pos, tables, chunk=-1), lambda: cache.attention(q[:, :, ::2], pos, tables), lambda: cache.attention(q, pos[::2], tables), lambda: cache.attention(q, pos, tables.repeat(2, 1).T)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        cache.attention(q, None, tables)
    for hs, page in ((80, 16), (64, 24)):
        with pytest.raises(pkg.native.UnsupportedOperation):
            pkg.PagedKVCache(2, page, 2, hs)
    with torch.no_grad():
        cache.append(on(k), k, pos, tables)
        cache.attention(on(q), pos, tables)
