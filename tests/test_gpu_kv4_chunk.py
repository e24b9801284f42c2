"""Attention of prompt chunks over the 4-bit cache with 16-bit results (the tensor-core form) against the plain 64-bit form."""
import ctypes as C

import pytest
import torch

import kv4_util as U
from test_gpu_kv4 import BF16, F16, F32, filled, gen, ints, rand

pytestmark = pytest.mark.gpu


def check(got, q, k, v, d, pos, slots, scale, window, dtype):
    assert got.dtype == dtype
    qq, pos, slots = q.double().cpu(), pos.cpu(), slots.cpu()
    want, _ = U.attention(qq, k, v, d, pos, slots, scale, window)
    bound = U.chunk_bound(qq, k, v, pos, slots, scale, window, want, dtype)
    off = (got.double().cpu() - want).abs()
    assert (off <= bound).all(), (off / bound).max()


@pytest.mark.parametrize("H,G,hs", [(8, 2, 128), (4, 4, 64), (6, 2, 96), (7, 1, 64), (64, 1, 128), (128, 1, 64), (24, 8, 96)])
@pytest.mark.parametrize("n,start", [(64, 0), (70, 300), (128, 1), (33, 127), (129, 511)])
def test_one_chunk(pkg, H, G, hs, n, start):
    """The tokens of a prompt from a position on: the first sees only itself, tiles end inside records and the other way round."""
    if n * (H // G) < 64:
        n = 64
    context = start + n
    cache, k, v, d = filled(pkg, 1, context, G, hs, n + hs)
    q = rand(gen(n), n, H, hs) * 1.4
    pos, slots = torch.arange(start, context, device="cuda", dtype=torch.int32), torch.zeros(n, device="cuda", dtype=torch.int32)
    for dtype in (F16, BF16):
        check(cache.attention(q, pos, slots=slots, chunk=n, max_len=context, dtype=dtype), q, k, v, d, pos, slots, U.rsqrt(hs), 0, dtype)


@pytest.mark.parametrize("H,G,hs,window,scale,pad", [(8, 2, 128, 0, None, 0), (8, 2, 64, 77, 0.3, 1), (6, 2, 96, 1, None, 4), (4, 1, 64, 0, -0.2, 8), (4, 1, 128, 300, 0.0, 0)])
def test_chunks_of_many_sequences(pkg, H, G, hs, window, scale, pad):
    """Runs of any length in any order of slots, rows that see nothing, padding in the middle and at the end, positions out of order, the same slot in two runs, padded rows."""
    g, slots, context = gen(hs), 4, 400
    cache, k, v, d = filled(pkg, slots, context, G, hs, hs + window)
    runs = [(2, 0, 50), (0, 399, 1), (1, 130, 90), (slots, 7, 5), (2, 200, 33), (3, -20, 40), (0, 100, 60), (1, context, 3), (3, 300, 64)]
    pos = torch.cat([torch.arange(p, p + n) for _, p, n in runs]).int().cuda()
    at = torch.cat([torch.full((n,), s) for s, _, n in runs]).int().cuda()
    pos[60:90] = pos[60:90].flip(0)
    n = len(pos)
    wide_q, wide_out = rand(g, n, H * hs + pad), torch.full((n, H * hs + pad), 7.5, device="cuda", dtype=BF16)
    q, out = wide_q[:, pad:].view(n, H, hs), wide_out[:, pad:].view(n, H, hs)
    cache.attention(q, pos, slots=at, chunk=50, window=window, scale=scale, out=out)
    padding = (at < 0) | (at >= slots) | (pos >= context)
    assert padding.sum() >= 8 and (out[padding] == 7.5).all() and (wide_out[:, :pad] == 7.5).all() and (out[(pos < 0) & ~padding] == 0).all()
    live = ~padding
    check(out[live], q[live], k, v, d, pos[live], at[live], U.rsqrt(hs) if scale is None else scale, window, BF16)


@pytest.mark.parametrize("H,G,hs,n", [(4, 1, 128, 40), (8, 2, 64, 100), (3, 1, 96, 64)])
def test_long_chunks_shared_by_many_blocks(pkg, H, G, hs, n):
    """Few rows over many positions: the blocks of a tile leave parts in the workspace."""
    context = 12000
    cache, k, v, d = filled(pkg, 2, context, G, hs, n)
    q = rand(gen(n), n, H, hs)
    pos, slots = torch.arange(context - n, context, device="cuda", dtype=torch.int32), torch.ones(n, device="cuda", dtype=torch.int32)
    a = pkg.native.KV4Attention()
    a.n, a.heads, a.out_type, a.chunk = n, H, 1, n
    raw, err = C.c_void_p(), C.create_string_buffer(256)
    assert pkg.native.lib().b200_kv4_create(2, context, G, hs, 0, C.byref(raw), err, 256) == 0
    assert pkg.native.lib().b200_kv4_attention_workspace(raw, C.byref(a)) > 0
    pkg.native.lib().b200_kv4_free(raw)
    check(cache.attention(q, pos, slots=slots, chunk=n, dtype=F16), q, k, v, d, pos, slots, U.rsqrt(hs), 0, F16)


@pytest.mark.parametrize("hs", [64, 96, 128])
def test_what_a_row_does_not_see_does_not_reach_it(pkg, hs):
    """NaN, infinities and values outside FP16 in keys and values, in front of, behind and between what the rows see: rows that see one are NaN, the others clean."""
    H, G, context, n = 4, 1, 300, 130
    cache, k, v, d = filled(pkg, 1, context, G, hs, 8)
    odd = torch.full((context, G, hs), float("nan"), device="cuda")
    odd[200] = float("inf")
    odd[40], odd[280] = 1e6, -3e5  # stored as numbers; FP16 does not hold them
    at = torch.arange(context, device="cuda", dtype=torch.int32)
    k_bad, v_bad = [3, 250, 200], [40, 230, 280]
    rows = torch.tensor(k_bad, device="cuda")
    cache.append(odd[rows], cache.read(rows.int())[1], rows.int())
    rows = torch.tensor(v_bad, device="cuda")
    cache.append(cache.read(rows.int())[0], odd[rows], rows.int())
    q, pos = rand(gen(2), n, H, hs), torch.arange(140, 140 + n, device="cuda", dtype=torch.int32)
    window = 60
    got = cache.attention(q, pos, window=window, chunk=n, dtype=F16)
    sees = torch.tensor([any(p - window < b <= p for b in k_bad + v_bad) for p in pos.tolist()])
    assert sees.any() and (~sees).any()
    assert torch.isnan(got.cpu()[sees]).flatten(1).any(1).all()  # (an entry of its group at least)
    clean = ~sees.cuda()
    kk, vv = cache.read(at)
    check(got[clean], q[clean], torch.nan_to_num(kk).double().cpu()[None], torch.nan_to_num(vv).double().cpu()[None], d, pos[clean], torch.zeros_like(pos[clean]), U.rsqrt(hs), window, F16)


def test_large_scores_and_growing_maxima(pkg):
    """Every tile moves the rows' maxima by far more than the threshold, in one order or the other."""
    H, G, hs, context, n = 2, 1, 64, 700, 64
    g = gen(6)
    for falling in (False, True):
        cache = pkg.KV4Cache(1, context, G, hs)
        one = torch.randn(hs, device="cuda", generator=g)
        ramp = torch.linspace(0, 200, context, device="cuda")
        k = (ramp.flip(0) if falling else ramp)[:, None, None] * one / (one @ one)
        v = rand(g, context, G, hs)
        at = torch.arange(context, device="cuda", dtype=torch.int32)
        cache.append(k, v, at)
        (kk, kd), (vv, vd) = U.quantize(k), U.quantize(v)
        q = one * (1 + 0.1 * rand(g, n, H, hs))
        pos = at[context - n:]
        got = cache.attention(q, pos, scale=1.0, chunk=n, dtype=F16)
        check(got, q, kk[None], vv[None], (kd[None], vd[None]), pos, torch.zeros_like(pos), 1.0, 0, F16)


def test_captured_side_by_side_and_again(pkg):
    """The same bits from captured graphs, on two streams at once and beside the form of single rows."""
    cache, _, _, _ = filled(pkg, 2, 3000, 2, 128, 11)
    q = rand(gen(1), 100, 8, 128)
    pos, slots = torch.arange(2500, 2600, device="cuda", dtype=torch.int32), torch.ones(100, device="cuda", dtype=torch.int32)
    call = lambda: cache.attention(q, pos, slots=slots, chunk=100, dtype=BF16)  # noqa: E731
    first = call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(4):
                outs.append(call())
                cache.attention(q[:5], pos[:5], slots=slots[:5])
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, first)
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)


def test_a_prompt_in_chunks_then_steps(pkg):
    """A prompt goes in by chunks (norms, rotation, append, attention), then tokens one by one: every row as if computed from the rotated keys directly."""
    H, G, hs, context = 8, 2, 64, 420
    g = gen(21)
    cache = pkg.KV4Cache(3, context, G, hs)
    cos, sin = (t.cuda() for t in U.tables(context, hs))
    qn, kn = 1 + 0.2 * rand(g, hs), 1 + 0.2 * rand(g, hs)
    qkv = rand(g, context, (H + 2 * G) * hs)
    q, k, v = (qkv[:, a * hs:b * hs].view(context, b - a, hs) for a, b in ((0, H), (H, H + G), (H + G, H + 2 * G)))
    outs, turned, at, done = [], [], torch.full((context,), 2, device="cuda", dtype=torch.int32), 0
    for n in [128, 200, 64] + [1] * 28:
        rows = slice(done, done + n)
        pos = torch.arange(done, done + n, device="cuda", dtype=torch.int32)
        turned.append(cache.append(k[rows], v[rows], pos, q=q[rows], slots=at[:n], q_norm=qn, k_norm=kn, cos=cos, sin=sin))
        outs.append(cache.attention(turned[-1], pos, slots=at[:n], chunk=n, max_len=done + n, dtype=F16))
        done += n
    every = torch.arange(context, device="cuda", dtype=torch.int32)
    kk, vv = (t.double().cpu()[None] for t in cache.read(every, slots=at))
    x = U.turn(k, kn, 1e-6, cos, sin, every, "half")
    d = U.quantize(x)[1], U.quantize(v)[1]
    assert (kk[0] - x).abs().max() <= d[0].abs().max() * 1.01  # a step of the cache at most
    check(torch.cat(outs), torch.cat(turned), kk, vv, [s[None] for s in d], every, torch.zeros_like(every), U.rsqrt(hs), 0, F16)


@pytest.mark.parametrize("window", [0, 150])
def test_scores_beyond_single_precision_exponentials(pkg, window):
    """Exact scores, thousands apart and up to 2^23: every row is the value at its largest one, wherever that stands.  (A score and the maximum that round apart would lose it.)
    The value is an FP16 operand and the result FP16: half a step each."""
    H, G, hs, context, n = 4, 1, 64, 500, 100
    g = gen(12)
    cache = pkg.KV4Cache(1, context, G, hs)
    order = torch.randperm(context, device="cuda", generator=g)
    k = torch.zeros(context, G, hs, device="cuda")
    k[:, 0, 0] = -(order + 1.0)  # the largest entry of its group: stored exactly
    at = torch.arange(context, device="cuda", dtype=torch.int32)
    cache.append(k, rand(g, context, G, hs), at)
    kk, vv = cache.read(at)
    assert torch.equal(kk, k)
    q = torch.zeros(n, H, hs, device="cuda")
    q[:, :, 0] = -16384.0
    pos = at[context - n:]
    got = cache.attention(q, pos, window=window, scale=1.0, chunk=n, dtype=F16)
    for r, p in enumerate(pos.tolist()):
        lo = max(0, p - window + 1) if window else 0
        want = vv[lo + int(order[lo:p + 1].argmax()), 0].double()
        assert ((got[r].double() - want).abs() <= want.abs() * 2 * U.half_step(F16) + 2.0 ** -25).all()


@pytest.mark.parametrize("context", [1, 16, 128, 129, 256, 257, 385])
def test_few_tiles(pkg, context):
    """One tile, two, three: a stream of tiles without work, or with one tile fewer than the other; all tokens at the same position, some of them twice."""
    H, G, hs, n = 4, 2, 96, 40
    cache, k, v, d = filled(pkg, 1, context, G, hs, context)
    q = rand(gen(context), n, H, hs)
    pos = torch.full((n,), context - 1, device="cuda", dtype=torch.int32)
    pos[::3] = 0
    check(cache.attention(q, pos, chunk=n, max_len=context, dtype=BF16), q, k, v, d, pos, torch.zeros_like(pos), U.rsqrt(hs), 0, BF16)


def test_a_crooked_workspace_is_refused(pkg):
    lib, raw, err = pkg.native.lib(), C.c_void_p(), C.create_string_buffer(256)
    assert lib.b200_kv4_create(1, 64, 1, 64, 0, C.byref(raw), err, 256) == 0
    x = torch.zeros(64, 64, device="cuda")
    a = pkg.native.KV4Attention()
    a.n, a.heads, a.chunk, a.q_stride, a.out_stride, a.q, a.out, a.workspace = 64, 1, 64, 64, 64, x.data_ptr(), x.data_ptr(), x.data_ptr() + 8
    assert lib.b200_kv4_attention(raw, C.byref(a), None) == -1
    lib.b200_kv4_free(raw)
