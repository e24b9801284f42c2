"""The 4-bit key/value cache and its attention on the GPU against their plain 64-bit forms."""
import ctypes as C

import pytest
import torch

import kv4_util as U

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=F32):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def ints(*v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


def filled(pkg, slots, context, G, hs, seed, gain=1.0):
    """A full cache and its values: (cache, k, v, the scales of both), [slots, context, G, ...] in float64 on the CPU."""
    g = gen(seed)
    cache = pkg.KV4Cache(slots, context, G, hs)
    k, v = rand(g, slots * context, G, hs) * gain, rand(g, slots * context, G, hs) * 0.5
    at = torch.arange(slots * context, device="cuda", dtype=torch.int32)
    cache.append(k, v, at % context, slots=at // context)
    (kv, kd), (vv, vd) = U.quantize(k), U.quantize(v)
    return cache, kv.view(slots, context, G, hs), vv.view(slots, context, G, hs), [d.view(slots, context, G, -1) for d in (kd, vd)]


# ---- append and read ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hs", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_append_stores_the_definitions_codes(pkg, hs, dtype):
    g, G, slots, context = gen(hs), 3, 2, 37
    cache = pkg.KV4Cache(slots, context, G, hs)
    places = torch.randperm(slots * context, generator=g, device="cuda")[:50].int()  # any order, both slots
    k, v = rand(g, 50, G, hs, dtype=dtype) * 3, rand(g, 50, G, hs, dtype=dtype)
    cache.append(k, v, places % context, slots=places // context)
    every = torch.arange(slots * context, device="cuda", dtype=torch.int32)
    rk, rv = cache.read(every % context, slots=every // context)
    for got, x in ((rk, k), (rv, v)):
        want = torch.zeros(slots * context, G, hs, dtype=torch.float64)
        want[places.cpu().long()] = U.quantize(x)[0]
        assert torch.equal(got.double().cpu(), want)  # a scale of 11 bits times a code of 4: FP32 holds it
        assert (got[~torch.isin(every, places)] == 0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_read_types(pkg, dtype):
    cache, k, v, _ = filled(pkg, 1, 20, 2, 64, 3)
    at = torch.arange(20, device="cuda", dtype=torch.int32)
    for got, want in zip(cache.read(at, dtype=dtype), (k[0], v[0])):
        assert got.dtype == dtype and torch.equal(got.cpu(), want.to(dtype))


@pytest.mark.parametrize("H,G,hs", [(4, 2, 32), (8, 8, 64), (6, 2, 96), (5, 1, 128), (3, 3, 256)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("norm,dtype,pad", [(True, F32, 0), (False, F32, 1), (True, BF16, 3), (False, F16, 8)])
def test_append_norms_and_rotates(pkg, H, G, hs, layout, norm, dtype, pad):
    """Queries within FP32 of the 64-bit form; keys within half a step of it (one where the other end of the range cuts them off)."""
    g, n, context = gen(H * hs + pad), 33, 64
    cache = pkg.KV4Cache(1, context, G, hs)
    wide = rand(g, n, (H + 2 * G) * hs + pad, dtype=dtype) * 2  # parts of a padded row, unaligned where pad is odd
    q, k, v = (wide[:, a * hs + pad:b * hs + pad].view(n, b - a, hs) for a, b in ((0, H), (H, H + G), (H + G, H + 2 * G)))
    cos, sin = (t.cuda() for t in U.tables(context, hs))
    qn, kn = (1 + 0.3 * rand(g, hs), 1 + 0.3 * rand(g, hs)) if norm else (None, None)
    pos = torch.randperm(context, generator=g, device="cuda")[:n].int()
    got = cache.append(k, v, pos, q=q, q_norm=qn, k_norm=kn, eps=1e-5, cos=cos, sin=sin, layout=layout)
    want = U.turn(q, qn, 1e-5, cos, sin, pos, layout)
    size = U.turn(q, qn, 1e-5, None, None, pos, layout).abs().amax(-1, keepdim=True)
    assert ((got.double().cpu() - want).abs() <= 8 * 2.0 ** -24 * size).all()  # norm: 3 roundings (s, s x, w s x), rotation: products and sum, 3 of at most |a| + |b|
    rk, rv = cache.read(pos)
    assert torch.equal(rv.double().cpu(), U.quantize(v)[0])
    x = U.turn(k, kn, 1e-5, cos, sin, pos, layout)
    _, d = U.quantize(x)
    step = d.abs().repeat_interleave(32, -1)
    off = (rk.double().cpu() - x).abs()
    cut = (x / d.repeat_interleave(32, -1)) > 7.4
    assert (off <= step * 0.501)[~cut].all() and (off <= step * 1.002)[cut].all() and cut.float().mean() < 0.05


def test_append_leaves_padding_alone(pkg):
    g, n, context = gen(1), 9, 16
    cache = pkg.KV4Cache(2, context, 2, 64)
    k, v, q = rand(g, n, 2, 64), rand(g, n, 2, 64), rand(g, n, 4, 64)
    pos, slots = ints(0, 16, -1, 3, 4, 2**31 - 1, -2**31, 7, 15), ints(0, 0, 0, 2, -1, 1, 1, 1, 1)
    out = torch.full((n, 4, 64), 7.5, device="cuda")
    cache.append(k, v, pos, q=q, slots=slots, q_out=out)
    kept = torch.tensor([True, False, False, False, False, False, False, True, True])
    assert (out[~kept] == 7.5).all() and torch.equal(out[kept], q[kept])
    every = torch.arange(2 * context, device="cuda", dtype=torch.int32)
    rk, _ = cache.read(every % context, slots=every // context)
    there = {0: 0, 16 + 7: 7, 16 + 15: 8}
    for i in range(2 * context):
        want = U.quantize(k[there[i]])[0] if i in there else torch.zeros(2, 64, dtype=torch.float64)
        assert torch.equal(rk[i].double().cpu(), want)


def test_append_odd_values(pkg):
    cache = pkg.KV4Cache(1, 8, 1, 64)
    x = torch.zeros(8, 1, 64, device="cuda")
    x[1, 0, 3], x[1, 0, 7] = 2.0, -2.0
    x[2, 0, 31], x[2, 0, 0] = -8.0, 0.5
    x[3, 0, 5] = float("nan")
    x[4, 0, 40] = float("-inf")
    x[5, 0, 0], x[5, 0, 32] = 1e30, 3e-8
    x[6] = 1e-7
    x[7] = torch.linspace(-1, 1, 64, device="cuda")
    at = torch.arange(8, device="cuda", dtype=torch.int32)
    cache.append(x, -x, at)
    rk, rv = cache.read(at)
    for got, y in ((rk, x), (rv, -x)):
        assert torch.equal(torch.nan_to_num(got.double().cpu(), nan=99.0), torch.nan_to_num(U.quantize(y)[0], nan=99.0))
    assert torch.isnan(rk[3, 0, :32]).all() and not torch.isnan(rk[3, 0, 32:]).any()


def test_reset_and_bytes(pkg):
    cache, _, _, _ = filled(pkg, 2, 30, 2, 96, 5)
    assert cache.device_bytes == 2 * 2 * 2 * 18 * 96  # two blocks of 16 positions a slot and head
    cache.reset()
    at = torch.arange(30, device="cuda", dtype=torch.int32)
    for t in cache.read(at, slots=torch.ones_like(at)):
        assert (t == 0).all()
    cache.free()
    with pytest.raises(pkg.native.B200Error):
        cache.reset()
    cache.free()


# ---- attention ------------------------------------------------------------------------------------------------------------------------
def check(got, q, k, v, d, pos, slots, scale, window):
    want, bound = U.attention(q.double().cpu(), k, v, d, pos.cpu(), slots.cpu(), scale, window)
    bound = bound + want.abs() * (0 if got.dtype == F32 else U.half_step(got.dtype)) + 1e-30
    off = (got.double().cpu() - want).abs()
    assert (off <= bound).all(), (off / bound).max()


@pytest.mark.parametrize("H,G,hs", [(4, 4, 32), (8, 2, 64), (6, 2, 96), (32, 8, 128), (4, 1, 256), (14, 2, 64), (20, 1, 128), (10, 1, 32), (8, 1, 256)])
@pytest.mark.parametrize("length", [1, 15, 16, 17, 129, 1000])
def test_single_rows(pkg, H, G, hs, length):
    cache, k, v, d = filled(pkg, 2, 1001, G, hs, length + hs)
    q = rand(gen(length), 1, H, hs)
    pos, slots = ints(length - 1), ints(1)
    for dtype in (F32, F16, BF16):
        got = cache.attention(q, pos, slots=slots, dtype=dtype)
        check(got, q, k, v, d, pos, slots, U.rsqrt(hs), 0)
    check(cache.attention(q, pos, slots=slots, window=100, max_len=length, scale=0.3), q, k, v, d, pos, slots, 0.3, 100)


@pytest.mark.parametrize("H,G,hs,n,window,max_len,pad", [(8, 2, 64, 40, 0, 300, 0), (8, 2, 128, 7, 33, 0, 1), (12, 4, 96, 200, 0, 300, 0), (16, 2, 64, 3, 16, 5, 4), (4, 4, 32, 64, 1, 300, 0),
                                                        (8, 1, 256, 25, 0, 300, 8)])
def test_batches(pkg, H, G, hs, n, window, max_len, pad):
    """Ragged batches with rows that see nothing and padding rows, queries cut out of padded rows; a hint that is wrong costs nothing but time."""
    g, slots, context = gen(n), 5, 300
    cache, k, v, d = filled(pkg, slots, context, G, hs, n + hs)
    q = (rand(g, n, H * hs + pad) * 2)[:, pad:].view(n, H, hs)
    pos = torch.randint(0, context, (n,), generator=g, device="cuda").int()
    at = torch.randint(0, slots, (n,), generator=g, device="cuda").int()
    pos[1], at[2] = -1, slots
    if n > 3:
        pos[3], at[n - 1], pos[n - 2] = context, -1, -300
    out = torch.full((n, H, hs), 7.5, device="cuda")
    cache.attention(q, pos, slots=at, window=window, max_len=max_len, out=out)
    padding = (at < 0) | (at >= slots) | (pos >= context)
    assert (out[padding] == 7.5).all() and (out[(pos < 0) & ~padding] == 0).all()
    live = ~padding
    check(out[live], q[live], k, v, d, pos[live], at[live], U.rsqrt(hs), window)


@pytest.mark.parametrize("chunk,dtype", [(1, F32), (9, F32), (21, F32)])
def test_what_lies_behind_the_mask_is_not_read(pkg, chunk, dtype):
    """Positions in front of the window and behind the row hold NaN and infinities."""
    H, G, hs, context = 4, 2, 64, 96
    cache, k, v, d = filled(pkg, 1, context, G, hs, 8)
    bad = torch.full((context, G, hs), float("nan"), device="cuda")
    at = torch.arange(context, device="cuda", dtype=torch.int32)
    hidden = (at < 20) | (at > 60)
    cache.append(bad[hidden], bad[hidden] * -1, at[hidden])
    q, pos = rand(gen(2), 21, H, hs), torch.arange(40, 61, device="cuda", dtype=torch.int32)
    for i in range(0, 21, chunk):
        rows = slice(i, i + chunk)
        got = cache.attention(q[rows], pos[rows], window=21, chunk=chunk, dtype=dtype)
        check(got, q[rows], k, v, d, pos[rows], torch.zeros_like(pos[rows]), U.rsqrt(hs), 21)
    assert torch.isnan(cache.attention(q[:1], ints(61))).all()  # a row that sees one is NaN


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1.0, 1e6, 1e30])
def test_queries_and_values_of_any_size(pkg, size):
    """No power of two in the queries, and none of FP16's range in the values, costs accuracy."""
    H, G, hs, context = 8, 2, 64, 200
    g = gen(4)
    cache = pkg.KV4Cache(1, context, G, hs)
    k, v = rand(g, context, G, hs), rand(g, context, G, hs) * (size if 1e-5 < size < 1e5 else 100.0 if size > 1 else 1e-3)
    at = torch.arange(context, device="cuda", dtype=torch.int32)
    cache.append(k, v, at)
    (kk, kd), (vv, vd) = U.quantize(k), U.quantize(v)
    q, scale = rand(g, 3, H, hs) * size, 0.125 / size
    got = cache.attention(q, ints(199, 100, 3), scale=scale)
    check(got, q, kk[None], vv[None], (kd[None], vd[None]), ints(199, 100, 3), ints(0, 0, 0), scale, 0)


def test_large_scores_and_growing_maxima(pkg):
    """Scores of hundreds that grow towards the end: every record moves the running maximum; and ones that fall, where the first holds all."""
    H, G, hs, context = 4, 1, 64, 400
    g = gen(6)
    for order in (1, -1):
        cache = pkg.KV4Cache(1, context, G, hs)
        q = rand(g, 1, H, hs)
        k = (torch.linspace(0, 300, context, device="cuda")[::1].flip(0) if order < 0 else torch.linspace(0, 300, context, device="cuda"))[:, None, None] * q[0, :1] / (q[0, 0] @ q[0, 0])
        v = rand(g, context, G, hs)
        at = torch.arange(context, device="cuda", dtype=torch.int32)
        cache.append(k, v, at)
        (kk, kd), (vv, vd) = U.quantize(k), U.quantize(v)
        got = cache.attention(q, ints(context - 1), scale=1.0)
        check(got, q, kk[None], vv[None], (kd[None], vd[None]), ints(context - 1), ints(0), 1.0, 0)


@pytest.mark.parametrize("H,G,hs", [(4, 1, 64), (8, 2, 128), (3, 1, 32), (2, 1, 96)])
def test_long_rows_shared_by_many_blocks(pkg, H, G, hs):
    """Few rows over many positions: parts go through a workspace; with and without it the same to FP32's rounding.  One row is empty, one is padding."""
    context = 30011
    cache, k, v, d = filled(pkg, 1, context, G, hs, hs)
    q = rand(gen(hs), 4, H, hs)
    pos, slots = ints(context - 1, -1, 777, 5), ints(0, 0, 0, 9)
    out = torch.full((4, H, hs), 7.5, device="cuda")
    cache.attention(q, pos, slots=slots, out=out)
    assert (out[3] == 7.5).all() and (out[1] == 0).all()
    check(out[:3], q[:3], k, v, d, pos[:3], slots[:3], U.rsqrt(hs), 0)
    L, a, one = pkg.native.lib(), pkg.native.KV4Attention(), q[:1].contiguous()
    raw, err = C.c_void_p(), C.create_string_buffer(256)
    assert L.b200_kv4_create(1, context, G, hs, 0, C.byref(raw), err, 256) == 0
    a.n, a.heads, a.q, a.q_stride, a.out_stride, a.start, a.scale = 1, H, one.data_ptr(), H * hs, H * hs, context - 1, 1.0
    need = L.b200_kv4_attention_workspace(raw, C.byref(a))
    assert need > 0 and need % (H * (hs + 2) * 4) == 0
    b = pkg.native.KV4Append()
    rows = torch.randn(context, 2, G, hs, device="cuda", generator=gen(1))
    b.n, b.k, b.v, b.k_stride, b.v_stride = context, rows.data_ptr(), rows[:, 1].data_ptr(), 2 * G * hs, 2 * G * hs
    assert L.b200_kv4_append(raw, C.byref(b), None) == 0
    outs = []
    for size in (need, need - 4, 0):  # too small a workspace is not used
        work, out = torch.full((need // 4 + 1,), float("nan"), device="cuda"), torch.empty(H * hs, device="cuda")
        a.out, a.workspace, a.workspace_bytes = out.data_ptr(), work.data_ptr(), size
        torch.cuda.synchronize()
        assert L.b200_kv4_attention(raw, C.byref(a), None) == 0
        torch.cuda.synchronize()
        assert torch.isnan(work[-1]) and (size == need or torch.isnan(work).all())
        outs.append(out)
    assert (outs[0] - outs[1]).abs().max() <= 1e-5 * outs[1].abs().max() and torch.equal(outs[1], outs[2])
    L.b200_kv4_free(raw)


def test_offsets_behind_four_gigabytes(pkg):
    """A slot that begins more than 2^32 bytes into the cache."""
    G, hs, context = 4, 128, 1 << 18
    slots = (1 << 32) // (context // 16 * 18 * hs * G) + 2
    cache = pkg.KV4Cache(slots, context, G, hs)
    assert cache.device_bytes > 1 << 32
    g, n = gen(3), 50
    k, v, q = rand(g, n, G, hs), rand(g, n, G, hs), rand(g, 1, 8, hs)
    pos = torch.arange(context - n, context, device="cuda", dtype=torch.int32)
    cache.append(k, v, pos, slots=torch.full_like(pos, slots - 1))
    (kk, kd), (vv, vd) = U.quantize(k), U.quantize(v)
    got = cache.attention(q, ints(context - 1), slots=ints(slots - 1), window=n)
    assert torch.equal(cache.read(pos, slots=torch.full_like(pos, slots - 1))[0].double().cpu(), kk)
    want, bound = U.attention(q.double().cpu(), kk[None], vv[None], (kd[None], vd[None]), [n - 1], [0], U.rsqrt(hs), 0)
    assert ((got.double().cpu() - want).abs() <= bound).all()


# ---- streams, graphs, a run of steps --------------------------------------------------------------------------------------------------
def test_captured_and_replayed(pkg):
    """One captured step (append, attention) serves every position: the graph reads positions from device memory.  Two graphs of one cache run side by side."""
    H, G, hs, context = 8, 2, 64, 200
    g = gen(9)
    cache = pkg.KV4Cache(2, context, G, hs)
    k, v = rand(g, 2, context, G, hs), rand(g, 2, context, G, hs)
    q = rand(g, 2, context, H, hs)
    side = [dict(k=k[s, :1].clone(), v=v[s, :1].clone(), q=q[s, :1].clone(), pos=ints(0), slot=ints(s), stream=torch.cuda.Stream()) for s in range(2)]
    for d in side:
        d["stream"].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(d["stream"]):
            for _ in range(2):  # the first call is not the captured one
                d["out"] = cache.attention(cache.append(d["k"], d["v"], d["pos"], q=d["q"], slots=d["slot"]), d["pos"], slots=d["slot"])
        torch.cuda.synchronize()
        d["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(d["graph"], stream=d["stream"]):
            d["out"] = cache.attention(cache.append(d["k"], d["v"], d["pos"], q=d["q"], slots=d["slot"]), d["pos"], slots=d["slot"])
    outs = [[], []]
    for i in range(context):
        for s, d in enumerate(side):
            with torch.cuda.stream(d["stream"]):
                d["k"].copy_(k[s, i:i + 1]); d["v"].copy_(v[s, i:i + 1]); d["q"].copy_(q[s, i:i + 1]); d["pos"].fill_(i)
                d["graph"].replay()
                outs[s].append(d["out"].clone())
    torch.cuda.synchronize()
    (kk, kd), (vv, vd) = U.quantize(k), U.quantize(v)
    for s in range(2):
        pos = torch.arange(context, dtype=torch.int32)
        check(torch.cat(outs[s]), q[s], kk, vv, (kd, vd), pos, torch.full_like(pos, s), U.rsqrt(hs), 0)


def test_results_do_not_depend_on_the_batch_or_the_time(pkg):
    """The same rows give the same bits again, and on another stream while others run."""
    cache, _, _, _ = filled(pkg, 3, 500, 2, 128, 11)
    q = rand(gen(1), 30, 8, 128)
    pos, slots = torch.randint(0, 500, (30,), generator=gen(2), device="cuda").int(), torch.arange(30, device="cuda", dtype=torch.int32) % 3
    first = cache.attention(q, pos, slots=slots)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs += [cache.attention(q, pos, slots=slots) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)


def test_no_rows(pkg):
    cache = pkg.KV4Cache(1, 16, 2, 64)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert cache.append(torch.empty(0, 2, 64, device="cuda"), torch.empty(0, 2, 64, device="cuda"), none, q=torch.empty(0, 4, 64, device="cuda")).shape == (0, 4, 64)
    assert cache.attention(torch.empty(0, 4, 64, device="cuda"), none).shape == (0, 4, 64)
    assert cache.read(none)[0].shape == (0, 2, 64)


def test_refusals(pkg):
    cache = pkg.KV4Cache(2, 16, 2, 64)
    k, q, pos = torch.zeros(3, 2, 64, device="cuda"), torch.zeros(3, 4, 64, device="cuda"), ints(0, 1, 2)
    cos, sin = (t.cuda() for t in U.tables(16, 64))
    bad = [lambda: cache.append(k, k.half(), pos), lambda: cache.append(k.double(), k.double(), pos), lambda: cache.append(k, k[:2], pos), lambda: cache.append(k, k, pos[:2]),
           lambda: cache.append(k, k, pos.long()), lambda: cache.append(k, k, pos.cpu()), lambda: cache.append(k.cpu(), k.cpu(), pos), lambda: cache.append(k, k, pos, q=q[..., :32]),
           lambda: cache.append(k, k, pos, q=q.half()), lambda: cache.append(k, k, pos, cos=cos), lambda: cache.append(k, k, pos, cos=cos[:8], sin=sin[:8]),
           lambda: cache.append(k, k, pos, layout="quarter"), lambda: cache.append(k, k, pos, q_norm=cos[0]), lambda: cache.append(k, k, None),
           lambda: cache.append(k.transpose(0, 1).contiguous().transpose(0, 1), k, pos), lambda: cache.attention(q[:, :3], pos), lambda: cache.attention(q.half(), pos),
           lambda: cache.attention(q, pos, dtype=torch.int32), lambda: cache.attention(q, pos, slots=pos[:1]), lambda: cache.attention(q, None), lambda: cache.read(pos, dtype=torch.int8)]
    for f in bad:
        with pytest.raises((ValueError, TypeError)):
            f()
    for kw in (dict(window=-1), dict(max_len=-1), dict(chunk=-1)):
        with pytest.raises(ValueError):
            cache.attention(q, pos, **kw)
    L, a = pkg.native.lib(), pkg.native.KV4Attention()
    a.n, a.heads, a.q, a.out, a.q_stride, a.out_stride, a.start, a.slot = 1, 4, q.data_ptr(), q.data_ptr(), 255, 256, 0, 0
    raw, err = C.c_void_p(), C.create_string_buffer(256)
    assert L.b200_kv4_create(2, 16, 2, 64, 0, C.byref(raw), err, 256) == 0
    assert L.b200_kv4_attention(raw, C.byref(a), None) == -1 and b"stride" in L.b200_kv4_last_error(raw)
    a.q_stride, a.start = 256, 16
    assert L.b200_kv4_attention(raw, C.byref(a), None) == -1 and b"positions" in L.b200_kv4_last_error(raw)
    a.start, a.slot = 15, 2
    assert L.b200_kv4_attention(raw, C.byref(a), None) == -1 and b"slot" in L.b200_kv4_last_error(raw)
    a.slot, a.window = 0, -1
    assert L.b200_kv4_attention(raw, C.byref(a), None) == -1 and b"negative" in L.b200_kv4_last_error(raw)
    a.window, a.heads = 0, 3
    assert L.b200_kv4_attention(raw, C.byref(a), None) == -1 and b"heads" in L.b200_kv4_last_error(raw)
    L.b200_kv4_free(raw)


@pytest.mark.parametrize("H,G,hs,n", [(16, 8, 64, 64), (32, 16, 128, 40), (16, 8, 32, 63)])
def test_batches_in_the_order_of_their_lengths(pkg, H, G, hs, n):
    """Enough rows for the order by length: equal lengths, padding, rows that see nothing, a window that makes most rows alike; the bits of every row are those it has alone in its batch's cut."""
    slots, context = 5, 300
    cache, k, v, d = filled(pkg, slots, context, G, hs, n)
    g = gen(n)
    q = rand(g, n, H, hs)
    pos, at = torch.randint(-3, context, (n,), device="cuda", generator=g, dtype=torch.int32), (torch.arange(n, device="cuda") % slots).int()
    pos[::7], pos[5], at[6] = 200, context, slots
    for window in (0, 31):
        out = torch.full((n, H, hs), 9.0, device="cuda")
        cache.attention(q, pos, slots=at, window=window, out=out)
        padding = (at >= slots) | (pos >= context)
        assert (out[padding] == 9).all() and (out[(pos < 0) & ~padding] == 0).all()
        live = ~padding
        want, bound = U.attention(q[live].double().cpu(), k, v, d, pos[live].cpu(), at[live].cpu(), U.rsqrt(hs), window)
        assert ((out[live].double().cpu() - want).abs() <= bound + want.abs() * U.half_step(F32)).all()
        turned = torch.arange(n - 1, -1, -1, device="cuda")
        again = cache.attention(q[turned], pos[turned], slots=at[turned], window=window)
        assert torch.equal(again[turned][live], out[live])
