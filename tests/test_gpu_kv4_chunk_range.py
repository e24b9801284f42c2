"""Chunks over everything that the 4-bit cache holds: entries outside FP16 in keys and values, groups of NaN."""
import pytest
import torch

import kv4_util as U
from test_gpu_kv4 import BF16, F16, filled, gen, ints, rand

pytestmark = pytest.mark.gpu


def stored(pkg, context, G, hs, seed, wide_k=(), wide_v=(), nan_v=()):
    """A cache whose keys / values at (position, entry, value) are outside FP16, with values of NaN in the groups (position, group): (cache, k, v, (scales of both)) as the cache holds them."""
    g = gen(seed)
    cache = pkg.KV4Cache(1, context, G, hs)
    k, v = rand(g, context, G, hs), rand(g, context, G, hs) * 0.5
    for at, entry, value in wide_k:
        k[at, :, entry] = value
    for at, entry, value in wide_v:
        v[at, :, entry] = value
    for at, group in nan_v:
        v[at, :, group * 32 + 5] = float("nan")
    every = torch.arange(context, device="cuda", dtype=torch.int32)
    cache.append(k, v, every)
    (kk, kd), (vv, vd) = U.quantize(k), U.quantize(v)
    return cache, kk[None], vv[None], (kd[None], vd[None])


def check(got, q, k, v, d, pos, scale, window, dtype):
    """test_gpu_kv4_chunk.check, with infinities where the result's type has no number for the right one.

    Scaling by 2^5 and back is exact; entries of the same position below 2^-9 of FP16's smallest normal scale lose bits, at most 2^-20 each, far below the bound's share of an entry of 2^16."""
    qq, pos, slots = q.double().cpu(), pos.cpu(), torch.zeros(len(pos), dtype=torch.int32)
    want, _ = U.attention(qq, k, v, d, pos, slots, scale, window)
    bound = U.chunk_bound(qq, k, v, pos, slots, scale, window, want, dtype)
    got = got.double().cpu()
    top = torch.finfo(dtype).max
    over = want.abs() - bound > top * (1 + torch.finfo(dtype).eps)
    assert torch.isinf(got[over]).all() and (torch.sign(got) == torch.sign(want))[over].all()
    near = ~over & (want.abs() + bound >= top)
    ok = ((got - want).abs() <= bound) | (near & torch.isinf(got))
    assert ok[~over].all(), ((got - want).abs() / bound)[~over].max()


WIDE = [(0, 0, 70000.0), (15, 40, -1e5), (16, 63, 3e5), (130, 1, -524032.0), (131, 2, 65535.0), (255, 33, 1e30), (300, 31, -66000.0), (399, 5, 9e4)]


@pytest.mark.parametrize("H,G,hs", [(4, 2, 64), (8, 2, 128), (6, 2, 96)])
@pytest.mark.parametrize("window", [0, 70])
def test_keys_outside_fp16(pkg, H, G, hs, window):
    """Keys of up to 524032, met by query entries that make scores of ordinary size of them, of either sign: single rows and chunks agree with the formula."""
    context, n = 400, 130
    cache, k, v, d = stored(pkg, context, G, hs, hs, wide_k=WIDE)
    q = rand(gen(1), n, H, hs)
    for _, entry, value in WIDE:
        q[:, :, entry] = q[:, :, entry] * 20 / min(abs(value), 524032.0)
    pos = torch.arange(context - n, context, device="cuda", dtype=torch.int32)
    for dtype in (F16, BF16):
        check(cache.attention(q, pos, window=window, chunk=n, dtype=dtype), q, k, v, d, pos, U.rsqrt(hs), window, dtype)


def test_a_key_outside_fp16_keeps_its_weight(pkg):
    """Two positions; the second one's key has the entry 70000 against a query's -1e-5: a score of -0.06, not minus infinity."""
    hs, n = 64, 64
    cache = pkg.KV4Cache(1, 16, 1, hs)
    k, v = torch.zeros(2, 1, hs, device="cuda"), torch.zeros(2, 1, hs, device="cuda")
    k[1, 0, 3], v[1] = 70000.0, 8.0
    cache.append(k, v, ints(0, 1))
    q = torch.zeros(n, 1, hs, device="cuda")
    q[..., 3] = torch.linspace(-2e-5, 2e-5, n, device="cuda")[:, None]
    pos = torch.ones(n, device="cuda", dtype=torch.int32)
    got = cache.attention(q, pos, chunk=n, dtype=F16)
    held = cache.read(ints(1))[0][0, 0, 3].double()
    want = 8 * torch.sigmoid(q[..., 3].double() * held / 8)
    assert ((got[:, 0, 0].double() - want[:, 0]).abs() <= want[:, 0] * 2.0 ** -9).all()  # scores of at most 0.18 (2^-10 of them), P, V and the result 2^-11 each


@pytest.mark.parametrize("H,G,hs", [(4, 2, 64), (8, 2, 128), (6, 2, 96)])
@pytest.mark.parametrize("window", [0, 70])
def test_values_outside_fp16(pkg, H, G, hs, window):
    context, n = 400, 130
    cache, k, v, d = stored(pkg, context, G, hs, hs + 1, wide_v=WIDE)
    q = rand(gen(2), n, H, hs)
    pos = torch.arange(context - n, context, device="cuda", dtype=torch.int32)
    for dtype in (F16, BF16):
        check(cache.attention(q, pos, window=window, chunk=n, dtype=dtype), q, k, v, d, pos, U.rsqrt(hs), window, dtype)


@pytest.mark.parametrize("context", [400, 12000])
def test_a_group_of_nan_reaches_its_entries_alone(pkg, context):
    """As in single rows: of a row that sees a value's NaN the entries of that group are NaN and the others right; with 12000 positions the parts go through a workspace."""
    H, G, hs, n = 8, 2, 128, 80
    nan_v = [(context - 60, 1), (context - 30, 3), (context - 2, 0), (17, 2)]
    window = 200 if context == 400 else 0
    cache, k, v, d = stored(pkg, context, G, hs, 5, nan_v=nan_v, wide_k=[(context - 90, 7, 1e5)], wide_v=[(context - 30, 2, 7e4), (context - 61, 70, -7e4)])
    q = rand(gen(3), n, H, hs)
    q[:, :, 7] *= 1e-4
    pos = torch.arange(context - n, context, device="cuda", dtype=torch.int32)
    got = cache.attention(q, pos, window=window, chunk=n, dtype=BF16)
    sees = torch.zeros(n, 4, dtype=torch.bool)
    for at, group in nan_v:
        sees[:, group] |= ((at <= pos) & ((at > pos - window) if window else True)).cpu()
    bad = sees[:, None, :].expand(n, H, 4).repeat_interleave(32, -1)
    assert torch.isnan(got.cpu())[bad].all() and not torch.isnan(got.cpu())[~bad].any() and bad.any() and (~bad).any()
    assert torch.equal(torch.isnan(cache.attention(q[:3], pos[:3], window=window)).cpu(), bad[:3])
    fine = got.clone()
    fine[bad.cuda()] = 0
    v = torch.nan_to_num(v)
    want, _ = U.attention(q.double().cpu(), k, v, [torch.nan_to_num(s) for s in d], pos.cpu(), torch.zeros(n, dtype=torch.int32), U.rsqrt(hs), window)
    bound = U.chunk_bound(q.double().cpu(), k, v, pos.cpu(), torch.zeros(n, dtype=torch.int32), U.rsqrt(hs), window, want, BF16)
    assert ((fine.double().cpu() - want).abs() <= bound)[~bad].all()


def test_entries_outside_fp16_beside_padding_and_other_sequences(pkg):
    """Keys and values outside FP16 in one slot: the other slot's rows of the same tile, rows without keys and padding do not notice."""
    H, G, hs, context = 4, 1, 64, 300
    cache, k, v, d = filled(pkg, 2, context, G, hs, 4)
    k2, v2 = torch.full((10, G, hs), 2e5, device="cuda"), torch.full((10, G, hs), -3e5, device="cuda")
    cache.append(k2, v2, torch.arange(100, 110, device="cuda", dtype=torch.int32), slots=torch.ones(10, device="cuda", dtype=torch.int32))
    n = 120
    q = rand(gen(8), n, H, hs)
    pos = torch.arange(150, 150 + n, device="cuda", dtype=torch.int32) % 290
    at = (torch.arange(n, device="cuda") // 30 % 2).int()
    pos[7], at[9] = -1, 5
    out = torch.full((n, H, hs), 7.5, device="cuda", dtype=BF16)
    cache.attention(q, pos, slots=at, chunk=n, out=out)
    assert (out[9] == 7.5).all() and (out[7] == 0).all()
    live = (at == 0) & (pos >= 0)
    check(out[live], q[live], k[:1], v[:1], (d[0][:1], d[1][:1]), pos[live], U.rsqrt(hs), 0, BF16)


@pytest.mark.parametrize("hs", [64, 128])
def test_rows_of_the_lowest_position_see_nothing(pkg, hs):
    """A row of a negative position has no keys, be it -1 or the lowest number, also beside rows that see NaN and infinities: zeros."""
    H, G, context, n = 4, 1, 300, 128
    cache, _, _, _ = filled(pkg, 1, context, G, hs, 4)
    at = ints(3, 150, 290)
    odd = torch.full((3, G, hs), float("nan"), device="cuda")
    cache.append(odd, odd, at)
    q = rand(gen(1), n, H, hs)
    pos = torch.arange(context - n, context, device="cuda", dtype=torch.int32)
    pos[::5], pos[1::5], pos[2::5], pos[3::5] = -2**31, -1, -2**31 + 300, -300
    for window in (0, 50):
        got = cache.attention(q, pos, window=window, chunk=n, dtype=BF16)
        assert (got[pos < 0] == 0).all()
        assert torch.equal(torch.isnan(got), torch.isnan(cache.attention(q, pos, window=window, dtype=BF16)))
