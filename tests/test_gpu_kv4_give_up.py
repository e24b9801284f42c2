"""A wait of a chunk's attention that runs out is heard of, whichever warp it was; no cache is made without the word that says so."""
import ctypes as C

import pytest
import torch

from test_gpu_kv4 import filled, gen, ints, rand

pytestmark = pytest.mark.gpu


def raw_cache(pkg, slots, context, G, hs):
    raw, err = C.c_void_p(), C.create_string_buffer(256)
    return pkg.native.lib().b200_kv4_create(slots, context, G, hs, 0, C.byref(raw), err, 256), raw, err


@pytest.mark.parametrize("context,n", [(128, 64), (100, 70), (640, 64), (6000, 40)])  # a tile; two blocks of rows; several tiles; parts through a workspace
def test_rows_that_give_up_their_last_wait(pkg, context, n):
    """The products are issued, and the warp that issues them has left: the call's rows stay as they were, the next call says so, and other caches and kernels go on."""
    H, G, hs = 2, 1, 64
    other, _, _, _ = filled(pkg, 1, 200, G, hs, 3)
    q = rand(gen(n), n, H, hs)
    p2 = torch.arange(100, 100 + n, device="cuda", dtype=torch.int32)
    before = other.attention(q, p2, chunk=n, dtype=torch.float16)
    lib = pkg.native.lib()
    rc, raw, _ = raw_cache(pkg, 1, context, G, hs)
    assert rc == 0
    rows = rand(gen(1), context, 2, G, hs)
    b = pkg.native.KV4Append()
    b.n, b.k, b.v, b.k_stride, b.v_stride = context, rows.data_ptr(), rows[:, 1].data_ptr(), 2 * G * hs, 2 * G * hs
    assert lib.b200_kv4_append(raw, C.byref(b), None) == 0
    out = torch.full((n, H, hs), 7.5, device="cuda", dtype=torch.float16)
    a = pkg.native.KV4Attention()
    a.n, a.heads, a.q, a.out, a.q_stride, a.out_stride, a.start, a.scale, a.chunk, a.out_type = n, H, q.data_ptr(), out.data_ptr(), H * hs, H * hs, context - n, 0.125, n, 1
    work = torch.zeros(max(4, lib.b200_kv4_attention_workspace(raw, C.byref(a)) // 4), device="cuda")
    a.workspace, a.workspace_bytes = work.data_ptr(), 4 * work.numel()
    assert lib.b200_kv4_attention(raw, C.byref(a), None) == 0
    torch.cuda.synchronize()
    right = out.clone()
    assert not (out == 7.5).any()
    out.fill_(7.5)
    torch.cuda.synchronize()
    assert lib.b200_test_kv4_give_up(raw, C.byref(a), None) == 0
    torch.cuda.synchronize()
    if context < 6000:  # (else the join has put together what it found)
        assert (out == 7.5).all()
    assert lib.b200_kv4_attention(raw, C.byref(a), None) == -6 and b"gave up" in lib.b200_kv4_last_error(raw)
    lib.b200_kv4_reset(raw, None)
    torch.cuda.synchronize()
    assert lib.b200_kv4_attention(raw, C.byref(a), None) == -6  # a reset does not take it back
    lib.b200_kv4_free(raw)
    assert torch.equal(other.attention(q, p2, chunk=n, dtype=torch.float16), before)
    rc, raw, _ = raw_cache(pkg, 1, context, G, hs)  # tensor memory and barriers are as they should be
    assert rc == 0 and lib.b200_kv4_append(raw, C.byref(b), None) == 0 and lib.b200_kv4_attention(raw, C.byref(a), None) == 0
    torch.cuda.synchronize()
    assert torch.equal(out, right)
    lib.b200_kv4_free(raw)


def test_refusals_of_the_hook(pkg):
    rc, raw, _ = raw_cache(pkg, 1, 64, 1, 128)
    a, lib = pkg.native.KV4Attention(), pkg.native.lib()
    a.n, a.heads, a.chunk, a.out_type = 64, 1, 64, 1
    assert rc == 0 and lib.b200_test_kv4_give_up(raw, C.byref(a), None) == -1 and lib.b200_test_kv4_give_up(None, C.byref(a), None) == -1
    lib.b200_kv4_free(raw)


def test_no_cache_without_the_word(pkg, monkeypatch):
    monkeypatch.setenv("B200_TEST_REFUSE", "kv4_word")
    rc, raw, err = raw_cache(pkg, 1, 64, 1, 64)
    assert rc != 0 and raw.value is None and b"memory" in err.value
    with pytest.raises(pkg.native.B200Error):
        pkg.KV4Cache(1, 64, 1, 64)
    monkeypatch.delenv("B200_TEST_REFUSE")
    rc, raw, _ = raw_cache(pkg, 1, 64, 1, 64)
    assert rc == 0
    pkg.native.lib().b200_kv4_free(raw)
    assert (pkg.KV4Cache(1, 64, 1, 64).read(ints(0))[0] == 0).all()
