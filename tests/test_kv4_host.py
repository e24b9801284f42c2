"""Refusals of the 4-bit cache and of the log probabilities that need no GPU, the layout of their argument blocks, and the plain form that the GPU tests hold the kernels to."""
import ctypes as C

import pytest
import torch

import kv4_util as U


def test_argument_blocks_have_the_headers_layout(pkg):
    assert [C.sizeof(t) for t in (pkg.native.KV4Append, pkg.native.KV4Attention, pkg.native.KV4Read, pkg.native.LogProbs)] == [144, 104, 48, 80]


@pytest.mark.parametrize("slots,context,heads,hs,code,word", [(0, 16, 1, 64, -1, "positive"), (1, 0, 1, 64, -1, "positive"), (1, 16, 0, 64, -1, "positive"), (1, 16, 1, 80, -2, "80"),
                                                              (1, 16, 1, 512, -2, "512"), (1, 2**31 - 1, 1, 64, -1, "positive")])
def test_cache_refuses(pkg, slots, context, heads, hs, code, word):
    out, err = C.c_void_p(1), C.create_string_buffer(256)
    assert pkg.native.lib().b200_kv4_create(slots, context, heads, hs, 0, C.byref(out), err, 256) == code
    assert out.value is None and word in err.value.decode()


def test_null_arguments(pkg):
    L = pkg.native.lib()
    assert L.b200_kv4_create(1, 16, 1, 64, 0, None, None, 0) == -1
    a, r, p = pkg.native.KV4Append(), pkg.native.KV4Read(), pkg.native.LogProbs()
    assert L.b200_kv4_append(None, C.byref(a), None) == -1 and L.b200_kv4_read(None, C.byref(r), None) == -1 and L.b200_kv4_reset(None, None) == -1
    assert L.b200_kv4_attention(None, None, None) == -1 and L.b200_log_probs(None, None, None, 0) == -1
    L.b200_kv4_free(None)
    assert L.b200_kv4_device_bytes(None) == 0
    err = C.create_string_buffer(256)
    for rows, vocab, top, kind, stride, code in ((-1, 8, 0, 0, 8, -1), (1, 0, 0, 0, 8, -1), (1, 8, 33, 0, 8, -1), (1, 8, 9, 0, 8, -1), (1, 8, -1, 0, 8, -1), (1, 8, 1, 8, 8, -2), (2, 8, 1, 0, 7, -1),
                                                 (1, 8, 1, 0, 8, -1)):
        p.rows, p.vocab, p.top, p.type, p.row_stride, p.logits = rows, vocab, top, kind, stride, None if (rows, stride, kind, top) == (1, 8, 0, 1) else 256
        assert L.b200_log_probs(C.byref(p), None, err, 256) == code and err.value
    p.rows, p.vocab, p.top, p.type = 0, 8, 1, 0
    assert L.b200_log_probs(C.byref(p), None, err, 256) == 0  # no rows: nothing to do


def test_python_refuses_what_is_not_on_a_gpu(pkg):
    with pytest.raises(ValueError):
        pkg.KV4Cache(1, 16, 1, 64, device="cpu")
    with pytest.raises(ValueError):
        pkg.log_probs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(AttributeError):
        pkg.no_such_operator


def test_plain_quantisation():
    x = torch.zeros(6, 32)
    x[1, 3], x[1, 7] = 2.0, -2.0  # equal magnitudes: the first counts, d = -0.25: 2 -> -8 d, -2 -> 7 d (clamped)
    x[2, 0], x[2, 1] = -8.0, 0.5  # d = 1; 0.5 rounds to the even 0
    x[3, 0], x[3, 5] = 1.0, float("nan")
    x[4, 0] = 1e30
    x[5, 9] = 1e-9
    v, d = U.quantize(x)
    assert (v[0] == 0).all() and d[0] == 0
    assert d[1] == -0.25 and v[1, 3] == 2.0 and v[1, 7] == -1.75
    assert d[2] == 1 and v[2, 0] == -8 and v[2, 1] == 0
    assert torch.isnan(v[3]).all()
    assert v[4, 0] == 8 * 65504 and (v[4, 1:] == 0).all()
    assert (v[5] == 0).all()
    y = torch.randn(50, 64, generator=torch.Generator().manual_seed(1))
    v, d = U.quantize(y)
    step = d.abs().repeat_interleave(32, -1)
    assert ((v - y.double()).abs() <= step * (1 + 2.0 ** -10)).all() and ((v - y.double()).abs() <= step / 2 + 1e-6).float().mean() > 0.97
