"""Calls on pages that are refused for what their results would be, without a GPU."""
import ctypes as C
import math

import pytest

from test_paged_host import cache_of


def attention_of(pkg, **kw):
    a = pkg.native.PagedAttention()
    for k, v in dict(dict(n=3, heads=4, out_type=0, q=1 << 20, out=1 << 21, q_stride=256, out_stride=256, positions=256, sequences=256, tables=256, table_stride=5, n_sequences=2, table_width=5, scale=1.0), **kw).items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("n", [0, 3])
def test_scales_that_are_no_numbers(pkg, scale, n):
    """A NaN would count as a scale near 0: a finite mean of everything."""
    L, err = pkg.native.lib(), C.create_string_buffer(256)
    assert L.b200_paged_attention(C.byref(cache_of(pkg)), C.byref(attention_of(pkg, scale=scale, n=n)), None, err, 256) == -1 and b"scale" in err.value


BASE = 1 << 20


def append_of(pkg, **kw):
    a = pkg.native.PagedAppend()
    wide = (4 + 2 + 2) * 64  # FP32 rows of a QKV product
    for k, v in dict(dict(n=3, heads=4, type=0, rope_layout=1, q=BASE, k=BASE + 4 * 64 * 4, v=BASE + 6 * 64 * 4, q_stride=wide, k_stride=wide, v_stride=wide, q_out_stride=256, positions=256, sequences=256, tables=256,
                          table_stride=5, n_sequences=2, table_width=5, q_out=2 * BASE), **kw).items():
        setattr(a, k, v)
    return a


END = BASE + 3 * 512 * 4
POOL = 4 * 2 * 16 * 64 * 2  # of cache_of, bytes


@pytest.mark.parametrize("kw", [dict(q_out=BASE), dict(q_out=BASE + 16), dict(q_out=BASE + 4 * 64 * 4), dict(q_out=BASE + 6 * 64 * 4), dict(q_out=END - 2), dict(q_out=BASE - 3 * 512 + 2), dict(q_out=BASE + 2, q_out_stride=1024),
                                dict(q_out=1 << 24), dict(q_out=(1 << 24) + POOL - 2), dict(q_out=(1 << 25) + 64), dict(n=1, q_out=BASE + 6 * 64 * 4 + 510)])
def test_append_refuses_results_over_its_inputs(pkg, kw):
    L, err = pkg.native.lib(), C.create_string_buffer(256)
    cache = cache_of(pkg, keys=1 << 24, values=1 << 25)
    assert L.b200_paged_append(C.byref(cache), C.byref(append_of(pkg, **kw)), None, err, 256) == -1 and b"overlap" in err.value


@pytest.mark.parametrize("kw", [dict(out=BASE + 2), dict(out=BASE - 2), dict(out_type=0, out=BASE), dict(out=BASE, out_stride=512), dict(out=BASE + 2 * 256 * 2), dict(n=1, out=BASE + 510), dict(q_stride=512, out_stride=512, out=BASE + 500),
                                dict(out=1 << 24), dict(out=(1 << 25) + POOL - 2)])
def test_attention_refuses_results_over_its_inputs(pkg, kw):
    L, err = pkg.native.lib(), C.create_string_buffer(256)
    cache = cache_of(pkg, keys=1 << 24, values=1 << 25)
    a = attention_of(pkg, **dict(dict(q=BASE, out_type=1), **kw))
    assert L.b200_paged_attention(C.byref(cache), C.byref(a), None, err, 256) == -1 and b"overlap" in err.value


@pytest.mark.parametrize("kw", [dict(out_tokens=BASE), dict(out_tokens=BASE - 20), dict(out_tokens=BASE + 12), dict(accepted=BASE + 4), dict(accepted=2 * BASE + 20), dict(accepted=2 * BASE - 4)])
def test_verification_refuses_results_over_its_drafts(pkg, kw):
    """Two sequences of two drafts: 16 bytes of drafts, 24 of tokens, 8 of counts."""
    L, err, a = pkg.native.lib(), C.create_string_buffer(256), pkg.native.VerifyDrafts()
    for k, v in dict(dict(logits=256, sequence_stride=24, row_stride=8, sequences=2, drafts=2, vocab=8, temperature=1.0, tokens=BASE, uniforms=256, out_tokens=2 * BASE, accepted=3 * BASE, workspace=4 * BASE,
                          workspace_bytes=1 << 16), **kw).items():
        setattr(a, k, v)
    assert L.b200_verify_drafts(C.byref(a), None, err, 256) == -1 and b"overlap" in err.value
