"""Refusals of the operators on pages and of the verification of drafts that need no GPU, and the plain forms that the GPU tests hold the kernels to."""
import ctypes as C

import pytest
import torch

import paged_util as P


def test_argument_blocks_have_the_headers_layout(pkg):
    assert [C.sizeof(t) for t in (pkg.native.PagedCache, pkg.native.PagedAppend, pkg.native.PagedAttention, pkg.native.VerifyDrafts)] == [40, 168, 120, 120]


def cache_of(pkg, **kw):
    c = pkg.native.PagedCache()
    for k, v in dict(dict(keys=4096, values=8192, pages=4, page_size=16, kv_heads=2, head_size=64, type=1, device=0), **kw).items():
        setattr(c, k, v)
    return c


BAD_CACHES = [(dict(type=0), -2, "type"), (dict(type=8), -2, "type"), (dict(head_size=80), -2, "80"), (dict(head_size=0), -2, "0"), (dict(pages=0), -1, "positive"), (dict(kv_heads=-1), -1, "positive"),
              (dict(page_size=0), -2, "power"), (dict(page_size=24), -2, "24"), (dict(page_size=131072), -2, "131072"), (dict(page_size=-16), -2, "power"),
              (dict(pages=2**31 - 1, kv_heads=64), -2, "2^32"), (dict(keys=4100), -1, "16-byte")]


@pytest.mark.parametrize("bad,code,word", BAD_CACHES)
def test_caches_that_are_refused(pkg, bad, code, word):
    L, err = pkg.native.lib(), C.create_string_buffer(256)
    c, a, b = cache_of(pkg, **bad), pkg.native.PagedAppend(), pkg.native.PagedAttention()
    a.rope_layout = 1
    b.heads = 2
    assert L.b200_paged_append(C.byref(c), C.byref(a), None, err, 256) == code and word in err.value.decode()
    assert L.b200_paged_attention(C.byref(c), C.byref(b), None, err, 256) == code and word in err.value.decode()


def test_append_refuses(pkg):
    L, err = pkg.native.lib(), C.create_string_buffer(256)
    good = dict(n=3, heads=4, type=0, rope_layout=1, rope_dims=64, rope_rows=10, q=256, k=256, v=256, q_stride=256, k_stride=128, v_stride=128, q_out_stride=256, positions=256, sequences=256, tables=256,
                table_stride=5, n_sequences=2, table_width=5, cos=256, sin=256, q_out=256)
    for bad, code in ((dict(n=-1), -1), (dict(heads=-1), -1), (dict(type=8), -2), (dict(rope_layout=7), -1), (dict(sin=None), -1), (dict(rope_dims=0), -1), (dict(rope_dims=66), -1), (dict(rope_dims=31), -1),
                      (dict(rope_rows=-1), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(q=None), -1), (dict(q_out=None), -1), (dict(k_stride=127), -1), (dict(q_stride=255), -1), (dict(q_out_stride=0), -1),
                      (dict(positions=None), -1), (dict(tables=None), -1), (dict(table_stride=4), -1), (dict(table_width=-1), -1), (dict(n_sequences=-1), -1),
                      (dict(table_width=2**26, table_stride=2**26), -2), (dict(heads=2**18, q_stride=2**25, q_out_stride=2**25), -2)):
        a = pkg.native.PagedAppend()
        for k, v in dict(good, **bad).items():
            setattr(a, k, v)
        assert L.b200_paged_append(C.byref(cache_of(pkg)), C.byref(a), None, err, 256) == code and err.value, bad
    assert L.b200_paged_append(None, C.byref(a), None, None, 0) == -1 and L.b200_paged_append(C.byref(cache_of(pkg)), None, None, None, 0) == -1
    a = pkg.native.PagedAppend()
    a.rope_layout = 1
    assert L.b200_paged_append(C.byref(cache_of(pkg)), C.byref(a), None, err, 256) == 0  # no rows: nothing to do


def test_attention_refuses(pkg):
    L, err = pkg.native.lib(), C.create_string_buffer(256)
    good = dict(n=3, heads=4, out_type=0, q=256, out=256, q_stride=256, out_stride=256, positions=256, sequences=256, tables=256, table_stride=5, n_sequences=2, table_width=5, scale=1.0)
    for bad, code in ((dict(n=-1), -1), (dict(heads=0), -1), (dict(heads=3), -1), (dict(out_type=8), -2), (dict(window=-1), -1), (dict(max_len=-1), -1), (dict(chunk=-1), -1), (dict(workspace=8), -1), (dict(q=None), -1),
                      (dict(out=None), -1), (dict(q_stride=255), -1), (dict(out_stride=255), -1), (dict(positions=None), -1), (dict(tables=None), -1), (dict(n=2**25 + 1), -2)):
        a = pkg.native.PagedAttention()
        for k, v in dict(good, **bad).items():
            setattr(a, k, v)
        assert L.b200_paged_attention(C.byref(cache_of(pkg)), C.byref(a), None, err, 256) == code and err.value, bad
    assert L.b200_paged_attention(None, C.byref(a), None, None, 0) == -1 and L.b200_paged_attention(C.byref(cache_of(pkg)), None, None, None, 0) == -1
    assert L.b200_paged_attention_workspace(None, None) == 0


def test_verify_refuses(pkg):
    L, err = pkg.native.lib(), C.create_string_buffer(256)
    good = dict(logits=256, draft_logits=256, sequence_stride=24, row_stride=8, draft_sequence_stride=16, draft_row_stride=8, sequences=2, drafts=2, vocab=8, temperature=1.0, tokens=256, uniforms=256,
                out_tokens=256, accepted=256, workspace=256, workspace_bytes=1 << 20)
    for bad, code in ((dict(sequences=-1), -1), (dict(drafts=-1), -1), (dict(vocab=0), -1), (dict(drafts=65), -2), (dict(vocab=2**24 + 1, row_stride=2**25), -2), (dict(sequences=2**16 + 1), -2), (dict(type=8), -2),
                      (dict(temperature=-1.0), -1), (dict(temperature=float("nan")), -1), (dict(temperature=1e-5), -1), (dict(temperature=float("inf")), -1), (dict(logits=None), -1), (dict(tokens=None), -1),
                      (dict(uniforms=None), -1), (dict(out_tokens=None), -1), (dict(accepted=None), -1), (dict(row_stride=7), -1), (dict(workspace=None), -1), (dict(workspace=8), -1), (dict(workspace_bytes=8), -1)):
        a = pkg.native.VerifyDrafts()
        for k, v in dict(good, **bad).items():
            setattr(a, k, v)
        assert L.b200_verify_drafts(C.byref(a), None, err, 256) == code and err.value, bad
    assert L.b200_verify_drafts(None, None, None, 0) == -1 and L.b200_verify_drafts_workspace(None) == 0
    a = pkg.native.VerifyDrafts()
    a.vocab, a.temperature = 8, 1.0
    assert L.b200_verify_drafts(C.byref(a), None, err, 256) == 0  # no sequences: nothing to do


def test_python_refuses_what_is_not_on_a_gpu(pkg):
    for kw in (dict(device="cpu"), dict(dtype=torch.float32), dict(dtype=torch.int8)):
        with pytest.raises(ValueError):
            pkg.PagedKVCache(4, 16, 2, 64, **kw)
    with pytest.raises(ValueError):
        pkg.PagedKVCache(0, 16, 2, 64)
    with pytest.raises(ValueError, match="GPU"):
        pkg.operators._ops.Paged(torch.zeros(4, 2, 16, 64), torch.zeros(4, 2, 16, 64))
    with pytest.raises(ValueError, match="GPU"):
        pkg.verify_drafts(torch.zeros(1, 2, 8), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 2))


def test_plain_attention_sees_pages_only():
    g = torch.Generator().manual_seed(1)
    keys, values = torch.randn(3, 1, 2, 4, generator=g), torch.randn(3, 1, 2, 4, generator=g)
    tables = torch.tensor([[2, 7, 0], [-1, -1, 1]])
    q = torch.randn(4, 1, 4, generator=g)
    out, _ = P.attention(q, keys, values, torch.tensor([4, 3, 5, -1]), torch.tensor([0, 1, 2, 0]), tables, scale=0.5)
    k, v = (torch.cat((t[2, 0], t[0, 0, :1])).double() for t in (keys, values))
    assert torch.allclose(out[0, 0], torch.softmax(q[0, 0].double() @ k.T * 0.5, -1) @ v) and (out[1:] == 0).all()


def test_plain_verification():
    x = torch.log(torch.tensor([[[0.5, 0.25, 0.25], [0.125, 0.125, 0.75]]], dtype=torch.float64))
    y = torch.log(torch.tensor([[[0.25, 0.5, 0.25]]], dtype=torch.float64))
    draft = torch.tensor([[1]], dtype=torch.int32)
    for u0, u1, want in ((0.49, 0.0, [1, 0]), (0.49, 0.2, [1, 1]), (0.49, 0.5, [1, 2]), (0.51, 0.99, [0, -1])):  # p / q = 0.5; the rest lies on token 0
        assert P.verify(x, draft, torch.tensor([[u0, u1]]), y, 1.0)[0].tolist() == [want]
    for u0, u1, want in ((0.24, 0.5, [1, 2]), (0.26, 0.6, [0, -1]), (0.26, 0.7, [2, -1])):  # looked up: p without the draft, 2 : 1
        assert P.verify(x, draft, torch.tensor([[u0, u1]]), None, 1.0)[0].tolist() == [want]
    assert P.verify(x, draft, None, None, 0)[0].tolist() == [[0, -1]] and P.verify(x, torch.tensor([[0]]), None, None, 0)[0].tolist() == [[0, 2]]
