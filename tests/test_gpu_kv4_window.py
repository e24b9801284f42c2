"""Windows of the largest number: 'no limit' for whoever passes one."""
import ctypes as C

import pytest
import torch

from test_gpu_kv4 import F16, F32, filled, gen, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("chunk", [1, 40])
def test_a_window_of_the_largest_number_is_none(pkg, chunk):
    """The same cut (the workspace shows it) and the same bits as without a window."""
    H, G, hs, context, n = 4, 1, 128, 12000, 40
    cache, _, _, _ = filled(pkg, 1, context, G, hs, 2)
    raw, err = C.c_void_p(), C.create_string_buffer(256)
    lib, a = pkg.native.lib(), pkg.native.KV4Attention()
    assert lib.b200_kv4_create(1, context, G, hs, 0, C.byref(raw), err, 256) == 0
    need = []
    a.n, a.heads, a.out_type, a.chunk = n if chunk > 1 else 1, H, 1, chunk
    for a.window in (0, 2**31 - 1, 2**31 - 20, context):
        need.append(lib.b200_kv4_attention_workspace(raw, C.byref(a)))
    lib.b200_kv4_free(raw)
    assert need[0] > 0 and need == need[:1] * 4
    q = rand(gen(1), a.n, H, hs)
    pos = torch.arange(context - a.n, context, device="cuda", dtype=torch.int32)
    for dtype in (F16, F32):
        assert torch.equal(cache.attention(q, pos, chunk=chunk, dtype=dtype), cache.attention(q, pos, chunk=chunk, dtype=dtype, window=2**40))
