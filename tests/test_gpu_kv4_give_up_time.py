"""A wait of a chunk's attention that cannot end is given up after seconds, not minutes."""
import ctypes as C
import time

import pytest
import torch

from test_gpu_kv4 import gen, rand
from test_gpu_kv4_give_up import raw_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [64, 3000])  # a block of rows; more of them than run at a time: the later ones do not wait as long again
def test_a_wait_ends_after_two_seconds(pkg, n):
    H, G, hs, context = 8, 2, 64, 4096
    lib = pkg.native.lib()
    rc, raw, _ = raw_cache(pkg, 1, context, G, hs)
    assert rc == 0
    q, out = rand(gen(n), n, H, hs), torch.full((n, H, hs), 7.5, device="cuda", dtype=torch.float16)
    a = pkg.native.KV4Attention()
    a.n, a.heads, a.q, a.out, a.q_stride, a.out_stride, a.start, a.scale, a.chunk, a.out_type = n, H, q.data_ptr(), out.data_ptr(), H * hs, H * hs, 0, 0.125, n, 1
    torch.cuda.synchronize()
    begin = time.perf_counter()
    assert lib.b200_test_kv4_give_up(raw, C.byref(a), None) == 0
    torch.cuda.synchronize()
    seconds = time.perf_counter() - begin
    assert 1.5 < seconds < 3.5  # 3.5e9 cycles at 1.0 to 2.3 GHz
    assert lib.b200_kv4_attention(raw, C.byref(a), None) == -6 and (out == 7.5).all()
    lib.b200_kv4_free(raw)
