"""The paged cache and its attention on the GPU where inputs are unusual: what padding holds, scores of any size, precision of long rows, overlapping results."""
import pytest
import torch

import paged_util as P
from test_gpu_paged import BF16, F16, F32, check, gen, ints, paged, probability, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,out", [(BF16, F32), (F16, F32), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("H,hs,slots,used", [(8, 64, 5, 3), (8, 128, 5, 3), (6, 32, 4, 1), (2, 256, 6, 5), (24, 96, 2, 1), (8, 64, 40, 17)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_padding_holds_does_not_matter(pkg, dtype, out, H, hs, slots, used, bad):
    """Draft slots that are not used (no sequence, or a position behind the table) and rows at negative positions: the other rows have the same bits whatever lies in their queries."""
    g = gen(hs + slots)
    cache, tables = paged(pkg, g, [320, 300, 310], 16, 2, hs, dtype)
    pos = torch.cat([torch.arange(n - used, n - used + slots, device="cuda") for n in (320, 300, 310)]).int()
    seq = torch.arange(3, device="cuda", dtype=torch.int32).repeat_interleave(slots)
    live = (torch.arange(slots, device="cuda") < used).repeat(3)
    kind = torch.arange(3 * slots, device="cuda") % 3
    seq[~live & (kind == 0)] = -1
    pos[~live & (kind == 1)] = 10**6
    pos[~live & (kind == 2)] = -1
    q = rand(g, 3 * slots, H, hs, dtype=dtype)
    q[~live] = 0
    want = check(cache, q, pos, tables, seq, out, chunk=slots)
    q[~live] = bad
    got = cache.attention(q, pos, tables, sequences=seq, dtype=out, chunk=slots)
    assert torch.equal(got[live], want[live]) and (got[~live & (kind == 2)] == 0).all()
