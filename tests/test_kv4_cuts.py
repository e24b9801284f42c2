"""How the attention of single rows over a 4-bit cache is cut, over the shapes and lengths that plans have (no GPU)."""
import ctypes as C
import itertools

import pytest


def cut(pkg, head_size, kv_heads, heads, n, context, max_len, window, sms, quants):
    out = (C.c_int32 * 4)()
    assert pkg.native.lib().b200_test_kv4_step_cut(head_size, kv_heads, heads, n, context, max_len, window, sms, quants, out) == 0
    return tuple(out)


@pytest.mark.parametrize("hs", [32, 64, 96, 128, 256])
def test_every_cta_joins_whole_blocks_of_quants(pkg, hs):
    """A CTA of a cluster joins heads * hs / cluster neighbouring entries; where they become blocks of 32 quants each block has to lie in one of them (a warp quantises a block)."""
    lengths = sorted({2 ** i + d for i in range(18) for d in (-1, 0, 1)} - {0})
    seen = set()
    for (kv_heads, mul), n, context, window, sms in itertools.product(((1, 1), (1, 3), (1, 4), (2, 5), (4, 1), (8, 4), (2, 8), (1, 13), (32, 1), (8, 8)), (1, 2, 7, 40), lengths, (0, 300), (148, 132)):
        for quants, max_len in itertools.product((0, 1), (0, 128)):
            heads, per_head, cluster, splits = cut(pkg, hs, kv_heads, kv_heads * mul, n, context, max_len, window, sms, quants)
            assert heads in (4, 8) and (per_head - 1) * heads < mul <= per_head * heads
            assert cluster in (1, 2, 4, 8) and 1 <= splits <= 296
            assert heads * hs % cluster == 0
            if quants:
                assert heads * hs // cluster % 32 == 0, (kv_heads, mul, n, context, max_len, window, cluster)
            seen.add(cluster)
    assert {1, 2, 4} <= seen


def test_the_cluster_of_heads_of_96(pkg):
    """Four key/value heads of 96 over 4096 positions: 12 blocks of quants a unit, so four CTAs and not eight; without quants eight."""
    assert cut(pkg, 96, 4, 4, 1, 4096, 0, 0, 148, 1)[2] == 4
    assert cut(pkg, 96, 4, 4, 1, 4096, 0, 0, 148, 0)[2] == 8


def test_refusals(pkg):
    out = (C.c_int32 * 4)()
    for bad in ((0, 1, 1, 1, 16, 0, 0, 148, 0), (64, 0, 1, 1, 16, 0, 0, 148, 0), (64, 2, 3, 1, 16, 0, 0, 148, 0), (64, 1, 1, 0, 16, 0, 0, 148, 0), (64, 1, 1, 1, 0, 0, 0, 148, 0),
                (64, 1, 1, 1, 16, -1, 0, 148, 0), (64, 1, 1, 1, 16, 0, -1, 148, 0), (64, 1, 1, 1, 16, 0, 0, 0, 0)):
        assert pkg.native.lib().b200_test_kv4_step_cut(*bad, out) == -1
    assert pkg.native.lib().b200_test_kv4_step_cut(64, 1, 1, 1, 16, 0, 0, 148, 0, None) == -1
