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
