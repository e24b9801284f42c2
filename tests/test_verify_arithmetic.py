"""The arithmetic of the verification of drafted tokens that decides whether it is right and whether it ends, on the host."""
import ctypes as C
import math
from decimal import Decimal, localcontext

import numpy as np
import pytest


def weights(pkg, x, top, temperature):
    x = np.asarray(x, dtype=np.float32)
    out = np.empty(len(x))
    rc = pkg.native.lib().b200_test_verify_weights(x.ctypes.data_as(C.POINTER(C.c_float)), len(x), C.c_float(top), C.c_float(temperature), out.ctypes.data_as(C.POINTER(C.c_double)))
    assert rc == 0
    return out


def exact(x, top, temperature):
    with localcontext() as c:
        c.prec = 60
        return ((Decimal(float(np.float32(x))) - Decimal(float(np.float32(top)))) / Decimal(float(np.float32(temperature)))).exp()


@pytest.mark.parametrize("temperature", [1e-4, 1e-3, 0.7, 1.0, 1e4])
@pytest.mark.parametrize("top", [0.0, 1.0, -3.5, 81920.0, 1048577.0, 1.5e6, 1e7, 6e9, 1e10, -1e10, 2.7e9, 1e20, -1e30, 3e38])
def test_weights_of_neighbours_of_large_logits(pkg, top, temperature):
    """A row's logits may be so far from 0 that neighbouring numbers are hundreds of temperatures apart: weights are e^-(distance), or 0 where that is below e^-690, never anything else.

    690 is told to 2^-20 of itself (the high word of a 64-bit number), so e^-690 to 690 * 2^-20 < 7e-4 of itself."""
    x = [np.float32(top)]
    for _ in range(40):
        x.append(np.nextafter(x[-1], np.float32(-np.inf)))
    x += [np.float32(top - d * temperature) for d in (1, 50, 500, 689, 689.9, 690.1, 691, 700, 710, 1000, 1380, 2000, 1e5, 1e30)] + [np.float32(-np.inf), np.float32(-3.4e38)]
    x = [v for v in x if v <= np.float32(top)]
    got = weights(pkg, x, top, temperature)
    assert got[0] == 1.0
    for v, w in zip(x, got):
        far = (float(np.float32(top)) - float(v)) / float(np.float32(temperature))
        if far > 690.001:
            assert w == 0.0, (float(v), w)
        else:
            assert far > 689.999 and w == 0.0 or abs(Decimal(float(w)) / exact(v, top, temperature) - 1) <= Decimal(1e-12), (float(v), w)


def test_passes_over_a_drawn_row_end(pkg):
    """Whatever a pass's sums are, the next pass has a higher number or there is none: at most three passes, and 4 or 5 behind them."""
    import itertools

    values = [0.0, 1.0, 0.5, 1e-300, 1e-13, -1.0, -6e171, 1e308, math.inf, -math.inf, math.nan]
    for kind in range(4):
        for sums in itertools.product(values, repeat=4):
            rows = (C.c_double * 2)(1.0, 1.0)
            then = pkg.native.lib().b200_test_verify_next(kind, (C.c_double * 4)(*sums), rows)
            assert kind < then <= 5, (kind, sums, then)
            if then == 4:  # there is something to draw from
                assert sums[0] > 0
            if kind == 3:
                assert then == (4 if 0 < sums[0] < 1e300 else 5)
    for bad in (-1, 4, 5):
        assert pkg.native.lib().b200_test_verify_next(bad, (C.c_double * 4)(), (C.c_double * 2)()) == -1


def test_what_follows_a_pass(pkg):
    def then(kind, *sums):
        rows = (C.c_double * 2)(7.0, 7.0)
        return pkg.native.lib().b200_test_verify_next(kind, (C.c_double * 4)(*sums), rows), tuple(rows)

    assert then(0, 3.0, 0, 0, 0)[0] == 4 and then(0, 0.0, 0, 0, 0)[0] == 3  # nothing but the draft: p as it is
    assert then(1, 2.0, 4.0, 1.0, 1.0) == (4, (2.0, 4.0))  # 1/2 - 1/4 is left over
    assert then(1, 2.0, 4.0, 1.0, 1.95) == (2, (2.0, 4.0))  # little: once more by exact sums
    assert then(2, 2.0, 4.0, 1.0, 1.95)[0] == 4 and then(2, 2.0, 4.0, 1.0, 2.0)[0] == 3  # the same distributions: p


@pytest.mark.parametrize("temperature", [1e-4, 0.1, 0.6, 0.7, 1.0, 1.3, 17.0, 1e4])
def test_weights_are_as_near_as_their_bound_says(pkg, temperature):
    """4.5e-16 |x - top| / T and 3e-15 of the weight over the whole range: four roundings of 2^-53 in the argument, 4.44e-16 of it; the series' first missing term, (ln(2) / 64)^6 / 720 = 2.25e-15, the table's
    2^-52 at most, and roundings of 2^-53 for the last step of the series and the product, and less than that in front of it, 0.45e-15.  Two of them and two sums (1.2e-13) stay below the margin of 2^-40."""
    rng = np.random.default_rng(7)
    for top in (0.0, 3.25, -11.0):
        x = np.unique(np.float32(top) - np.float32(temperature) * np.concatenate([rng.uniform(0, 689, 1500), rng.uniform(0, 1, 300), 10.0 ** rng.uniform(-9, 2, 200)]).astype(np.float32)).astype(np.float32)
        x = x[(x <= np.float32(top)) & (x >= np.float32(top) - np.float32(689.5 * temperature))]
        for v, w in zip(x, weights(pkg, x, top, temperature)):
            far = (float(np.float32(top)) - float(v)) / float(np.float32(temperature))
            assert abs(Decimal(float(w)) / exact(v, top, temperature) - 1) <= Decimal(4.5e-16 * far + 3e-15), far
    assert 2 * (4.5e-16 * 690 + 3e-15) + 2 * 1.2e-13 < 2.0 ** -40
