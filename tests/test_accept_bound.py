"""The bound of the sampled accept's fp32 sums, which decides what is judged again in 64 bits.

A token's power 2^-a of two is off by 3 ln 2 a 2^-24 of itself (rate, difference and product are a
rounding each), and a row's sum by the mean of that over its mass.  The kernels count 7/4 log2 V for it,
with 20 more for sums in a row and the exponentials' last bits."""
import math

import numpy as np
import pytest


def largest_mean(V):
    """Most that the mean of a, weighted with 2^-a, is over V tokens of which one has a = 0.

    Where the mean is f, its derivative by one a is 0 at a = f + 1/ln 2 alone and positive below, so
    that all others have that a: f = W((V-1)/e) / ln 2 with Lambert's W, here by Newton's steps."""
    n = (V - 1) / math.e
    w = math.log1p(n)
    for _ in range(60):
        e = math.exp(w)
        w -= (w * e - n) / (e * (w + 1))
    return w / math.log(2)


@pytest.mark.parametrize("V", [2, 3, 10, 257, 5000, 50257, 151936, 700001, 2 ** 24, 2 ** 30 - 1])
def test_three_roundings_stay_below_the_coefficient(V):
    assert 3 * math.log(2) * largest_mean(V) < 7 / 4 * math.log2(V)


def test_the_largest_mean():
    rng = np.random.default_rng(7)
    for V in (2, 3, 40, 5000, 151936):
        most = largest_mean(V)
        alike = np.full(V, most + 1 / math.log(2))
        alike[0] = 0
        rows = [alike] + [rng.uniform(0, 2 * most, V) for _ in range(8)]
        rows += [np.abs(rng.normal(0, s, V)) for s in (0.3, 1, 3, 10, 30)]
        rows += [alike * s for s in (0.9, 1.1)]
        for a in rows:
            a = a - a.min()
            mean = (np.exp2(-a) * a).sum() / np.exp2(-a).sum()
            assert mean <= most * (1 + 1e-12), V
        a = alike
        assert abs((np.exp2(-a) * a).sum() / np.exp2(-a).sum() - most) < 1e-9
    assert 12.6 < largest_mean(151936) < 12.7
