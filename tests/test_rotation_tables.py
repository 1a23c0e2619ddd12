"""Tables of turns against exact fractions, on the CPU."""
import math
import random
from fractions import Fraction

import pytest

import dflash_qmm


def arctan_of(n, bits):
    """arctan(1/n) 2^bits in whole numbers."""
    total, power, k = 0, (1 << bits) // n, 0
    while power:
        total += (-1) ** k * (power // (2 * k + 1))
        power //= n * n
        k += 1
    return total


# 2 pi to some 1590 bits, by Machin's formula
TWO_PI = Fraction(8 * (4 * arctan_of(5, 1600) - arctan_of(239, 1600)), 1 << 1600)

# every size that a double has in a frequency's range: angles of one step, and of many turns
VALUES = [0.0, -0.0, 1.0, -1.0, 0.3, 1e-9, -1e-30, 1e-300, 5e-324, 2 * math.pi, math.pi, 7.0,
          12345.678, 1e6, -1e6, 1e15, -3e17, 2.0 ** 52 + 1, 1e22, 1e30, 2.0 ** 100, -1e38,
          math.nextafter(2.0 ** 127, 0), -math.nextafter(2.0 ** 127, 0)]


def random_values():
    rng = random.Random(5)
    return [rng.choice((-1, 1)) * rng.uniform(1, 2) * 2.0 ** rng.randint(-80, 126)
            for _ in range(400)]


@pytest.mark.parametrize("values", [VALUES, random_values()], ids=["chosen", "random"])
def test_turns_are_right_to_their_last_unit(values):
    """Half a unit of 2^-64 turns, so that position 2^31 is right to 2^-34 turns, and a thousandth
    more for what is left out behind it."""
    rope = dflash_qmm.Rope(2 * len(values), frequencies=values, device="cpu")
    for f, t in zip(values, rope.turns.tolist()):
        off = (Fraction(t % 2 ** 64, 2 ** 64) - Fraction(f) / TWO_PI) % 1
        assert min(off, 1 - off) <= Fraction(501, 1000) / 2 ** 64, f


def test_frequencies_that_are_refused():
    for f in (2.0 ** 127, -2.0 ** 127, 1e300, math.inf, -math.inf, math.nan):
        with pytest.raises(dflash_qmm.DfqError):
            dflash_qmm.Rope(4, frequencies=[1.0, f], device="cpu")
