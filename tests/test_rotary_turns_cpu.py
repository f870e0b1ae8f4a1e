"""The table of a rotary plan: turns per position are the nearest 64-bit fraction to frequency / 2 pi, whatever the frequency."""
import math
from fractions import Fraction

import pytest

# pi from the arithmetic-geometric mean, another series than the plan's own
BITS = 1400


def _pi():
    one = 1 << BITS
    root = lambda x: math.isqrt(x << BITS)  # noqa: E731
    a, b, t, p = one, root(one // 2), one // 4, 1
    for _ in range(12):
        a, b, t, p = (a + b) // 2, root(a * b >> BITS), t - p * (((a - (a + b) // 2) ** 2) >> BITS), 2 * p
    return Fraction((a + b) ** 2 // (4 * t), one)


PI = _pi()
FREQUENCIES = [1.0, 10000.0 ** (-1 / 64), 10000.0 ** (-63 / 64), 1e-30, 5e-324, 0.0, -1.0, -0.3, math.pi, 2 * math.pi, -2 * math.pi, 100.0, 12345.678, 1e15, 3.7e300, -1.7e308, 2.0 ** 40]


def test_pi():
    assert abs(PI - Fraction(math.pi)) < Fraction(1, 2 ** 51) and str(int(PI * 10 ** 60)).startswith("314159265358979323846264338327950288419716939937510582097494")


@pytest.mark.parametrize("f", FREQUENCIES)
def test_turns_are_the_nearest(f):
    from acctransformer_b200.rotary import turns_of
    got = turns_of(f)
    assert -2 ** 63 <= got < 2 ** 63
    want = Fraction(f) / (2 * PI) * 2 ** 64
    off = (got - want) % 2 ** 64
    off = min(off, 2 ** 64 - off)
    # half a unit, and what the plan's pi leaves of the quotient: 2^-96 of at most one turn more than 2^64 units
    assert off <= Fraction(1, 2) + Fraction(1, 2 ** 24)
