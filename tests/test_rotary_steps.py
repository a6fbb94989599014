"""How far a plan's steps are from their frequencies, by exact fractions (no
GPU): what include/fp8lin.h says of fp8lin_rotary_steps."""
import ctypes
import random
from fractions import Fraction

import pytest

# 2 pi to 60 digits, from the published expansion of pi
TURN = 2 * Fraction(314159265358979323846264338327950288419716939937510582097494, 10 ** 59)


def steps(fp8lin, freq, axes):
    got = (ctypes.c_uint64 * len(freq))()
    assert fp8lin.lib().fp8lin_rotary_steps((ctypes.c_double * len(freq))(*freq), (ctypes.c_int32 * len(freq))(*axes), len(freq), got) == 0
    return list(got)


def off(step, frequency):
    """|step / 2^64 - frequency / (2 pi)| modulo a turn."""
    d = (Fraction(step, 2 ** 64) - Fraction(frequency) / TURN) % 1
    return min(d, 1 - d)


@pytest.mark.parametrize("sign", [1, -1])
def test_steps_bound(fp8lin, sign):
    rng = random.Random(1)
    freq = [sign * 10.0 ** rng.uniform(-9, 1) for _ in range(500)] + [sign * f for f in (1.0, 0.5, 1e-12, 3.0, 6.283185307179586)]
    axes = [rng.randrange(4) for _ in freq]
    for s, f, a in zip(steps(fp8lin, freq, axes), freq, axes):
        assert s % 4 == a
        # half a unit of 2^-62 and the axis; the quotient by 2 pi; below 0 the turn that is added
        bound = Fraction(5, 2 ** 64) + abs(Fraction(f)) / TURN / 2 ** 52 + (Fraction(1, 2 ** 54) if f < 0 else 0)
        assert off(s, f) <= bound


def test_far_positions_multiply_it(fp8lin):
    """What a step is off is multiplied by the position: more than 2^-33 turns at 2^24 already, and within the bound times the position."""
    s, = steps(fp8lin, [1.0], [2])
    for bits in (24, 30, 40):
        p = 1 << bits
        d = (Fraction(p * s % 2 ** 64, 2 ** 64) - p / TURN) % 1
        d = min(d, 1 - d)
        assert Fraction(p, 2 ** 57) < d <= p * (Fraction(5, 2 ** 64) + 1 / TURN / 2 ** 52)
