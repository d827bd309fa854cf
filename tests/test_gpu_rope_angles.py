"""Angles of the rotation by position where their digits are hardest to keep, against rational arithmetic."""
import math
from fractions import Fraction

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from test_gpu_kv4 import run_norm_rope

TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211706798214808651")


def exact(positions, frequencies):
    """cos and sin [tokens][pairs] of positions * frequencies, and how far an angle is from a multiple of a quarter turn, in turns."""
    cos, sin, off = [np.zeros((len(positions), len(frequencies))) for _ in range(3)]
    for j, f in enumerate(frequencies):
        turns = Fraction(float(f)) / TWO_PI
        for i, p in enumerate(positions):
            t = turns * int(p)
            quarters = round(4 * t)
            left = float(t - Fraction(quarters, 4))
            c, s = math.cos(2 * math.pi * left), math.sin(2 * math.pi * left)
            cos[i, j], sin[i, j] = ((c, s), (-s, c), (-c, -s), (s, -c))[quarters % 4]
            off[i, j] = abs(left)
    return cos, sin, off


def rotated(positions, frequencies, dtype):
    """What the op makes of the pairs (1, 0): cos and sin."""
    pairs = len(frequencies)
    x = np.zeros((len(positions), 1, 2 * pairs), dtype)
    x[..., :pairs] = 1
    y, _ = run_norm_rope(x, x, positions, 2 * pairs, False, dtype, frequencies=frequencies)
    return y[:, 0, :pairs].astype(np.float64), y[:, 0, pairs:].astype(np.float64)


# fp32: sine and cosine are at most 4 ulp off (2^-23 of the value each: the factor to radians and its product, the square's two roundings, the series' last
# steps), the product with 1 and the sum with 0 half an ulp each. The angle left of a quarter turn is rounded to 24 bits, and 2^-32 of a turn and less is cut off in front of that, the table's own 2^-65 at positions of 2^31 in it.
def tolerance(value, other, off):
    return 5 * 2.0**-23 * np.abs(value) + 2 * math.pi * (2.0**-24 * off + 2.0**-31) * np.abs(other)


def check(positions, frequencies):
    cos, sin, off = exact(positions, frequencies)
    got_cos, got_sin = rotated(positions, frequencies, np.float32)
    for got, want, other in ((got_cos, cos, sin), (got_sin, sin, cos)):
        err, tol = np.abs(got - want), tolerance(want, other, off)
        assert (err <= tol).all(), (err / tol).max()
    # halfs: the hardware's sine and cosine, 2^-19 off, the angle's 2^-26 turns, one rounding
    got_cos, got_sin = rotated(positions, frequencies, np.float16)
    for got, want in ((got_cos, cos), (got_sin, sin)):
        assert (np.abs(got - want) <= 2.0**-11 * np.abs(want) + 2.0**-19 + 2 * math.pi * 2.0**-26 + 2.0**-25).all()


def test_angles_next_to_quarter_turns():
    """Sines and cosines that are small have all their digits: angles a little off a quarter, a half and three quarters of a turn."""
    rng = np.random.default_rng(1)
    away = np.concatenate([2.0**-rng.uniform(8, 20, 32), -(2.0**-rng.uniform(8, 20, 32))])
    frequencies = 2 * math.pi * (rng.integers(0, 4, 64) / 4 + away)
    check(np.array([1, 3, 5, -1, 1001, 2**20 + 1]), frequencies)


def test_frequencies_of_many_turns():
    """Given frequencies of 10 to 2^50 radians at near and far positions."""
    rng = np.random.default_rng(2)
    frequencies = np.concatenate([2.0**rng.uniform(3, 50, 56), -(2.0**rng.uniform(3, 30, 4)), [0.0, 1.0, 2.0**-40, 1e6]])
    check(np.array([0, 1, -1, 77, 4095, 10**6, 10**9 + 7, 2**31 - 1, -2**31]), frequencies)
