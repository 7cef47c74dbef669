"""Rotary positions far beyond fp32's whole numbers, against angles of exact rationals."""
from fractions import Fraction
from math import cos, sin

import numpy as np
import pytest

from qutai_amd.backends import amd, amd_lm
from qutai_amd.lm import Rotary
from tests.helpers import download, upload

pytestmark = pytest.mark.gpu

PI = Fraction(31415926535897932384626433832795028841971693993751, 10 ** 49)  # to 50 digits


def rest(angle):
    """The angle of a rational number of radians less its whole turns."""
    turns = angle / (2 * PI)
    return float((turns - round(turns)) * 2 * PI)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("place", [2 ** 24 + 1, 2 ** 31 + 5, 2 ** 40 + 1, -(2 ** 40 + 1)])
def test_far_positions(place, layout):
    """Pair 0 turns by 1 radian a position, pair 1 by 2^-10.  What is kept of a turn: the
    turns of one position are a quotient of doubles (2^-53 of it, and less than half of that
    for pi's own), their product with the position rounds once more: 2.5 x 2^-53 of the
    angle in all, then 9 half steps of fp32 as near 0.  At 2^40 positions: 2^-12 radians and
    a quarter of pair 0, 2^-22 of pair 1."""
    turns = Rotary(4, theta=2.0 ** 20, layout=layout)
    assert turns.frequencies == (1.0, 2.0 ** -10)
    x = np.array([1.0, 1.0, 0.0, 0.0] if layout == "half" else [1.0, 0.0, 1.0, 0.0])
    for where in (dict(offset=place), dict(positions=amd.storage([place], dtype="int64")),
                  dict(offset=5, starts=amd.storage([place - 5], dtype="int64"))):
        got, _ = amd_lm.rotary(upload(x, "float32"), None, turns, 1, 1, 1, 0, 4, **where)
        got = download(got).reshape(2, 2)
        for pair, frequency in enumerate((Fraction(1), Fraction(1, 1024))):
            a, b = got[:, pair] if layout == "half" else got[pair]
            angle = rest(place * frequency)
            bound = abs(place) * float(frequency) * 2.5 * 2.0 ** -53 + 9 * 2.0 ** -24
            assert abs(a - cos(angle)) <= bound and abs(b - sin(angle)) <= bound, (place, pair)
