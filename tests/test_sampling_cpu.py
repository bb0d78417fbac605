"""The weights of sampling are 2^y by a table and a polynomial: how far that is off, evaluated from the source's own coefficients."""
import re
from fractions import Fraction
from pathlib import Path

import numpy as np

SOURCE = (Path(__file__).resolve().parent.parent / "demonic_b200" / "csrc" / "sample.cu").read_text()


def coefficients():
    """Degree 4 down to 1, in r, from `scaled`; the constant term is 1."""
    body = SOURCE[SOURCE.index("double scaled(float x)"):]
    body = body[:body.index("table[q")]
    first = re.search(r"double p = fma\(([\d.e-]+) / (\d+), r, ([\d.e-]+) / (\d+)\)", body)
    rest = re.findall(r"p = fma\(p, r, ([\d.e-]+)(?: / (\d+))?\)", body)
    got = [(first[1], first[2]), (first[3], first[4])] + rest
    assert len(got) == 5 and got[-1] == ("1.0", "")
    return [float(a) / float(b or 1) for a, b in got]


def test_the_polynomial_is_off_by_less_than_it_says():
    r = np.linspace(-0.5, 0.5, 400001)
    p = np.zeros_like(r)
    for c in coefficients():
        p = p * r + c                             # (f64; each step rounds to 2^-53)
    off = np.abs(p / np.exp2(r / 16) - 1)
    assert off.max() <= 2.0 ** -38
    assert off.max() >= 2.0 ** -40                # what is said is not far from what is


def test_the_offset_that_a_rows_weights_share():
    """y = x c + b is off by half a unit of b's last place, |b| <= 16 log2(e) 45000: a factor of 2^(off / 16) on every weight."""
    b = 16 * 1.4426950408889634 * 45000
    half_unit = Fraction(2) ** (int(np.floor(np.log2(b))) - 53)
    assert float(half_unit) * np.log(2) / 16 <= 2.0 ** -38
