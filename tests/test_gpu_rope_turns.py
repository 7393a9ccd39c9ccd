"""Rotary positions far out with frequencies of the caller's own, against angles whose full turns are taken off in whole numbers.

The bound is test_gpu_rope.py's: a frequency's part of a turn is rounded to 2^-65 and multiplied by up to 2^31, and the angle is cut to 2^-32,
so it is off by 1.25 * 2^-32 of a turn (2^-29 rad), beside fp32 roundings of 5 * 2^-24 in all for a cosine or sine.
"""
from fractions import Fraction

import numpy as np
import pytest
import torch

import q4hip

pytestmark = pytest.mark.gpu

BITS = 1300


def two_pi():
    """2 pi * 2^BITS, by J. Machin's 16 arctan(1/5) - 4 arctan(1/239)."""
    def arctan(x):
        t = s = (1 << BITS + 32) // x
        n, sign = 3, -1
        while t:
            t //= x * x
            s += sign * (t // n)
            n, sign = n + 2, -sign
        return s
    return (8 * (4 * arctan(5) - arctan(239))) >> 32


def angles(pos, freq):
    """Radians without the full turns, correct to 2^-50."""
    turn = Fraction(two_pi(), 1 << BITS)
    parts = [[Fraction(float(f)) * int(p) / turn % 1 for f in freq] for p in pos]
    return 2 * np.pi * np.array([[float(a) for a in row] for row in parts])


FREQ = [1e6, -1e6, 2 * np.pi, 1e15, 2.0 ** 53 + 2, -3e17, 2.0 ** 64, 1e100, -1.7976931348623157e308, 2.0 ** 970, 2.0 ** -11, 1e-18, 1e-40, 5e-324,
        0.0, -0.0, 0.75, -1e-9, np.pi, 2.0 ** 63]
POS = [0, 1, -1, 2, 499, 65537, -1000003, 2 ** 24 + 1, 2 ** 30 + 12345, 2 ** 31 - 1, -2 ** 31]


@pytest.mark.parametrize("order", ["halves", "pairs"])
def test_any_frequency_at_any_position(order):
    n, half = len(POS), len(FREQ)
    r = q4hip.Rope(2 * half, 2 * half, order, np.array(FREQ))
    rng = np.random.default_rng(1)
    x = torch.tensor(rng.standard_normal((n, 2 * half)).astype(np.float32)).cuda()
    p = torch.tensor(POS, dtype=torch.int32, device="cuda")
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    r.run(x.data_ptr(), y.data_ptr(), 1, q4hip.F32, 2 * half, 2 * half, p.data_ptr(), n)
    t, z, got = angles(POS, FREQ), x.double().cpu().numpy(), y.double().cpu().numpy()
    first, second = (np.s_[:, :half], np.s_[:, half:]) if order == "halves" else (np.s_[:, ::2], np.s_[:, 1::2])
    a, b = z[first], z[second]
    for at, want in ((first, a * np.cos(t) - b * np.sin(t)), (second, b * np.cos(t) + a * np.sin(t))):
        err = np.abs(got[at] - want)
        bound = (np.abs(a) + np.abs(b)) * 8 * 2.0 ** -24 + np.abs(want) * 2.0 ** -24
        assert (err <= bound).all(), float((err / bound).max())
