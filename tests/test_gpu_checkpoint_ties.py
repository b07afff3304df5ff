"""Codes of 8-bit checkpoints next to a tie: round(127 x / m) in real arithmetic, ties to even, against exact fractions."""
from fractions import Fraction

import numpy as np
import pytest

from test_gpu_sequence_ops import DTYPES, _t

pytestmark = pytest.mark.gpu


def _exact(x, m):
    t = 127 * Fraction(abs(x)) / Fraction(m)
    low, rest = t.numerator // t.denominator, t - t.numerator // t.denominator
    c = low + (rest > Fraction(1, 2) or (rest == Fraction(1, 2) and low % 2))
    return -c if x < 0 else c


def _near_ties(dt, m, rng):
    """A block whose largest magnitude is m, the others at the ties and up to two steps beside them, of either sign."""
    f = np.finfo(dt)
    v = np.empty(128, dt)
    v[0] = m
    for i in range(1, 128):
        k = int(rng.integers(0, 127))
        x = dt(float(Fraction(2 * k + 1) * Fraction(float(m)) / 254))
        for _ in range(int(rng.integers(0, 3))):
            x = np.nextafter(x, dt(0) if rng.random() < 0.5 else f.max)
        v[i] = -x if rng.random() < 0.5 else x
    assert np.abs(v).max() == m
    return v


@DTYPES
def test_codes_next_to_ties(dt):
    rng, f = np.random.default_rng(1), np.finfo(dt)
    low, high = (-300, 300) if dt is np.float64 else (-37, 38)
    mags = [dt(v) for v in rng.uniform(0.5, 1.5, 120)] + [dt(10.0 ** e * u) for e, u in zip(rng.uniform(low, high, 60), rng.uniform(1, 2, 60))]
    mags += [dt(254), dt(127), dt(1), dt(254 * 3), f.max, f.max / dt(3), f.tiny, f.tiny * dt(5), f.smallest_subnormal * dt(12345), f.smallest_subnormal * dt(254),
             dt(1e300) if dt is np.float64 else dt(1e37), dt(1e-280) if dt is np.float64 else dt(1e-30)]
    x = np.concatenate([_near_ties(dt, m, rng) for m in mags])
    want = np.array([_exact(float(v), float(m)) for b, m in zip(x.reshape(-1, 128), mags) for v in b])
    got = _t(x).checkpoint8().codes.cpu().numpy().astype(np.int64)
    wrong = np.nonzero(got != want)[0]
    assert wrong.size == 0, (wrong.size, [(float(x[i]), float(mags[i // 128]), int(got[i]), int(want[i])) for i in wrong[:4]])


@DTYPES
def test_codes_of_every_tie_of_a_whole_magnitude(dt):
    """m = 254: the odd numbers are ties, all of them and with their signs; beside them random values of the same block."""
    rng = np.random.default_rng(2)
    x = np.concatenate([np.arange(1, 254, 2), -np.arange(1, 254, 2), [254.0, -254.0]]).astype(dt)
    rng.shuffle(x)
    x[0], x[128] = 254, -254
    want = np.array([_exact(float(v), 254.0) for v in x])
    assert np.array_equal(_t(x).checkpoint8().codes.cpu().numpy().astype(np.int64), want)
