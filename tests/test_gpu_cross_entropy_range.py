"""The softmax cross-entropy over the whole range of the type: masks of any common value over all classes of a thread, maxima far
from zero, maxima that differ by the type's last bit.

Tolerances are those of the general test, roundings counted per exponential and per sum.  Far from zero x - m, its product with
log2 e and that constant round once each, 2.3 u |x - m| in all, within the 2 u |x - m| + 88 u counted there as long as the exponential is
not zero.  Exponentials below the smallest normal number count as zero: `tiny` more in the map."""
import numpy as np
import pytest

from test_gpu_sequence_ops import DTYPES, U, _ce_ref, _close, _t

pytestmark = pytest.mark.gpu

# a class count for each way a row is dealt out: a thread, some threads of a warp (whole vectors and not), a CTA of every kind, clusters, a
# CTA that reads the row twice
CLASSES = [10, 20, 63, 250, 700, 701, 1023, 1500, 5000, 8191, 20000, 40000, 40001, 140000, 262149, 300000]


def _check(x, t, reduction="sum"):
    from rtensors_b200.tensor import cross_entropy_loss
    dt = x.dtype.type
    with np.errstate(over="ignore"):
        loss_w, loss_tol, g_w, g_tol = _ce_ref(x, t, reduction == "mean", U[dt])
    loss, g = cross_entropy_loss(_t(x), _t(t), True, reduction)
    _close(g.cpu(), g_w, g_tol + 2 * float(np.finfo(dt).tiny))
    assert abs(float(loss.item()) - loss_w) <= loss_tol
    assert cross_entropy_loss(_t(x), _t(t), reduction=reduction).cpu().tobytes() == loss.cpu().tobytes()


@DTYPES
@pytest.mark.parametrize("classes", CLASSES)
def test_masks_over_whole_threads(dt, classes):
    """An ordinary row with all but a few classes masked, whatever the mask's value."""
    rng = np.random.default_rng(classes)
    fills = [-1e4, -1e7, -1e9, -3e9, -1e10, -1e12, -1e18, -1e20, -1e30, -1e36]
    x = rng.standard_normal((len(fills), classes)).astype(dt)
    t = np.zeros(len(fills), np.int64)
    for r, fill in enumerate(fills):
        left = rng.choice(classes, 3, replace=False)
        masked = np.ones(classes, bool)
        masked[left] = False
        x[r, masked] = fill
        t[r] = left[0]
    _check(x, t)
    _check(x, t, "mean")


@DTYPES
@pytest.mark.parametrize("classes", CLASSES)
@pytest.mark.parametrize("sign", [1, -1])
def test_maxima_far_from_zero(dt, classes, sign):
    """Rows around +-1e6 ... +-1e37, next to each other in steps of the type, and on both sides of a power of two."""
    rng = np.random.default_rng(classes + 1)
    around = [1e6, 2.0 ** 22, 6e6, 3e7, 1e9, 2.0 ** 30, 3e9, 1e10, 1e12, 1e20, 1e30, 9e36, 1.2e38]
    x = np.empty((len(around), classes), dt)
    t = np.empty(len(around), np.int64)
    for r, v in enumerate(around):
        step = max(float(np.spacing(dt(v))), 1.0)
        # a few steps above and below, most of them equal: ties of the maximum in different threads
        x[r] = sign * v + step * np.minimum(rng.integers(-6, 4, classes), 1)
        t[r] = int(np.argmax(x[r]))
    _check(x, t)


@pytest.mark.parametrize("classes", [20, 700, 5000, 40000, 140000, 300000])
@pytest.mark.parametrize("base", [1.2e38, -1.2e38, 1.5e37, -2.5e37, 3.4e38, 5e9])
def test_maxima_one_step_apart_stay_apart(classes, base):
    """Beyond 2^30 one step is 64 and more: only the larger of two neighbouring floats counts, in whichever thread it is."""
    base, rng = np.float32(base), np.random.default_rng(classes + 2)
    x = np.empty((20, classes), np.float32)
    t = np.empty(20, np.int64)
    for r in range(20):
        above = np.nextafter(base, np.float32(np.inf))
        assert float(above) - float(base) >= 64
        x[r] = base
        t[r] = rng.integers(0, classes)
        x[r, t[r]] = above
        base = above if base < 0 or r < 10 else base
    _check(x, t)


@DTYPES
@pytest.mark.parametrize("classes", CLASSES)
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_targets_far_below_the_maximum(dt, classes, reduction):
    """A masked target has a loss as large as its distance from the maximum: finite as long as the type can hold it."""
    rng = np.random.default_rng(classes + 3)
    low = float(np.finfo(dt).min)
    rows = [(0.0, -200.0), (1.0, -1e6), (3.0, -5e6), (-4.1e6, -4.3e6), (0.0, -1e10), (5e9, -5e9), (0.0, -2.4e38), (1.0, low), (3e37, -3e37),
            (2.0 ** 22, -2.0 ** 22), (1e37, -1e37), (low / 4, low)]
    for top, target in rows:
        # one row at a time: a sum of all would only show the largest
        x = np.full((2, classes), target, dt)
        x[0] = (rng.standard_normal(classes) + top).astype(dt)
        t = np.array([rng.integers(0, classes), -1])
        x[0, t[0]] = target
        _check(x, t, reduction)


def test_a_loss_that_only_the_mean_can_hold():
    """Two rows' losses of 0.65 times the largest float each: their sum is beyond f32, their mean is not."""
    from rtensors_b200.tensor import cross_entropy_loss
    for classes in CLASSES:
        x = np.full((2, classes), -2.0 ** 126, np.float32)
        x[:, 0] = 2.0 ** 127 * 0.8
        t = np.array([1, classes - 1])
        want = 2.0 ** 126 + float(np.float32(2.0 ** 127 * 0.8))
        # log2 e as a float is off by half a rounding, its product with the difference is the loss
        assert abs(float(cross_entropy_loss(_t(x), _t(t)).item()) - want) <= 4 * U[np.float32] * want
        assert cross_entropy_loss(_t(x), _t(t), reduction="sum").item() == np.inf


@DTYPES
@pytest.mark.parametrize("classes", CLASSES)
def test_infinities_next_to_far_maxima(dt, classes):
    """Classes masked with -inf in rows far from zero take no part; one +inf, a NaN or nothing but -inf give NaN, in that row alone."""
    from rtensors_b200.tensor import cross_entropy_loss
    rng = np.random.default_rng(classes + 4)
    x = rng.standard_normal((7, classes)).astype(dt)
    t = np.zeros(7, np.int64)
    for r, v in enumerate((5e6, -1e10, 1e20, -3e37)):
        x[r] = -np.inf
        left = rng.choice(classes, 2, replace=False)
        x[r, left] = v
        t[r] = left[0]
    x[4, classes // 2], x[5, classes // 2], x[6] = np.inf, np.nan, -np.inf
    x[4:6, 0] = -1e20
    _check(x[:4].copy(), t[:4])
    loss, g = cross_entropy_loss(_t(x), _t(t), True)
    g, (_, _, g_w, g_tol) = g.cpu(), _ce_ref(x[:4], t[:4], False, U[dt])
    assert np.isnan(loss.item()) and np.isnan(g[4:]).all()
    _close(g[:4] * 7, g_w, g_tol + 4 * U[dt] * np.abs(g_w))     # a seventh each: the mean's factor rounds, and its product
