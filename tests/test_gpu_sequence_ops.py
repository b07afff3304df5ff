"""The gated recurrence, 8-bit checkpoints and the softmax cross-entropy against plain 64-bit restatements.

Tolerances count roundings, u = half a step of the type.  Recurrence: a term x_j enters h_s through s - j products and at most
as many sums (however they are associated), plus a fixed number of compositions per tile, so
|error| <= E_s + 24 u A_s with A_s = |a| A_{s-1} + |x_s| and E_s = |a| E_{s-1} + 2 u A_s."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}
DTYPES = pytest.mark.parametrize("dt", [np.float32, np.float64], ids=["f32", "f64"])


def _b():
    from cuda_engine import backend
    return backend()


def _t(a):
    from rtensors_b200.tensor import Tensor
    return Tensor.from_buf(a, a.shape, a.dtype.type, _b())


def _recur(a, b, first, u=None):
    """h, and the tolerance; time in dim 0, in processing order."""
    h, mag, err = np.zeros_like(b), np.zeros_like(b), np.zeros_like(b)
    last, m, e = first.copy(), np.abs(first), np.zeros_like(first)
    for s in range(len(b)):
        last = a[s] * last + b[s]
        m = np.abs(a[s]) * m + np.abs(b[s])
        if u is not None:
            e = np.abs(a[s]) * e + 2 * u * m
        h[s], mag[s], err[s] = last, m, e
    return (h, err + 24 * (u or 0) * mag, mag)


def _oriented(v, axis, reverse):
    v = np.moveaxis(v, axis, 0)
    return v[::-1] if reverse else v


def _back(v, axis, reverse):
    return np.moveaxis(v[::-1] if reverse else v, 0, axis)


def _scan_ref(x, gate, axis, h0, reverse, coupled, u):
    x, a = x.astype(np.float64), np.broadcast_to(gate.astype(np.float64), x.shape)
    xo, ao = _oriented(x, axis, reverse), _oriented(a, axis, reverse)
    bo = (1 - ao) * xo if coupled else xo
    first = np.zeros(xo.shape[1:]) if h0 is None else np.moveaxis(h0.astype(np.float64), axis, 0)[0]
    h, tol, mag = _recur(ao, bo, first, u)
    return _back(h, axis, reverse), _back(tol, axis, reverse)


def _scan_back_ref(up, gate, axis, h, x, h0, reverse, coupled, u):
    shape = up.shape
    a = np.broadcast_to(gate.astype(np.float64), shape)
    ao, uo, ho = (_oriented(v.astype(np.float64), axis, reverse) for v in (a, up, h))
    later = np.concatenate([ao[1:], np.zeros_like(ao[:1])])
    g, tol, mag = _recur(later[::-1], uo[::-1], np.zeros(uo.shape[1:]), u)
    g, tol, mag = g[::-1], tol[::-1], mag[::-1]
    first = np.zeros(uo.shape[1:]) if h0 is None else np.moveaxis(h0.astype(np.float64), axis, 0)[0]
    before = np.concatenate([first[None], ho[:-1]])
    if coupled:
        xo = _oriented(x.astype(np.float64), axis, reverse)
        dx, dx_tol = (1 - ao) * g, np.abs(1 - ao) * (tol + 3 * u * mag)
        da, da_tol = g * (before - xo), tol * np.abs(before - xo) + 4 * u * mag * (np.abs(before) + np.abs(xo))
    else:
        dx, dx_tol = g, tol
        da, da_tol = g * before, tol * np.abs(before) + 2 * u * mag * np.abs(before)
    out = [(_back(v, axis, reverse), _back(t, axis, reverse)) for v, t in ((dx, dx_tol), (da, da_tol))]
    d0 = (ao[0] * g[0], np.abs(ao[0]) * tol[0] + 2 * u * np.abs(ao[0]) * mag[0])
    # the gate's broadcast dims are summed
    v, t = out[1]
    gs = (1,) * (len(shape) - gate.ndim) + gate.shape
    dims = tuple(k for k in range(len(shape)) if gs[k] == 1 and shape[k] != 1)
    if dims:
        n = int(np.prod([shape[k] for k in dims]))
        t = t.sum(axis=dims, keepdims=True) + n * u * np.abs(v).sum(axis=dims, keepdims=True)
        v = v.sum(axis=dims, keepdims=True)
    out[1] = (v.reshape(gate.shape), t.reshape(gate.shape))
    return out[0], out[1], tuple(np.expand_dims(q, axis) for q in d0)


def _close(got, want, tol):
    got = got.astype(np.float64)
    bad = ~(np.abs(got - want) <= tol + 1e-300)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3].tolist(), float(np.abs(got - want).max()))


def _data(dt, shape, gate_shape, axis, h0, seed=0):
    rng = np.random.default_rng(seed + 7 * len(shape) + shape[axis])
    x = rng.standard_normal(shape).astype(dt)
    a = (1 / (1 + np.exp(-rng.standard_normal(gate_shape) - 2))).astype(dt)
    if a.size > 3:
        a.reshape(-1)[:: 17] = 0          # resets
        a.reshape(-1)[1:: 23] = 1
        a.reshape(-1)[2:: 29] *= -1
    first = tuple(1 if k == axis else n for k, n in enumerate(shape))
    return rng, x, a, rng.standard_normal(first).astype(dt) if h0 else None


# shape, gate's shape (None: full), axis.  Tiles are 32 or 64 steps by 32 to 128 lanes, 2048 or 4096 steps along a contiguous axis.
SHAPES = [
    ((1,), None, 0), ((5,), None, 0), ((3, 1, 2), None, 1), ((2, 7, 3), None, 1), ((2, 64, 128), None, 1), ((1, 65, 130), None, 1),
    ((3, 33, 36), None, 1), ((129, 40), None, 0), ((2, 5000, 12), None, 1), ((1, 2600, 260), None, 1), ((4, 3, 257), None, 0),
    ((3, 511), None, 1), ((2, 512), None, 1), ((2, 9001), None, 1), ((1, 20000), None, 1), ((5000, 6), None, 1), ((2500, 700), None, 1),
    ((2, 96, 4, 32), (2, 96, 4, 1), 1), ((2, 70, 3, 5), (2, 70, 3, 1), 1), ((3, 50, 24), (24,), 1), ((3, 50, 24), (1, 1, 1), 1),
    ((4, 300), (4, 1), 1), ((2, 3, 100, 2, 8), (3, 1, 2, 1), 2),
]


@DTYPES
@pytest.mark.parametrize("reverse,coupled,h0", [(False, False, False), (True, False, True), (False, True, True), (True, True, False)])
@pytest.mark.parametrize("shape,gate_shape,axis", SHAPES, ids=lambda v: str(v).replace(" ", "") if isinstance(v, tuple) else None)
def test_scan_and_its_gradient(dt, shape, gate_shape, axis, reverse, coupled, h0):
    from rtensors_b200.tensor import gated_scan_backward
    rng, x, a, first = _data(dt, shape, gate_shape or shape, axis, h0)
    tx, ta, t0 = _t(x), _t(a), _t(first) if h0 else None
    got = tx.gated_scan_at(axis, ta, t0, reverse=reverse, coupled=coupled)
    _close(got.cpu(), *_scan_ref(x, a, axis, first, reverse, coupled, U[dt]))
    up, h = rng.standard_normal(shape).astype(dt), rng.standard_normal(shape).astype(dt)
    want = _scan_back_ref(up, a, axis, h, x, first, reverse, coupled, U[dt])
    grads = gated_scan_backward(_t(up), axis, ta, _t(h), tx if coupled else None, t0, reverse, coupled)
    for g, w in zip(grads[:2], want[:2]):
        _close(g.cpu(), *w)
    assert (grads[2] is None) == (not h0)
    if h0:
        _close(grads[2].cpu(), *want[2])
    # the same from the states' 8-bit checkpoint: h is then what the codes stand for, one more rounding
    ck = _t(h).checkpoint8()
    kept = ck.restore().cpu()
    want8 = _scan_back_ref(up, a, axis, kept, x, first, reverse, coupled, U[dt])
    grads8 = gated_scan_backward(_t(up), axis, ta, ck, tx if coupled else None, t0, reverse, coupled)
    for g, w in zip(grads8[:2], want8[:2]):
        _close(g.cpu(), *w)
    only_x = gated_scan_backward(_t(up), axis, ta, None, None, None, reverse, coupled, want=(True, False, False))
    assert only_x[1] is None and only_x[0].cpu().tobytes() == grads[0].cpu().tobytes()


@DTYPES
@pytest.mark.parametrize("case", ["transposed", "reversed", "window", "odd_offset", "six_dims", "batch_last"])
def test_scan_over_views(dt, case):
    rng = np.random.default_rng(3)

    def view(t):
        if case == "transposed":
            return t.permute((1, 0, 2))
        if case == "reversed":
            return t.slice(2, None, None, -1).slice(1, None, None, -1)
        if case == "window":
            return t.slice(2, 4, 20).slice(1, 3, 60)
        if case == "odd_offset":
            return t.slice(2, 1, 18)
        if case == "batch_last":
            return t.permute((2, 1, 0))
        return t

    def np_view(v):
        return {"transposed": lambda: v.transpose(1, 0, 2), "reversed": lambda: v[:, ::-1, ::-1], "window": lambda: v[:, 3:60, 4:20],
                "odd_offset": lambda: v[:, :, 1:18], "batch_last": lambda: v.transpose(2, 1, 0), "six_dims": lambda: v}[case]()
    if case == "six_dims":
        # no two neighbouring dims merge for all operands
        shape, axis = (2, 3, 40, 2, 3, 2, 3), 2
        xb, ab = rng.standard_normal((3, 2, 40, 3, 2, 3, 2)).astype(dt), rng.uniform(0, 1, shape).astype(dt)
        x, gate = _t(xb).permute((1, 0, 2, 4, 3, 6, 5)), _t(ab)
        xn, an = xb.transpose(1, 0, 2, 4, 3, 6, 5), ab
    else:
        base = rng.standard_normal((4, 70, 24)).astype(dt), rng.uniform(0, 1, (4, 70, 24)).astype(dt)
        axis = 1
        x, gate = view(_t(base[0])), view(_t(base[1]))
        xn, an = np_view(base[0]), np_view(base[1])
    _close(x.gated_scan_at(axis, gate).cpu(), *_scan_ref(xn, an, axis, None, False, False, U[dt]))
    from rtensors_b200.tensor import gated_scan_backward
    h = rng.standard_normal(xn.shape).astype(dt)
    want = _scan_back_ref(xn, an, axis, h, xn, None, False, True, U[dt])
    dx, dg, _ = gated_scan_backward(x, axis, gate, _t(h), x, coupled=True)
    _close(dx.cpu(), *want[0])
    _close(dg.cpu(), *want[1])


def test_scan_of_nothing():
    from rtensors_b200.tensor import gated_scan_backward
    e = np.zeros((2, 0, 3), np.float32)
    h0 = np.ones((2, 1, 3), np.float32)
    assert _t(e).gated_scan_at(1, _t(e), _t(h0)).shape == (2, 0, 3)
    gate = np.ones((1, 1, 3), np.float32)
    dx, dg, d0 = gated_scan_backward(_t(e), 1, _t(gate), _t(e), h0=_t(h0))
    assert dx.shape == (2, 0, 3) and not dg.cpu().any() and dg.shape == (1, 1, 3) and not d0.cpu().any()


def test_scan_is_deterministic_and_chunks_do_not_show():
    """The chain's folds have one order: repeated runs agree bit for bit, and non-finite values do not leave their lane."""
    rng = np.random.default_rng(11)
    x = rng.standard_normal((1, 30000, 160)).astype(np.float32)
    a = rng.uniform(0.9, 1, x.shape).astype(np.float32)
    x[0, 5000, 3] = np.inf
    x[0, 7000, 5] = np.nan
    tx, ta = _t(x), _t(a)
    first = tx.gated_scan_at(1, ta).cpu()
    for _ in range(4):
        assert tx.gated_scan_at(1, ta).cpu().tobytes() == first.tobytes()
    ok = np.ones(160, bool)
    ok[[3, 5]] = False
    assert np.isfinite(first[:, :, ok]).all() and np.isfinite(first[0, :5000, 3]).all() and np.isfinite(first[0, :7000, 5]).all()
    assert not np.isfinite(first[0, 5000:, 3]).any() and np.isnan(first[0, 7000:, 5]).all()


@DTYPES
@pytest.mark.parametrize("shape,gate_shape", [((1,), (1,)), ((64, 2048), (64, 2048)), ((7, 33), (7, 1)), ((3, 5, 6), (6,)), ((), ())])
@pytest.mark.parametrize("coupled", [False, True])
def test_step_in_place(dt, shape, gate_shape, coupled):
    rng = np.random.default_rng(5)
    h, x, a = (np.asarray(rng.standard_normal(s)).astype(dt) for s in (shape, shape, gate_shape))
    t = _t(h)
    assert t.gated_step_inplace(_t(a), _t(x), coupled=coupled) is t
    a64, x64, h64 = a.astype(np.float64), x.astype(np.float64), h.astype(np.float64)
    want = a64 * h64 + ((1 - a64) * x64 if coupled else x64)
    _close(t.cpu(), want, 4 * U[dt] * (np.abs(a64 * h64) + (1 + np.abs(a64)) * np.abs(x64)))


def test_steps_equal_the_scan_and_leave_the_rest_of_a_pool():
    """Token by token on a strided slice of a larger state pool: the same states as the scan, the other slots untouched."""
    rng = np.random.default_rng(6)
    pool = rng.standard_normal((6, 10, 36)).astype(np.float32)
    x, a = rng.standard_normal((6, 40, 16)).astype(np.float32), rng.uniform(0, 1, (6, 40, 16)).astype(np.float32)
    tp = _t(pool)
    state = tp.index(1, 4).slice(1, 8, 24) if tp.index(1, 4).rank == 2 else tp.index(1, 4).squeeze(1).slice(1, 8, 24)
    tx, ta = _t(x), _t(a)
    h = tx.gated_scan_at(1, ta, _t(pool[:, 4:5, 8:24])).cpu()
    for s in range(40):
        step = [v.index(1, s) for v in (ta, tx)]
        step = [v if v.rank == 2 else v.squeeze(1) for v in step]
        state.gated_step_inplace(*step)
    got = tp.cpu()
    # the scan associates the same products and sums otherwise than the steps do: each is within the bound of the exact states
    exact, tol = _scan_ref(x, a, 1, pool[:, 4:5, 8:24], False, False, U[np.float32])
    _close(h, exact, tol)
    _close(got[:, 4, 8:24], exact[:, -1], tol[:, -1])
    got[:, 4, 8:24] = pool[:, 4, 8:24]
    assert got.tobytes() == pool.tobytes()


def test_scan_refusals():
    import rtensors_b200 as rt
    from rtensors_b200.tensor import cross_entropy_loss, gated_scan_backward
    x, a = _t(np.ones((2, 3, 4), np.float32)), _t(np.ones((2, 3, 4), np.float32))
    i = _t(np.ones((2, 3, 4), np.int32))
    codes = []
    for call in (lambda: x.gated_scan_at(3, a), lambda: x.gated_scan_at(1, _t(np.ones((2, 3, 5), np.float32))),
                 lambda: x.gated_scan_at(1, _t(np.ones((3, 2, 3, 4), np.float32))), lambda: x.gated_scan_at(1, a, _t(np.ones((2, 3, 4), np.float32))),
                 lambda: x.gated_scan_at(1, _t(np.ones((2, 3, 4)))), lambda: i.gated_scan_at(1, i),
                 lambda: gated_scan_backward(x, 1, a, None), lambda: gated_scan_backward(x, 1, a, x, coupled=True),
                 lambda: gated_scan_backward(x, 1, a, _t(np.ones((2, 4), np.float32)).checkpoint8()),
                 lambda: i.checkpoint8(), lambda: x.checkpoint8().grad("cosh", x), lambda: x.checkpoint8().grad("mul", x.slice(0, 0, 1)),
                 lambda: cross_entropy_loss(x, i), lambda: cross_entropy_loss(x, _t(np.ones((2, 3), np.float32))),
                 lambda: cross_entropy_loss(x, _t(np.ones((2, 3), np.int32)), reduction="max"),
                 lambda: cross_entropy_loss(i, _t(np.ones((2, 3), np.int32)))):
        with pytest.raises(rt.RtbError) as e:
            call()
        codes.append(e.value.code)
    assert codes == [-5, -3, -3, -6, -2, -2, -6, -1, -6, -2, -1, -6, -6, -2, -1, -2]


# ---- 8-bit checkpoints ------------------------------------------------------------------------------------

def _codes_ref(x):
    flat = x.reshape(-1).astype(np.float64)
    v = np.zeros((-(-flat.size // 128), 128))
    v.reshape(-1)[: flat.size] = flat
    m = np.abs(v).max(axis=1, keepdims=True)
    with np.errstate(all="ignore"):
        c = np.where(m > 0, np.rint(127.0 * v / np.where(m > 0, m, 1)), 0)
        bad = ~np.isfinite(m[:, 0])
        c[bad] = 0
        m[bad] = np.nan
    return c.reshape(-1)[: flat.size], m[:, 0], (c * m / 127.0).reshape(-1)[: flat.size]


@DTYPES
@pytest.mark.parametrize("n", [1, 3, 4, 127, 128, 129, 4095, 4096, 4097, 100003])
def test_checkpoint_codes_restore_and_maps(dt, n):
    rng = np.random.default_rng(n)
    x = (rng.standard_normal(n) * np.exp(rng.standard_normal(n))).astype(dt)
    x[rng.integers(0, n, n // 7)] = 0
    if n > 600:
        x[128:256] = np.round(x[128:256] * 4)                         # ties: m = 127 k / 2
        x[130] = 127 * 4
        x[256:384] = 0
        x[384:512] *= np.finfo(dt).tiny * 3                           # magnitudes near and below the smallest normal
        x[512:600] *= np.finfo(dt).max / 1e6
    c, m, r = _codes_ref(x)
    ck = _t(x).checkpoint8()
    assert np.array_equal(ck.codes.cpu().numpy()[:n], c.astype(np.int8))
    assert np.array_equal(ck.mags.cpu().numpy()[: m.size].astype(np.float64), m)
    got = ck.restore().cpu()
    tiny = float(np.nextafter(dt(0), dt(1)))
    # one rounding of the kernel's; in f64 the restatement's product and quotient round too, by U each
    _close(got, r, (1.01 * U[dt] + 2 * U[np.float64]) * np.abs(r) + tiny)
    top = np.abs(x.reshape(-1)) == np.repeat(m, 128)[:n]
    assert np.array_equal(got[top], x[top])
    up = rng.standard_normal(n).astype(dt)
    r, u64 = got.astype(np.float64), up.astype(np.float64)
    with np.errstate(over="ignore"):
        maps = {"mul": r * u64, "square": 2 * r * u64}
        for kind, want in maps.items():
            fits = np.abs(want) < np.finfo(dt).max / 4
            _close(ck.grad(kind, _t(up)).cpu()[fits], want[fits], 2 * U[dt] * np.abs(want[fits]) + 2 * tiny)
    y = np.tanh(x).astype(dt)
    cy = _t(y).checkpoint8()
    ry = cy.restore().cpu().astype(np.float64)
    _close(cy.grad("tanh", _t(up)).cpu(), (1 - ry * ry) * u64, 4 * U[dt] * (1 + ry * ry) * np.abs(u64) + tiny)
    _close(cy.grad("sigmoid", _t(up)).cpu(), ry * (1 - ry) * u64, 4 * U[dt] * np.abs(ry) * (1 + np.abs(ry)) * np.abs(u64) + tiny)


@DTYPES
def test_checkpoint_of_masks_is_exact_and_non_finite_blocks_show(dt):
    rng = np.random.default_rng(2)
    mask = (rng.random(1000) < 0.5).astype(dt)
    assert np.array_equal(_t(mask).checkpoint8().restore().cpu(), mask)
    x = rng.standard_normal(640).astype(dt)
    x[130], x[300], x[511] = np.inf, np.nan, -np.inf
    r = _t(x).checkpoint8().restore().cpu()
    assert np.isnan(r[128:512]).all() and np.isfinite(r[:128]).all() and np.isfinite(r[512:]).all()


@DTYPES
def test_checkpoint_of_views(dt):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((37, 50)).astype(dt)
    for view, want in ((_t(x).transpose(), x.T), (_t(x).slice(0, 1, 30), x[1:30]), (_t(x).slice(1, None, None, -1), x[:, ::-1])):
        assert np.array_equal(view.checkpoint8().codes.cpu().numpy()[: want.size], _codes_ref(np.ascontiguousarray(want))[0])
    ck = _t(x.T.copy()).checkpoint8()
    up = rng.standard_normal((37, 50)).astype(dt)
    assert np.array_equal(ck.grad("mul", _t(up).transpose()).cpu(), ck.grad("mul", _t(up.T.copy())).cpu())


# ---- cross-entropy ----------------------------------------------------------------------------------------

def _ce_ref(x, t, mean, u):
    x = x.astype(np.float64)
    rows, classes = x.shape
    m = x.max(axis=1, keepdims=True)
    e = np.exp(x - m)
    s = e.sum(axis=1, keepdims=True)
    hit = np.arange(classes)[None, :] == t[:, None]
    ok = t >= 0
    n = ok.sum() if mean else 1
    # an entry 800 below the maximum has an exponential of zero in either type, in the kernel and here: it adds no error
    d = np.where(np.isfinite(x), np.maximum(x - m, -800), 0)
    # exp: the argument's rounding and a few units in its result; the sum: a chain of classes / 32 terms, each
    # rescaled at most once per term
    chain = 4 * (classes / 32 + 20)
    rel = u * (np.abs(d) + chain + 8 + np.abs(d).max(axis=1, keepdims=True))
    p = e / s
    g = np.where(ok[:, None], (p - hit) / n, 0)
    g_tol = np.where(ok[:, None], (p * rel + 4 * u * np.abs(p - hit)) / n, 0)
    xt = (np.where(np.isfinite(x), x - m, 0))[np.arange(rows), np.where(ok, t, 0)]
    per = np.where(ok, np.log(s[:, 0]) - xt, 0)
    per_tol = np.where(ok, rel.max(axis=1) + 4 * u * (np.abs(np.log(s[:, 0])) + np.abs(xt)), 0)
    return per.sum() / n, per_tol.sum() / n + 4 * u * abs(per.sum() / n), g, g_tol


@DTYPES
@pytest.mark.parametrize("rows,classes", [(1, 1), (1, 2), (5, 10), (4096, 10), (33, 31), (70, 32), (9, 1023), (9, 1024), (7, 1025), (3, 4100),
                                          (300, 2000), (2, 32768), (2, 50001), (3, 131072)])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_cross_entropy_and_its_map(dt, rows, classes, reduction):
    from rtensors_b200.tensor import cross_entropy_loss
    rng = np.random.default_rng(rows * 7 + classes)
    x = (rng.standard_normal((rows, classes)) * 3).astype(dt)
    t = rng.integers(0, classes, rows)
    if rows > 3:
        t[1::4] = -1 - np.arange(t[1::4].size)
        x[2, : classes // 2] = -np.inf                 # masked classes, the target among the others
        t[2] = classes - 1
        x[3] += 80
    loss_w, loss_tol, g_w, g_tol = _ce_ref(x, t, reduction == "mean", U[dt])
    for tt in (t.astype(np.int64), t.astype(np.int32)):
        loss, g = cross_entropy_loss(_t(x), _t(tt), True, reduction)
        _close(g.cpu(), g_w, g_tol)
        assert abs(float(loss.item()) - loss_w) <= loss_tol
    assert cross_entropy_loss(_t(x), _t(t), reduction=reduction).cpu().tobytes() == loss.cpu().tobytes()
    again = cross_entropy_loss(_t(x), _t(t), True, reduction)
    assert again[0].cpu().tobytes() == loss.cpu().tobytes() and again[1].cpu().tobytes() == g.cpu().tobytes()


@DTYPES
def test_cross_entropy_edges(dt):
    from rtensors_b200.tensor import cross_entropy_loss
    rng = np.random.default_rng(8)
    x = rng.standard_normal((6, 40)).astype(dt)
    none = np.full(6, -1)
    loss, g = cross_entropy_loss(_t(x), _t(none), True)
    assert np.isnan(loss.item()) and not g.cpu().any()
    loss, g = cross_entropy_loss(_t(x), _t(none), True, "sum")
    assert loss.item() == 0 and not g.cpu().any()
    t = np.arange(6)
    t[3] = 40                                           # one class too far: NaN there, the other rows as they are
    loss, g = cross_entropy_loss(_t(x), _t(t), True)
    g = g.cpu()
    assert np.isnan(loss.item()) and np.isnan(g[3]).all() and np.isfinite(np.delete(g, 3, 0)).all()
    x[1], x[2, 5], x[4, 7] = -np.inf, np.nan, np.inf
    t[3] = 0
    g = cross_entropy_loss(_t(x), _t(t), True)[1].cpu()
    assert np.isnan(g[[1, 2, 4]]).all() and np.isfinite(g[[0, 3, 5]]).all()
    x = rng.standard_normal((3, 4)).astype(dt)
    x[0, 1] = -np.inf
    loss, g = cross_entropy_loss(_t(x), _t(np.array([1, 0, 0])), True)      # the target itself is masked
    assert loss.item() == np.inf and np.isfinite(g.cpu()).all()
    e = _t(np.zeros((0, 5), dt))
    assert np.isnan(cross_entropy_loss(e, _t(np.zeros(0, np.int64))).item())


@DTYPES
def test_cross_entropy_of_views(dt):
    from rtensors_b200.tensor import cross_entropy_loss
    rng = np.random.default_rng(9)
    x = rng.standard_normal((8, 3, 21)).astype(dt)
    t = rng.integers(0, 21, (8, 3))
    want = _ce_ref(x.reshape(24, 21), t.reshape(-1), True, U[dt])
    loss, g = cross_entropy_loss(_t(x), _t(t), True)
    _close(g.cpu().reshape(24, 21), *want[2:])
    wide = rng.standard_normal((9, 40)).astype(dt)
    for view, v in ((_t(wide).slice(1, 3, 24), wide[:, 3:24]), (_t(wide).slice(0, None, None, -1), wide[::-1]), (_t(wide.T.copy()).transpose(), wide),
                    (_t(wide).slice(1, None, None, -1), wide[:, ::-1])):
        tt = rng.integers(0, v.shape[1], 9)
        want = _ce_ref(v, tt, True, U[dt])
        loss, g = cross_entropy_loss(view, _t(tt), True)
        _close(g.cpu(), *want[2:])
        assert abs(float(loss.item()) - want[0]) <= want[1]


# ---- together -----------------------------------------------------------------------------------------------

def _block(x, w, u, g_bias, t, h0, checkpoint8):
    """One recurrent layer and its loss on the tape -> (loss, gradients)."""
    from rtensors_b200 import grad
    from rtensors_b200.tensor import cross_entropy_loss_tracked
    b, n, d = x.shape
    with grad.enabled(checkpoint8=checkpoint8) as ctx:
        leaves = [w, u, g_bias, h0]
        for p in leaves:
            p.param()
        z = x.reshape((b * n, d)).matmul(w)
        gate = (z + g_bias).sigmoid().reshape((b, n, d))
        h = z.tanh().reshape((b, n, d)).gated_scan_at(1, gate, h0, coupled=True)
        y = (h * gate).reshape((b * n, d)).relu()
        loss = cross_entropy_loss_tracked(y.matmul(u), t)
        ctx.backwards(loss)
        return loss.item(), [p.grad.value.cpu() for p in leaves]


def _block_ref(x, w, u, g_bias, t, h0):
    x, w, u, g_bias, h0 = (torch.tensor(v, dtype=torch.float64, requires_grad=k > 0) for k, v in enumerate((x, w, u, g_bias, h0)))
    z = x.reshape(-1, x.shape[2]) @ w
    gate = torch.sigmoid(z + g_bias).reshape(x.shape)
    b = (1 - gate) * torch.tanh(z).reshape(x.shape)
    last, hs = h0[:, 0], []
    for s in range(x.shape[1]):
        last = gate[:, s] * last + b[:, s]
        hs.append(last)
    y = torch.relu((torch.stack(hs, 1) * gate).reshape(-1, x.shape[2]))
    loss = torch.nn.functional.cross_entropy(y @ u, torch.tensor(t), ignore_index=-1)
    loss.backward()
    return loss.item(), [v.grad.numpy() for v in (w, u, g_bias, h0)]


@pytest.mark.parametrize("dt", [np.float32, np.float64], ids=["f32", "f64"])
def test_recurrent_layer_trains_on_the_tape(dt):
    """Product, gates, recurrence, head and loss: every leaf's gradient against the same model in 64 bits; with 8-bit activations
    within what a step of the codes can do."""
    torch.backends.cuda.matmul.allow_tf32 = False
    rng = np.random.default_rng(12)
    b, n, d, c = 3, 70, 24, 11
    arrays = [rng.standard_normal((b, n, d)), rng.standard_normal((d, d)) / 5, rng.standard_normal((d, c)) / 3, rng.standard_normal((1, d)),
              rng.integers(0, c, b * n), rng.standard_normal((b, 1, d))]
    arrays = [v.astype(dt) if v.dtype.kind == "f" else v for v in arrays]
    arrays[4][5::9] = -1
    want_loss, want = _block_ref(*arrays)
    for checkpoint8 in (False, True):
        x, w, u, g_bias, t, h0 = (_t(v) for v in arrays)
        loss, grads = _block(x, w, u, g_bias, t, h0, checkpoint8)
        assert abs(loss - want_loss) <= 400 * U[dt] * abs(want_loss)         # the forward pass does not see the checkpoints
        # in full: sums of about a thousand terms; in 8 bits each saved value is off by m / 254 at most, which a product of
        # two or three saved values turns into a few hundredths of the gradient's size at the very most
        share = 0.05 if checkpoint8 else 4000 * U[dt]
        for got, ref in zip(grads, want):
            assert got.shape == ref.shape
            assert np.abs(got - ref).max() <= share * np.abs(ref).max()


def test_gradients_against_differences():
    """f64: d loss / d leaf by central differences through the tape's own forward pass."""
    from rtensors_b200.tensor import cross_entropy_loss
    rng = np.random.default_rng(13)
    shape, t = (2, 9, 5), rng.integers(0, 5, (2, 9))
    x, a, h0 = rng.standard_normal(shape), rng.uniform(0.1, 0.9, (2, 9, 1)), rng.standard_normal((2, 1, 5))

    def loss_of(x, a, h0):
        return cross_entropy_loss(_t(x).gated_scan_at(1, _t(a), _t(h0), reverse=True, coupled=True), _t(t)).item()
    from rtensors_b200 import grad
    from rtensors_b200.tensor import cross_entropy_loss_tracked
    leaves = [_t(v) for v in (x, a, h0)]
    with grad.enabled() as ctx:
        for p in leaves:
            p.param()
        ctx.backwards(cross_entropy_loss_tracked(leaves[0].gated_scan_at(1, leaves[1], leaves[2], reverse=True, coupled=True), _t(t)))
    for k, v in enumerate((x, a, h0)):
        got = leaves[k].grad.value.cpu()
        for i in rng.choice(v.size, 6, replace=False):
            args = [[q.copy() for q in (x, a, h0)] for _ in range(2)]
            eps = 1e-5
            args[0][k].reshape(-1)[i] += eps
            args[1][k].reshape(-1)[i] -= eps
            slope = (loss_of(*args[0]) - loss_of(*args[1])) / (2 * eps)
            # central differences: eps^2 of curvature, and 2^-53 / eps of cancellation
            assert abs(slope - got.reshape(-1)[i]) <= 1e-8


def test_tape_keeps_activations_in_eight_bits():
    from rtensors_b200 import grad
    from rtensors_b200.tensor import Checkpoint8, Tensor
    with grad.enabled(checkpoint8=True) as ctx:
        w = _t(np.ones((4, 6), np.float32)).param()
        x = _t(np.ones((4, 6), np.float32))
        s = (x * w).sigmoid()                        # x and the leaf stay as they are
        y = s * s
        h = y.gated_scan_at(1, s)
        kinds = {n.kind: n.saved for n in ctx.nodes.values()}
        assert isinstance(kinds["Sigmoid"]["result"], Checkpoint8) and isinstance(kinds["GatedScan"]["h"], Checkpoint8)
        assert isinstance(kinds["GatedScan"]["gate"], Tensor)
        muls = [n.saved for n in ctx.nodes.values() if n.kind == "BroadcastMul"]
        assert isinstance(muls[0]["lhs"], Tensor) and isinstance(muls[0]["rhs"], Tensor) and isinstance(muls[1]["lhs"], Checkpoint8)
        del h


def test_on_another_stream_and_in_a_graph():
    """The context follows torch's stream; a captured run replays on new inputs, two graphs one after the other."""
    from rtensors_b200.tensor import cross_entropy_loss, gated_scan_backward
    be = _b()
    rng = np.random.default_rng(14)
    x, a = rng.standard_normal((2, 700, 40)).astype(np.float32), rng.uniform(0, 1, (2, 700, 40)).astype(np.float32)
    t = rng.integers(0, 40, (2, 700))
    tx, ta, tt = _t(x), _t(a), _t(t)

    def passes():
        h = tx.gated_scan_at(1, ta)
        ck = h.checkpoint8()
        loss, g = cross_entropy_loss(h, tt, True)
        dx, dg, _ = gated_scan_backward(g, 1, ta, ck)
        return [h.buf, loss.buf, g.buf, dx.buf, dg.buf]
    want = [v.cpu().numpy().tobytes() for v in passes()]
    side = torch.cuda.Stream()
    try:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            be.sync_stream()
            got = passes()
        side.synchronize()
        assert [v.cpu().numpy().tobytes() for v in got] == want
        graphs, outs = [], []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
                be.sync_stream()
                outs.append(passes())
            graphs.append(g)
    finally:
        torch.cuda.current_stream().wait_stream(side)
        be.sync_stream()
    for k in (0, 1, 0):
        for v in outs[k]:
            v.zero_()
        graphs[k].replay()
        torch.cuda.synchronize()
        assert [v.cpu().numpy().tobytes() for v in outs[k]] == want
    tx.buf.mul_(2.0)
    graphs[0].replay()
    graphs[1].replay()
    torch.cuda.synchronize()
    new = [v.cpu().numpy().tobytes() for v in passes()]
    assert new != want
    for o in outs:
        assert [v.cpu().numpy().tobytes() for v in o] == new


# ---- far ends -------------------------------------------------------------------------------------------------

def test_offsets_beyond_32_bits():
    """Views that reach past 2^31 elements of a 9 GB buffer: the recurrence on the last channels of long rows, the loss of the last
    rows, the checkpoint of everything."""
    from rtensors_b200.meta import Meta
    from rtensors_b200.tensor import Tensor, cross_entropy_loss
    be, rows, width = _b(), 70001, 32768
    buf = torch.zeros(rows * width, device="cuda")
    rng = np.random.default_rng(15)
    tail = rng.standard_normal((rows, 5)).astype(np.float32)
    whole = Tensor(be, buf, Meta.contiguous((rows, width)))
    buf.view(rows, width)[:, -5:] = torch.from_numpy(tail).cuda()
    gate = np.full((1, 5), 0.75, np.float32)
    x = whole.slice(1, width - 5, width)
    got = x.gated_scan_at(0, _t(gate)).cpu()
    want, tol = _scan_ref(tail[-300:], gate, 0, None, False, False, U[np.float32])
    # 300 steps back nothing is left of earlier states: 0.75^300 < 1e-37
    _close(got[-100:], want[-100:], tol[-100:] + 1e-30)
    t = np.full(rows, -1)
    t[-2:] = width - 1, 7
    loss = cross_entropy_loss(whole, _t(t)).item()
    v = np.zeros((2, width))
    v[:, -5:] = tail[-2:]
    assert abs(loss - _ce_ref(v, t[-2:], True, U[np.float32])[0]) <= _ce_ref(v, t[-2:], True, U[np.float32])[1]
    ck = whole.checkpoint8()
    last = ck.restore().buf.view(rows, width)[-2:, -128:].cpu().numpy()
    assert np.array_equal(last[1], _codes_ref(v[1, -128:].astype(np.float32))[2].astype(np.float32)) and not last[0, :-5].any()
    del whole, x, ck, buf
    torch.cuda.empty_cache()


@DTYPES
@pytest.mark.parametrize("rows,classes", [(1, 262144), (2, 262149), (3, 140000), (2, 300001), (5, 2048), (40, 1536), (17, 8191)])
def test_cross_entropy_of_long_rows(dt, rows, classes):
    """Clusters of every size, and rows beyond them."""
    from rtensors_b200.tensor import cross_entropy_loss
    rng = np.random.default_rng(classes)
    x = (rng.standard_normal((rows, classes)) * 3).astype(dt)
    t = rng.integers(0, classes, rows)
    t[-1] = classes - 1
    if rows > 2:
        t[1] = -7
    loss_w, loss_tol, g_w, g_tol = _ce_ref(x, t, True, U[dt])
    loss, g = cross_entropy_loss(_t(x), _t(t), True)
    _close(g.cpu(), g_w, g_tol)
    assert abs(float(loss.item()) - loss_w) <= loss_tol


@DTYPES
@pytest.mark.parametrize("classes", [3, 40, 700, 1030, 20000, 40001])
def test_cross_entropy_of_extreme_logits(dt, classes):
    """Masks of the type's lowest value, alone and with others; logits near the type's largest; far from zero."""
    from rtensors_b200.tensor import cross_entropy_loss
    low, rng = np.finfo(dt).min, np.random.default_rng(classes)
    x = rng.standard_normal((7, classes)).astype(dt)
    t = rng.integers(0, classes, 7)
    x[0] = low                                  # nothing but masked: every class alike
    x[1, ::2] = low
    t[1] = 1
    x[2] = low
    x[2, t[2]] = 0                              # one class left
    x[3] = -low
    x[4] = np.where(np.arange(classes) == t[4], dt(3e37), dt(-3e37))
    x[5] += dt(1000)
    x[6] -= dt(1000)
    with np.errstate(over="ignore"):
        loss_w, loss_tol, g_w, g_tol = _ce_ref(x, t, False, U[dt])
    loss, g = cross_entropy_loss(_t(x), _t(t), True, "sum")
    # rows 5 and 6: the shift by 1000 has rounded the inputs themselves, exactly as the restatement reads them
    _close(g.cpu(), g_w, g_tol)
    assert abs(float(loss.item()) - loss_w) <= loss_tol + 4 * U[dt] * 1000


def test_cross_entropy_map_in_the_logits_place():
    from rtensors_b200._lib import check, lib
    be, rng = _b(), np.random.default_rng(16)
    for rows, classes in ((300, 7), (40, 100), (9, 1000), (30, 2049), (20, 5000), (7, 33001), (3, 150001), (2, 300000)):
        x = rng.standard_normal((rows, classes)).astype(np.float32)
        t = torch.from_numpy(rng.integers(-1, classes, rows)).cuda()
        a, loss = torch.from_numpy(x).cuda(), torch.zeros(2, device="cuda")
        out = torch.empty_like(a)
        for k, g in enumerate((out, a)):
            check(lib().rtb_cross_entropy(be._ctx, 10, a.data_ptr(), rows, classes, classes, t.data_ptr(), 0, loss.data_ptr() + 4 * k, g.data_ptr()))
        assert torch.equal(out, a) and float(loss[0]) == float(loss[1]) or bool((t < 0).all())


def test_two_contexts_at_once():
    """Two contexts on two streams, their calls interleaved: the same bits as one after the other."""
    from rtensors_b200.backend import CudaB200
    from rtensors_b200.meta import Meta
    from rtensors_b200.tensor import Tensor, cross_entropy_loss, gated_scan_backward
    rng = np.random.default_rng(17)
    x, a = rng.standard_normal((2, 3000, 96)).astype(np.float32), rng.uniform(0, 1, (2, 3000, 96)).astype(np.float32)
    t = rng.integers(0, 96, (2, 3000))

    def run(be):
        tx, ta, tt = (Tensor(be, torch.from_numpy(v).cuda().view(-1), Meta.contiguous(v.shape)) for v in (x, a, t))
        outs = []
        for _ in range(4):
            h = tx.gated_scan_at(1, ta)
            loss, g = cross_entropy_loss(h, tt, True)
            outs += [h.buf, loss.buf, g.buf, *(v.buf for v in gated_scan_backward(g, 1, ta, h.checkpoint8())[:2])]
        return outs
    want = [v.cpu().numpy().tobytes() for v in run(_b())]
    streams, backends, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            backends.append(CudaB200(0))
            outs.append(run(backends[-1]))
    torch.cuda.synchronize()
    for o in outs:
        assert [v.cpu().numpy().tobytes() for v in o] == want
    for b in backends:
        b.close()


def test_calls_follow_the_current_stream():
    """Without sync_stream: a call made under another stream is enqueued there, behind what that stream holds."""
    from rtensors_b200.backend import CudaB200
    from rtensors_b200.meta import Meta
    from rtensors_b200.tensor import Tensor, cross_entropy_loss
    rng = np.random.default_rng(18)
    be = CudaB200(0)
    x, a = rng.standard_normal((4, 500, 64)).astype(np.float32), rng.uniform(0, 1, (4, 500, 64)).astype(np.float32)
    tx, ta = (Tensor(be, torch.from_numpy(v).cuda().view(-1), Meta.contiguous(v.shape)) for v in (x, a))
    want = tx.gated_scan_at(1, ta).buf.clone() * 2      # linear: twice the input, twice the states
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)                   # some ten milliseconds
        tx.buf.mul_(2.0)
        got = tx.gated_scan_at(1, ta)
        ck = got.checkpoint8()
        loss = cross_entropy_loss(got, Tensor(be, torch.zeros(2000, dtype=torch.int64, device="cuda"), Meta.contiguous((4, 500))))
    side.synchronize()
    assert torch.equal(got.buf, want) and bool(torch.isfinite(loss.buf).all()) and bool((ck.codes != 0).any())
    torch.cuda.synchronize()
    be.close()


@DTYPES
@pytest.mark.parametrize("coupled,reverse,heads", [(False, False, 0), (True, True, 0), (False, True, 4), (True, False, 4)])
@pytest.mark.parametrize("shape", [(700, 16, 64), (257, 17, 132), (160, 61, 256), (400, 3, 1000), (40, 9, 31 * 4)])
def test_many_lanes_and_few_steps(dt, coupled, reverse, heads, shape):
    """Sizes where a thread walks its lanes alone, at whole vectors and odd ends; heads share a gate."""
    from rtensors_b200.tensor import gated_scan_backward
    b, n, d = shape
    full = (b, n, heads, d // heads) if heads else shape
    gate = (b, n, heads, 1) if heads else shape
    rng, x, a, first = _data(dt, full, gate, 1, True, seed=3)
    tx, ta, t0 = _t(x), _t(a), _t(first)
    _close(tx.gated_scan_at(1, ta, t0, reverse=reverse, coupled=coupled).cpu(), *_scan_ref(x, a, 1, first, reverse, coupled, U[dt]))
    up, h = rng.standard_normal(full).astype(dt), rng.standard_normal(full).astype(dt)
    ck = _t(h).checkpoint8()
    for kept, values in ((_t(h), h), (ck, ck.restore().cpu())):
        want = _scan_back_ref(up, a, 1, values, x, first, reverse, coupled, U[dt])
        got = gated_scan_backward(_t(up), 1, ta, kept, tx if coupled else None, t0, reverse, coupled)
        for g, w in zip(got, want):
            _close(g.cpu(), *w)


@pytest.mark.parametrize("d", [256, 255])
def test_very_many_lanes_agree_with_a_few_at_a_time(d):
    """Enough lanes that a thread walks each; the same lanes in parts go by rounds.  With gates of at most 0.9 and |values| <= 1 a
    state's A is 10 at most and E 2 u A / (1 - 0.9), so each way is within (20 + 24) u 10 of the exact states, twice that apart."""
    from rtensors_b200.meta import Meta
    from rtensors_b200.tensor import Tensor, gated_scan_backward
    be, b, n = _b(), 1250 if d == 256 else 320, 70
    g = torch.Generator(device="cuda")
    g.manual_seed(d)
    x, a, up, h = (torch.rand(b, n, d, device="cuda", generator=g) * 2 - 1 for _ in range(4))
    a = (a + 1) * 0.45

    def run(lo, hi):
        t = [Tensor(be, v[lo:hi].contiguous().view(-1), Meta.contiguous((hi - lo, n, d))) for v in (x, a, up, h)]
        states = t[0].gated_scan_at(1, t[1], coupled=True)
        dx, da, _ = gated_scan_backward(t[2], 1, t[1], t[3], t[0], coupled=True)
        return [v.buf.view(hi - lo, n, d) for v in (states, dx, da)]
    whole = run(0, b)
    for lo in range(0, b, 50):
        for got, part in zip(whole, run(lo, min(lo + 50, b))):
            # da multiplies by two values of at most 1 each
            assert float((got[lo: lo + 50] - part).abs().max()) <= 2 * 2 * 44 * 2.0 ** -24 * 10


@DTYPES
@pytest.mark.parametrize("coupled,reverse", [(False, False), (True, True)])
@pytest.mark.parametrize("shape,gate_shape,axis", [((1, 24001, 20), None, 1), ((1, 5000, 300), None, 1), ((1, 13001, 33), None, 1), ((2, 9000, 8, 16), (2, 9000, 8, 1), 1),
                                                   ((3, 1, 70003), None, 2), ((1, 1, 65536), None, 2), ((2, 4100, 640), (2, 4100, 1), 1)])
def test_few_lanes_and_many_steps(dt, coupled, reverse, shape, gate_shape, axis):
    """Sizes where clusters of every size up to the widest share a group of lanes."""
    from rtensors_b200.tensor import gated_scan_backward
    rng, x, a, first = _data(dt, shape, gate_shape or shape, axis, True, seed=5)
    tx, ta, t0 = _t(x), _t(a), _t(first)
    _close(tx.gated_scan_at(axis, ta, t0, reverse=reverse, coupled=coupled).cpu(), *_scan_ref(x, a, axis, first, reverse, coupled, U[dt]))
    up, h = rng.standard_normal(shape).astype(dt), rng.standard_normal(shape).astype(dt)
    ck = _t(h).checkpoint8()
    for kept, values in ((_t(h), h), (ck, ck.restore().cpu())):
        want = _scan_back_ref(up, a, axis, values, x, first, reverse, coupled, U[dt])
        got = gated_scan_backward(_t(up), axis, ta, kept, tx if coupled else None, t0, reverse, coupled)
        for g, w in zip(got, want):
            _close(g.cpu(), *w)
