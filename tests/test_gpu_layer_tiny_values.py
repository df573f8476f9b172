"""Products of the layer operators with values below 2^-110 among others, whose parts do not hold all of their digits:
results keep theirs, wherever such values decide them, and a few of them cost little.

Tolerances: a sum of K products in any order is off by (K + 3) u sum |a||b|, u = 2^-24, a result of which parts were lost
by a rounding more; products below the smallest number count for nothing."""
import time
import zlib

import numpy as np
import pytest

from layer_shapes import GROUPED, LINEAR

pytestmark = pytest.mark.gpu
F = np.float32
U = 2.0 ** -24


def _values(rows, cols, *key):
    """ordinary values, between 1/2 and 2; some are far below 2^-110, and so is all of line 3; of line 5 all but the first,
    and of line 6 all are 0 but one of them"""
    g = np.random.RandomState(zlib.crc32(repr(key + (rows, cols)).encode()) & 0x7FFFFFFF)
    v = g.choice([-1.0, 1.0], (rows, cols)) * g.uniform(0.5, 2, (rows, cols))
    low = g.choice([-1.0, 1.0], (rows, cols)) * 2.0 ** g.uniform(-125, -109, (rows, cols))
    v = np.where(g.uniform(0, 1, (rows, cols)) < 0.02, low, v)
    if rows > 6:
        v[3], v[5, 1:], v[6] = low[3], low[5, 1:], 0
        v[6, cols // 2] = low[6, cols // 2]
    return v.astype(F)


def _check(got, a, b, what):
    a, b = a.astype(np.float64), b.astype(np.float64)
    want, tol = a @ b, (a.shape[1] + 4) * U * (np.abs(a) @ np.abs(b)) + a.shape[1] * 2.0 ** -149
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4].tolist(), want[bad][:4].tolist())


@pytest.mark.parametrize("rows,inner,outer", [s for s in LINEAR if s[0] >= 33])
def test_linear_keeps_the_digits_of_tiny_values(cl, rows, inner, outer):
    x, w, gy = _values(rows, inner, "x"), _values(outer, inner, "w"), _values(rows, outer, "gy")
    # line 5 of x has one ordinary value, which meets nothing; the same for the gradients
    w[:, 0] = 0
    gy[0] = 0
    X, W, GY = cl.ClTensor(x), cl.ClTensor(w), cl.ClTensor(gy)
    _check(cl.ClTensor().linear(X, W).float(), x, w.T, "y")
    gx, gw, gx1, gw1 = (cl.ClTensor() for _ in range(4))
    cl.linearBackward(gx, gw, None, GY, X, W)
    cl.linearBackward(gx1, None, None, GY, X, W)
    cl.linearBackward(None, gw1, None, GY, X, W)
    for got, what in ((gx, "gx"), (gx1, "gx alone")):
        _check(got.float(), gy, w, what)
    for got, what in ((gw, "gw"), (gw1, "gw alone")):
        _check(got.float(), gy.T, x, what)


@pytest.mark.parametrize("rows,inner,outer,sizes", [s for s in GROUPED if s[0] >= 90])
def test_groupedmm_keeps_the_digits_of_tiny_values(cl, rows, inner, outer, sizes):
    x, gy = _values(rows, inner, "x"), _values(rows, outer, "gy")
    w = np.stack([_values(inner, outer, "w", g) for g in range(len(sizes))]) if inner * outer * len(sizes) < 3e7 else \
        np.repeat(_values(inner, outer, "w")[None], len(sizes), 0)
    w[:, 0] = 0
    X, W, GY = cl.ClTensor(x), cl.ClTensor(w), cl.ClTensor(gy)
    y, gx, gw = cl.ClTensor(rows, outer).fill(0.0), cl.ClTensor(rows, inner).fill(0.0), cl.ClTensor()
    y.groupedmm(X, W, sizes)
    cl.groupedmmBackward(gx, gw, GY, X, W, sizes)
    Y, GX, GW, at = y.float(), gx.float(), gw.float(), 0
    for k, n in enumerate(sizes):
        r = slice(at, at + n)
        at += n
        _check(Y[r], x[r], w[k], ("y", k))
        _check(GX[r], gy[r], w[k].T, ("gx", k))
        _check(GW[k], x[r].T, gy[r], ("gw", k))


def test_large_values_beside_tiny_ones(cl):
    """the largest value of a tile decides what tiny ones may lose"""
    g = np.random.RandomState(9)
    x, w = _values(300, 400, "large"), _values(260, 400, "large")
    x[40, 7], w[9, 11], w[3] = 1e30, -3e37, (2.0 ** g.uniform(90, 110, 400)).astype(F)
    w[3, 7] = 1                                                  # 1e30 2^110 is no number of fp32
    _check(cl.ClTensor().linear(cl.ClTensor(x), cl.ClTensor(w)).float(), x, w.T, "y")


def test_one_tiny_value_in_each_row_costs_little(cl):
    """taking all of it again takes eleven times as long as the product"""
    rows, inner, outer = 2048, 2048, 2048
    g = np.random.RandomState(1)
    x, w = g.standard_normal((rows, inner)).astype(F), g.standard_normal((outer, inner)).astype(F)
    low = x.copy()
    low[:, 7] = 1e-35
    y, W = cl.ClTensor(rows, outer), cl.ClTensor(w)
    best = []
    for a in (x, low):
        A, times = cl.ClTensor(a), []
        for _ in range(12):
            cl.synchronize()
            t = time.perf_counter()
            y.linear(A, W)
            cl.synchronize()
            times.append(time.perf_counter() - t)
        best.append(min(times))
    _check(y.float(), low, w.T, "y")
    assert best[1] < 4 * best[0], best
