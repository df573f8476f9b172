"""Gradients of layer norm where the rows' means lie far from 0, against the formula in fp64 with statistics of its own:
the mean that the forward pass keeps is rounded to fp32, which moves every x - mean of a row by up to 2^-24 of the mean.

Tolerances, u = 2^-24 and h = (x - mean) rstd: h is off by five roundings (x - mean in two steps, rstd's two, the
product) and by 2 u beside them, half of one where the mean is within a standard deviation of 0 and its rounding is let
stand, one where what it lost is summed from rounded differences."""
import zlib

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
F = np.float32
U = 2.0 ** -24
EPS = 1e-5


def _rng(*key):
    return np.random.RandomState(zlib.crc32(repr(key).encode()) & 0x7FFFFFFF)


def _within(got, want, tol, what):
    bad = ~(np.abs(got.astype(np.float64) - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3].tolist(), float((np.abs(got - want) / tol).max()))


def _reference(x, gy, w):
    x, gy = x.astype(np.float64), gy.astype(np.float64)
    r = 1 / np.sqrt(x.var(1, keepdims=True) + EPS)
    h, g = (x - x.mean(1, keepdims=True)) * r, gy * w
    eh = U * (5 * np.abs(h) + 2)
    c1, c2 = g.mean(1, keepdims=True), (g * h).mean(1, keepdims=True)
    # the gradient is a dozen roundings of terms no larger than these off, and by what h is
    size = np.abs(g) + np.abs(g).mean(1, keepdims=True) + np.abs(h) * np.abs(g * h).mean(1, keepdims=True)
    moved = eh * np.abs(c2) + np.abs(h) * (np.abs(g) * eh).mean(1, keepdims=True)
    gw, gb = (gy * h).sum(0), gy.sum(0)
    return ((r * (g - c1 - h * c2), r * (12 * U * size + moved)), (gw, (np.abs(gy) * (eh + 2 * U * np.abs(h))).sum(0) + U * np.abs(gw)),
            (gb, 2 * U * np.abs(gb) + 1e-15 * np.abs(gy).sum(0)))


SHAPES = [(1, 33), (3, 64), (6, 777), (5, 1000), (40, 1025), (33, 2048), (7, 4096), (2, 8192), (3, 8195), (2, 20001), (500, 96),
          (1100, 40), (1100, 130), (1100, 260), (1100, 777), (1100, 1024), (2049, 1537), (1030, 4096), (1030, 6001), (1030, 8192), (1030, 8195),
          (16500, 1024), (3000, 8192), (11000, 1537)]


@pytest.mark.parametrize("rows,width", SHAPES)
def test_gradients_of_rows_with_far_means(cl, rows, width):
    g = _rng("far mean", rows, width)
    # near, far on either side, and so far that the values themselves are steps of 1/16
    mean = np.choose(g.randint(0, 4, (rows, 1)), [0.1, 4096.3, -300.7, 1e6])
    x = (g.standard_normal((rows, width)) + mean).astype(F)
    gy, w = g.standard_normal((rows, width)).astype(F), (1 + 0.3 * g.standard_normal(width)).astype(F)
    X, GY, W = cl.ClTensor(x), cl.ClTensor(gy), cl.ClTensor(w)
    m, r = cl.ClTensor(), cl.ClTensor()
    cl.ClTensor().layerNorm(X, W, None, EPS, mean=m, rstd=r)
    wants = _reference(x, gy, w)
    got = [cl.ClTensor() for _ in range(3)]
    cl.layerNormBackward(*got, GY, X, W, m, r)
    for t, (want, tol), what in zip(got, wants, ("gx", "gw", "gb")):
        _within(t.float(), want, tol, (rows, width, what))
    # each by itself, and gx in place of either operand
    for i in range(3):
        only = cl.ClTensor()
        cl.layerNormBackward(*[only if j == i else None for j in range(3)], GY, X, W, m, r)
        assert np.array_equal(only.float(), got[i].float()), i
    gw, gb = cl.ClTensor(), cl.ClTensor()
    for place, other in ((GY.clone(), X), (X.clone(), GY)):
        cl.layerNormBackward(place, gw, gb, *((place, other) if other is X else (other, place)), W, m, r)
        assert np.array_equal(place.float(), got[0].float()) and np.array_equal(gw.float(), got[1].float()) and np.array_equal(gb.float(), got[2].float())


@pytest.mark.parametrize("rows,width", [(6, 300), (1100, 300), (3, 9000)])
def test_a_mean_of_ones_own_is_taken_as_it_is(cl, rows, width):
    """statistics that are not the row's own, rounded: the formula with what it is given"""
    g = _rng("own", rows, width)
    x, gy = (g.standard_normal((rows, width)) + 50).astype(F), g.standard_normal((rows, width)).astype(F)
    m, r = np.full(rows, 40.0, dtype=F), np.full(rows, 0.5, dtype=F)
    gx, gw = cl.ClTensor(), cl.ClTensor()
    cl.layerNormBackward(gx, gw, None, cl.ClTensor(gy), cl.ClTensor(x), None, cl.ClTensor(m), cl.ClTensor(r))
    h, g64 = (x.astype(np.float64) - 40) * 0.5, gy.astype(np.float64)
    c1, c2 = g64.mean(1, keepdims=True), (g64 * h).mean(1, keepdims=True)
    size = np.abs(g64) + np.abs(g64).mean(1, keepdims=True) + np.abs(h) * np.abs(g64 * h).mean(1, keepdims=True)
    _within(gx.float(), 0.5 * (g64 - c1 - h * c2), 12 * U * 0.5 * size, "gx")
    _within(gw.float(), (g64 * h).sum(0), 4 * U * np.abs(g64 * h).sum(0), "gw")


def test_gradients_of_far_views_and_of_rows_that_are_not_finite(cl):
    g = _rng("far views")
    x, gy = (g.standard_normal((60, 131)) + 4096).astype(F), g.standard_normal((60, 131)).astype(F)
    X = cl.ClTensor(60, 140).fill(-7.0).narrow(2, 4, 131)
    X.copy(cl.ClTensor(x))
    GY = cl.ClTensor(131, 60).fill(0.0).t()
    GY.copy(cl.ClTensor(gy))
    m, r, gx, gw, gb = (cl.ClTensor() for _ in range(5))
    cl.ClTensor().layerNorm(X, None, None, EPS, mean=m, rstd=r)
    cl.layerNormBackward(gx, gw, gb, GY, X, None, m, r)
    for t, (want, tol), what in zip((gx, gw, gb), _reference(x, gy, 1.0), ("gx", "gw", "gb")):
        _within(t.float(), want, tol, what)
    # infinities and NaN keep to their rows of gx
    x[7, 3], x[20, 5] = np.inf, np.nan
    X.copy(cl.ClTensor(x))
    cl.ClTensor().layerNorm(X, None, None, EPS, mean=m, rstd=r)
    cl.layerNormBackward(gx, None, gb, GY, X, None, m, r)
    got, rest = gx.float(), [i for i in range(60) if i not in (7, 20)]
    assert np.isnan(got[[7, 20]]).all()
    _within(got[rest], *_reference(x[rest], gy[rest], 1.0)[0], "the others")
