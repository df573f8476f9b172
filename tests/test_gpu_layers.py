"""GPU parity of the layer operators (layer norm, linear layer, grouped matrix products, forward and backward) against
plain fp64 numpy forms.

Tolerances follow from the arithmetic, u = 2^-24 being fp32's rounding error relative to a value.  A sum of K products
accumulated in fp32 in any order is off by at most about (K + 3) u sum |a||b|, element by element; for independent
entries of random sign the error's norm grows like sqrt(K) u instead (a running sum after j of K terms has size
sqrt(j), each addition rounds it by 0.58 u rms, which makes 0.41 sqrt(K) u of the result's norm), and twice that model
is what whole results are held to.  An activation scales its input's error by its largest slope (1.13) and adds a few
roundings of its own."""
import math
import zlib

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
F = np.float32
U = 2.0 ** -24
EPS = 1e-5


def _rng(*key):
    return np.random.RandomState(zlib.crc32(repr(key).encode()) & 0x7FFFFFFF)


def _normal(rng, *shape, scale=1.0, mean=0.0):
    return (rng.randn(*shape) * scale + mean).astype(F)


def _padded(cl, arr, before=3, after=5):
    """arr as a view of a wider buffer, odd offset and pitch; returns (view, buffer)."""
    r, c = arr.shape
    buf = cl.ClTensor(r, c + before + after).fill(-77.0)
    view = buf.narrow(2, before + 1, c)
    view.copy(cl.ClTensor(arr))
    return view, buf


def _erfc(z):
    return np.vectorize(math.erfc, otypes=[float])(z)


def _act(name, z):
    if name == "relu":
        return np.where(z < 0, 0.0, z)
    if name == "gelu":
        return 0.5 * z * _erfc(-z / math.sqrt(2))
    if name == "silu":
        return z / (1 + np.exp(-z))
    return z


def _slope(name, z):
    if name == "relu":
        return (z > 0).astype(np.float64)
    if name == "gelu":
        return 0.5 * _erfc(-z / math.sqrt(2)) + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        s = 1 / (1 + np.exp(-z))
        return s * (1 + z * (1 - s))
    return np.ones_like(z)


def _within(got, want, tol, what):
    bad = ~(np.abs(got.astype(np.float64) - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3].tolist(), float(np.abs(got - want).max()))


def _norm_within(got, want, depth, what):
    """The sqrt(K) model of the header; 16 keeps short sums from being held to less than a few roundings."""
    rel = np.linalg.norm(got.astype(np.float64) - want) / max(np.linalg.norm(want), 1e-300)
    assert rel <= 0.82 * math.sqrt(max(depth, 16)) * U, (what, rel, depth)


# ------------------------------------------------------------------ layer norm ---
NORM_SHAPES = [(1, 1), (3, 1), (1, 2), (2, 5), (7, 63), (5, 64), (4, 65), (1, 255), (3, 256), (2, 257), (9, 1000), (3, 1023), (2, 1024),
               (5, 1025), (1, 4096), (300, 96), (17, 2047), (3, 4099), (2, 8192), (2, 8195), (2, 20001), (1, 70000), (2000, 33)]


def _norm_reference(x, w, b):
    x = x.astype(np.float64)
    mean = x.mean(-1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + EPS)
    h = (x - mean) * rstd
    return mean[..., 0], rstd[..., 0], h, h * w + b


def _check_norm(x, w, b, y, mean, rstd, what):
    m, r, h, want = _norm_reference(x, w, b)
    # x - mean rounds twice, rstd three times (the variance's terms once each on average), the product and the sum once
    _within(y, want, U * (7 * np.abs(h * w) + 2 * np.abs(want)) + 1e-37, (what, "y"))
    _within(mean, m, U * np.abs(m) + 1e-37, (what, "mean"))
    _within(rstd, r, 4 * U * r, (what, "rstd"))


@pytest.mark.parametrize("rows,width", NORM_SHAPES)
def test_layer_norm_forward(cl, rows, width):
    g = _rng("norm", rows, width)
    x = _normal(g, rows, width, scale=2.0, mean=1.5)
    w, b = _normal(g, width, scale=0.3, mean=1.0), _normal(g, width, scale=0.2)
    y, mean, rstd = cl.ClTensor(), cl.ClTensor(), cl.ClTensor()
    assert y.layerNorm(cl.ClTensor(x), cl.ClTensor(w), cl.ClTensor(b), EPS, mean=mean, rstd=rstd) is y
    _check_norm(x, w, b, y.float(), mean.float(), rstd.float(), (rows, width))
    again = cl.ClTensor().layerNorm(cl.ClTensor(x), cl.ClTensor(w), cl.ClTensor(b), EPS)
    assert np.array_equal(again.float().view(np.uint32), y.float().view(np.uint32))


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
def test_layer_norm_without_weight_or_bias_in_place_and_far_mean(cl, weight, bias):
    g = _rng("plain", weight, bias)
    x = _normal(g, 6, 777, mean=4096.0)          # the mean is far larger than what varies around it
    w, b = _normal(g, 777, mean=1.0), _normal(g, 777)
    X = cl.ClTensor(x)
    X.layerNorm(X, cl.ClTensor(w) if weight else None, cl.ClTensor(b) if bias else None)
    ones, zeros = np.ones(777), np.zeros(777)
    want = _norm_reference(x, w if weight else ones, b if bias else zeros)
    _within(X.float(), want[3], U * (7 * np.abs(want[2] * (w if weight else ones)) + 2 * np.abs(want[3])), "in place")


def test_layer_norm_views_shapes_and_what_it_leaves_alone(cl):
    g = _rng("views")
    x, w, b = _normal(g, 10, 131), _normal(g, 131), _normal(g, 131)
    xv, _ = _padded(cl, x)
    yv, ybuf = _padded(cl, np.zeros_like(x))
    W = cl.ClTensor(np.repeat(w, 2)).strided([131], [2], 1)
    B = cl.ClTensor(np.repeat(b, 3)).strided([131], [3], 1)
    mean = cl.ClTensor(30).fill(5.0).strided([10], [3], 1)
    yv.layerNorm(xv, W, B, EPS, mean=mean)
    want = _norm_reference(x, w, b)
    _within(yv.float(), want[3], U * (7 * np.abs(want[2] * w) + 2 * np.abs(want[3])), "views")
    _within(mean.float(), want[0], U * np.abs(want[0]) + 1e-37, "strided mean")
    out = ybuf.float()
    assert (out[:, :3] == -77).all() and (out[:, 134:] == -77).all()
    # more dimensions, one row as a vector, transposed input and result
    x3 = _normal(g, 3, 4, 50)
    for X in (cl.ClTensor(x3), cl.ClTensor(np.ascontiguousarray(x3.transpose(1, 0, 2))).transpose(1, 2), cl.ClTensor(np.ascontiguousarray(x3.transpose(0, 2, 1))).transpose(2, 3)):
        y, rstd = cl.ClTensor(), cl.ClTensor()
        y.layerNorm(X, rstd=rstd)
        m, r, h, _ = _norm_reference(x3, 1.0, 0.0)
        assert y.size() == (3, 4, 50) and rstd.size() == (3, 4)
        _within(y.float(), h, 9 * U * np.abs(h) + 1e-37, "3d")
        _within(rstd.float(), r, 4 * U * r, "3d rstd")
    yt = cl.ClTensor(50, 12).fill(0.0).t()
    yt.layerNorm(cl.ClTensor(x3.reshape(12, 50)))
    _within(yt.float(), h.reshape(12, 50), 9 * U * np.abs(h.reshape(12, 50)) + 1e-37, "transposed result")
    v = cl.ClTensor()
    mean = cl.ClTensor()
    v.layerNorm(cl.ClTensor(x3[0, 0]), mean=mean)
    assert v.size() == (50,) and mean.size() == (1,)
    # expanded rows
    e = cl.ClTensor().layerNorm(cl.ClTensor(x3[:1, 0]).expand(4, 50)).float()
    assert (e == e[0]).all()


def test_layer_norm_constant_rows_and_rows_with_infinities_keep_to_themselves(cl):
    g = _rng("inf")
    x = _normal(g, 5, 300)
    x[1] = 3.25                     # nothing varies: the normalised row is zero
    x[2, 7] = np.inf
    x[3, 9] = np.nan
    b = _normal(g, 300)
    y = cl.ClTensor().layerNorm(cl.ClTensor(x), None, cl.ClTensor(b)).float()
    assert np.array_equal(y[1], b)
    assert np.isnan(y[2]).all() and np.isnan(y[3]).all()
    want = _norm_reference(x[[0, 4]], 1.0, b)
    _within(y[[0, 4]], want[3], U * (7 * np.abs(want[2]) + 2 * np.abs(want[3])), "the others")


def _norm_backward_reference(gy, x, w, mean, rstd):
    gy, x, mean, rstd = (a.astype(np.float64) for a in (gy, x, mean[:, None], rstd[:, None]))
    h, g = (x - mean) * rstd, gy * w
    c1, c2 = g.mean(1, keepdims=True), (g * h).mean(1, keepdims=True)
    gx = rstd * (g - c1 - h * c2)
    # errors: h by its two roundings, g by one, the means by their terms' and one of their own
    eh = 3 * U * np.abs(h)
    e2 = (np.abs(g) * eh + 3 * U * np.abs(g * h)).mean(1, keepdims=True) + U * np.abs(c2)
    e1 = U * np.abs(g).mean(1, keepdims=True) + U * np.abs(c1)
    tx = rstd * (3 * U * np.abs(g) + e1 + 2 * U * np.abs(c1) + np.abs(h) * e2 + np.abs(c2) * eh + 3 * U * np.abs(h * c2)) + 4 * U * np.abs(gx)
    tw = (np.abs(gy) * eh + 2 * U * np.abs(gy * h)).sum(0)
    return gx, (gy * h).sum(0), gy.sum(0), tx, tw


@pytest.mark.parametrize("rows,width", NORM_SHAPES)
def test_layer_norm_backward(cl, rows, width):
    g = _rng("norm backward", rows, width)
    x, gy, w = _normal(g, rows, width, scale=2.0, mean=0.5), _normal(g, rows, width), _normal(g, width, scale=0.3, mean=1.0)
    X, W, GY = cl.ClTensor(x), cl.ClTensor(w), cl.ClTensor(gy)
    mean, rstd = cl.ClTensor(), cl.ClTensor()
    cl.ClTensor().layerNorm(X, W, None, EPS, mean=mean, rstd=rstd)
    gx, gw, gb = cl.ClTensor(), cl.ClTensor(), cl.ClTensor()
    cl.layerNormBackward(gx, gw, gb, GY, X, W, mean, rstd)
    wx, ww, wb, tx, tw = _norm_backward_reference(gy, x, w, mean.float(), rstd.float())
    assert gx.size() == x.shape and gw.size() == (width,) and gb.size() == (width,)
    _within(gx.float(), wx, tx + 1e-37, (rows, width, "gx"))
    _within(gw.float(), ww, tw + U * np.abs(ww) + 1e-37, (rows, width, "gw"))
    _within(gb.float(), wb, 2 * U * np.abs(wb) + 1e-15 * np.abs(gy).sum(0), (rows, width, "gb"))
    # each result by itself is the same, also in place of gradOutput and of the input
    only = [cl.ClTensor() for _ in range(3)]
    for i in range(3):
        cl.layerNormBackward(*[only[j] if j == i else None for j in range(3)], GY, X, W, mean, rstd)
    for a, b in zip(only, (gx, gw, gb)):
        assert np.array_equal(a.float().view(np.uint32), b.float().view(np.uint32))
    G2, X2 = GY.clone(), X.clone()
    cl.layerNormBackward(G2, gw, gb, G2, X, W, mean, rstd)
    cl.layerNormBackward(X2, None, None, GY, X2, W, mean, rstd)
    assert np.array_equal(G2.float(), gx.float()) and np.array_equal(X2.float(), gx.float())
    assert np.array_equal(gw.float(), only[1].float())


def test_layer_norm_backward_views(cl):
    g = _rng("backward views")
    x, gy = _normal(g, 40, 77), _normal(g, 40, 77)
    xv, _ = _padded(cl, x)
    gv, _ = _padded(cl, gy, 1, 2)
    gxv, gbuf = _padded(cl, np.zeros_like(x), 4, 1)
    gwv = cl.ClTensor(154).fill(9.0).strided([77], [2], 1)
    mean, rstd = cl.ClTensor(), cl.ClTensor()
    cl.ClTensor().layerNorm(xv, mean=mean, rstd=rstd)
    cl.layerNormBackward(gxv, gwv, None, gv, xv, None, mean, rstd)
    wx, ww, wb, tx, tw = _norm_backward_reference(gy, x, 1.0, mean.float(), rstd.float())
    _within(gxv.float(), wx, tx, "gx")
    _within(gwv.float(), ww, tw + U * np.abs(ww), "gw")
    out = gbuf.float()
    assert (out[:, :4] == -77).all() and (out[:, 81:] == -77).all()
    # a gradient that is the same for every row and column: one element, expanded
    one = cl.ClTensor(np.full((1, 1), 0.5, dtype=F)).expand(40, 77)
    gb = cl.ClTensor()
    cl.layerNormBackward(None, None, gb, one, xv, None, mean, rstd)
    assert (gb.float() == 20.0).all()


def test_layer_norm_gradient_against_differences(cl):
    g = _rng("differences")
    x, w, b, gy = _normal(g, 3, 20), _normal(g, 20, mean=1.0), _normal(g, 20), _normal(g, 3, 20)
    mean, rstd, gx, gw = (cl.ClTensor() for _ in range(4))
    cl.ClTensor().layerNorm(cl.ClTensor(x), cl.ClTensor(w), cl.ClTensor(b), EPS, mean=mean, rstd=rstd)
    cl.layerNormBackward(gx, gw, None, cl.ClTensor(gy), cl.ClTensor(x), cl.ClTensor(w), mean, rstd)
    loss = lambda xx: float((_norm_reference(xx, w, b)[3] * gy).sum())  # noqa: E731
    step = 1e-5
    for i, j in [(0, 0), (1, 7), (2, 19)]:
        up, down = x.astype(np.float64), x.astype(np.float64)
        up[i, j] += step
        down[i, j] -= step
        want = (loss(up) - loss(down)) / (2 * step)
        # the difference's own error: a third derivative of order 100 times step^2 / 6, and fp64 noise over the step
        assert abs(gx.float()[i, j] - want) <= 1e-6 * np.abs(gy).max() * 10


# ---------------------------------------------------------------- linear layer ---
LINEAR_SHAPES = [(1, 1, 1), (1, 2, 3), (3, 1, 2), (2, 3, 1), (1, 64, 64), (5, 17, 33), (8, 100, 64), (16, 256, 130), (17, 31, 257),
                 (33, 1000, 65), (64, 512, 128), (65, 129, 255), (100, 77, 300), (128, 256, 256), (130, 1027, 131), (257, 48, 260),
                 (300, 513, 512), (1, 4096, 515), (2, 2050, 1025), (7, 1536, 640), (512, 16, 512), (31, 8200, 40), (600, 260, 1)]


def _linear_tolerance(x, w, depth):
    return (depth + 3) * U * (np.abs(x).astype(np.float64) @ np.abs(w).astype(np.float64).T)


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("rows,inner,outer", LINEAR_SHAPES)
def test_linear_forward(cl, rows, inner, outer, act):
    g = _rng("linear", rows, inner, outer)
    x, w = _normal(g, rows, inner), _normal(g, outer, inner, scale=inner ** -0.5)
    b, r = _normal(g, outer), _normal(g, rows, outer)
    X, W = cl.ClTensor(x), cl.ClTensor(w)
    z = x.astype(np.float64) @ w.astype(np.float64).T + b
    tol = _linear_tolerance(x, w, inner) + 2 * U * np.abs(z)
    want = _act(act, z) + r
    pre, y = cl.ClTensor(), cl.ClTensor()
    assert y.linear(X, W, cl.ClTensor(b), residual=cl.ClTensor(r), activation=act, preact=pre) is y
    _within(pre.float(), z, tol, "preact")
    _within(y.float(), want, 1.13 * tol + 8 * U * np.abs(_act(act, z)) + U * np.abs(want) + 1e-37, "y")
    plain = cl.ClTensor().linear(X, W).float()
    product = x.astype(np.float64) @ w.astype(np.float64).T
    _within(plain, product, _linear_tolerance(x, w, inner), "no epilogue")
    _norm_within(plain, product, inner, "no epilogue")
    # in the residual's place
    R = cl.ClTensor(r)
    R.linear(X, W, cl.ClTensor(b), residual=R, activation=act)
    assert np.array_equal(R.float().view(np.uint32), y.float().view(np.uint32))


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("rows,inner,outer", LINEAR_SHAPES)
def test_linear_backward(cl, rows, inner, outer, act):
    g = _rng("linear backward", rows, inner, outer)
    x, w, gy = _normal(g, rows, inner), _normal(g, outer, inner, scale=inner ** -0.5), _normal(g, rows, outer)
    z = _normal(g, rows, outer, scale=1.5)
    X, W, GY, Z = (cl.ClTensor(a) for a in (x, w, gy, z))
    gx, gw, gb = cl.ClTensor(), cl.ClTensor(), cl.ClTensor()
    cl.linearBackward(gx, gw, gb, GY, X, W, preact=None if act == "none" else Z, activation=act)
    slope = _slope(act, z.astype(np.float64))
    gz = gy * slope
    # a slope of size up to 1.13 is a few roundings off, absolutely: its terms cancel where it is small
    ez = 0.0 if act in ("none", "relu") else np.abs(gy) * 10 * U * 1.5 + U * np.abs(gz)
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    az = np.abs(gz)
    tx = (outer + 3) * U * (az @ np.abs(w64)) + (ez @ np.abs(w64) if act in ("gelu", "silu") else 0) + 1e-37
    tw = (rows + 3) * U * (az.T @ np.abs(x64)) + (ez.T @ np.abs(x64) if act in ("gelu", "silu") else 0) + 1e-37
    _within(gx.float(), gz @ w64, tx, "gx")
    _within(gw.float(), gz.T @ x64, tw, "gw")
    _within(gb.float(), gz.sum(0), (ez.sum(0) if act in ("gelu", "silu") else 0) + 2 * U * np.abs(gz.sum(0)) + 1e-15 * az.sum(0) + 1e-37, "gb")
    if act == "none":
        _norm_within(gx.float(), gz @ w64, outer, "gx")
        _norm_within(gw.float(), gz.T @ x64, rows, "gw")
    only = [cl.ClTensor() for _ in range(3)]
    for i in range(3):
        cl.linearBackward(*[only[j] if j == i else None for j in range(3)], GY, X, W, preact=Z, activation=act)
    # together they may share a launch, whose sums are cut at other places than those of a product by itself
    _within(only[0].float(), gz @ w64, tx, "gx alone")
    _within(only[1].float(), gz.T @ x64, tw, "gw alone")
    assert np.array_equal(only[2].float().view(np.uint32), gb.float().view(np.uint32))
    again = [cl.ClTensor() for _ in range(3)]
    cl.linearBackward(*again, GY, X, W, preact=Z, activation=act)
    for a, b in zip(again, (gx, gw, gb)):
        assert np.array_equal(a.float().view(np.uint32), b.float().view(np.uint32))


@pytest.mark.parametrize("rows,inner,outer", [(1, 37, 70), (6, 130, 67), (40, 129, 131), (150, 260, 200)])
def test_linear_views(cl, rows, inner, outer):
    g = _rng("linear views", rows, inner, outer)
    x, w, b = _normal(g, rows, inner), _normal(g, outer, inner), _normal(g, outer)
    want = x.astype(np.float64) @ w.astype(np.float64).T + b
    tol = _linear_tolerance(x, w, inner) + 2 * U * np.abs(want)
    xv, _ = _padded(cl, x)
    weights = {"padded": _padded(cl, w, 1, 1)[0], "transposed": cl.ClTensor(np.ascontiguousarray(w.T)).t(),
               "every second": cl.ClTensor(np.repeat(w, 2, axis=1)).strided([outer, inner], [2 * inner, 2], 1)}
    B = cl.ClTensor(np.repeat(b, 3)).strided([outer], [3], 1)
    gy = _normal(g, rows, outer)
    gv, _ = _padded(cl, gy, 2, 2)
    for name, W in weights.items():
        yv, ybuf = _padded(cl, np.zeros((rows, outer), dtype=F), 2, 3)
        zt = cl.ClTensor(outer, rows).fill(0.0).t()
        yv.linear(xv, W, B, preact=zt)
        _within(yv.float(), want, tol, name)
        _within(zt.float(), want, tol, name)
        out = ybuf.float()
        assert (out[:, :2] == -77).all() and (out[:, outer + 2:] == -77).all()
        gxv, gbuf = _padded(cl, np.zeros_like(x))
        gwt = cl.ClTensor(inner, outer).fill(0.0).t()
        cl.linearBackward(gxv, gwt, None, gv, xv, W)
        g64 = gy.astype(np.float64)
        _within(gxv.float(), g64 @ w, (outer + 3) * U * (np.abs(g64) @ np.abs(w)), name)
        _within(gwt.float(), g64.T @ x, (rows + 3) * U * (np.abs(g64).T @ np.abs(x)), name)
        out = gbuf.float()
        assert (out[:, :3] == -77).all() and (out[:, inner + 3:] == -77).all()
    # [batch, time, features], features last but not dense in front, and a single vector
    x3 = np.stack([x, 2 * x])
    X3 = cl.ClTensor(np.ascontiguousarray(x3.transpose(1, 0, 2))).transpose(1, 2)
    y3 = cl.ClTensor().linear(X3, weights["padded"], B)
    assert y3.size() == (2, rows, outer)
    _within(y3.float()[0], want, tol, "3d")
    v = cl.ClTensor().linear(cl.ClTensor(x[0]), weights["transposed"], B)
    assert v.size() == (outer,)
    _within(v.float(), want[0], tol[0], "vector")
    # a bias and an input that repeat, and a broadcast gradient
    e = cl.ClTensor().linear(cl.ClTensor(x[:1]).expand(5, inner), weights["padded"], cl.ClTensor(b[:1]).expand(outer)).float()
    _within(e, np.repeat(want[:1] - b + b[0], 5, 0), np.repeat(tol[:1], 5, 0) + 4 * U * (np.abs(b) + np.abs(b[0])), "expanded")
    gw, gb = cl.ClTensor(), cl.ClTensor()
    cl.linearBackward(None, gw, gb, cl.ClTensor(np.full((1, 1), 0.25, dtype=F)).expand(rows, outer), xv, weights["padded"])
    assert (gb.float() == 0.25 * rows).all()
    s = 0.25 * x.astype(np.float64).sum(0)
    _within(gw.float(), np.repeat(s[None], outer, 0), (rows + 3) * U * np.abs(x).sum(0), "broadcast gradient")


@pytest.mark.parametrize("rows,inner,outer", [(3, 40, 70), (20, 300, 150), (140, 270, 300)])
def test_linear_with_infinities_huge_and_tiny_values(cl, rows, inner, outer):
    g = _rng("inf", rows, inner, outer)
    x, w = _normal(g, rows, inner), _normal(g, outer, inner)
    x[1, 3] = np.inf
    w[5, 4] = -np.inf
    x[0, 7] = np.nan
    got = cl.ClTensor().linear(cl.ClTensor(x), cl.ClTensor(w)).float()
    with np.errstate(invalid="ignore"):
        want = x.astype(np.float64) @ w.astype(np.float64).T
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isposinf(got), np.isposinf(want))
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    fine = np.isfinite(want)
    xc, wc = np.where(np.isfinite(x), x, 0), np.where(np.isfinite(w), w, 0)
    _within(np.where(fine, got, 0), np.where(fine, want, 0), _linear_tolerance(xc, wc, inner), "beside infinities")
    # the largest and smallest magnitudes of normal numbers
    for sx, sw in ((1e37, 1e-3), (1e-30, 1.0), (1e-36, 1e10), (3.3e38, 1e-38)):
        a, b = np.clip(_normal(g, rows, inner), -1, 1) * F(sx), _normal(g, outer, inner) * F(sw)
        a[np.abs(a) < 1.2e-38] = 0
        b[np.abs(b) < 1.2e-38] = 0
        got = cl.ClTensor().linear(cl.ClTensor(a), cl.ClTensor(b)).float()
        want = a.astype(np.float64) @ b.astype(np.float64).T
        # 1e-38 per term: products and sums below the normal range may round to its grid or to zero
        _within(got, want, _linear_tolerance(a, b, inner) + inner * 1.2e-38, (sx, sw))
    # a finite product that overflows on the way to a finite sum is an infinity or NaN in fp32, never a finite wrong value
    a, b = np.full((1, 4), 3e38, dtype=F), np.array([[1, 1, -1, -1]], dtype=F)
    got = cl.ClTensor().linear(cl.ClTensor(a), cl.ClTensor(b)).float()
    assert not np.isfinite(got[0, 0]) or got[0, 0] == 0


# ------------------------------------------------------------ grouped products ---
GROUPED = [(1, 1, 1, [1]), (4, 3, 2, [4]), (5, 7, 9, [2, 3]), (10, 33, 65, [0, 10, 0]), (12, 64, 64, [5, 0, 4, 3]), (20, 100, 70, [1] * 20),
           (64, 128, 130, [3, 0, 0, 20, 1, 33, 0, 7]), (200, 65, 129, [64, 65, 63, 8]), (300, 257, 131, [129, 0, 171]),
           (130, 1027, 66, [2] * 65), (90, 40, 40, [1, 0] * 40 + [50, 0]), (700, 96, 256, [600, 100]), (33, 2050, 300, [32, 1])]


def _spans(sizes):
    at = 0
    for g, n in enumerate(sizes):
        yield g, slice(at, at + n)
        at += n


@pytest.mark.parametrize("rows,inner,outer,sizes", GROUPED)
@pytest.mark.parametrize("behind", [0, 5])
def test_groupedmm_forward_and_backward(cl, rows, inner, outer, sizes, behind):
    g = _rng("grouped", rows, inner, outer, behind)
    G, total = len(sizes), rows + behind
    x, w, gy = _normal(g, total, inner), _normal(g, G, inner, outer, scale=inner ** -0.5), _normal(g, total, outer)
    X, W, GY = cl.ClTensor(x), cl.ClTensor(w), cl.ClTensor(gy)
    S = cl.ClTensor(np.array(sizes, dtype=F))
    y, gx, gw = cl.ClTensor(total, outer).fill(-3.0), cl.ClTensor(total, inner).fill(-4.0), cl.ClTensor()
    assert y.groupedmm(X, W, S) is y
    cl.groupedmmBackward(gx, gw, GY, X, W, S)
    Y, GX, GW = y.float(), gx.float(), gw.float()
    assert GW.shape == w.shape
    for k, rows_k in _spans(sizes):
        a, b, c = x[rows_k].astype(np.float64), w[k].astype(np.float64), gy[rows_k].astype(np.float64)
        _within(Y[rows_k], a @ b, (inner + 3) * U * (np.abs(a) @ np.abs(b)), ("y", k))
        _within(GX[rows_k], c @ b.T, (outer + 3) * U * (np.abs(c) @ np.abs(b).T), ("gx", k))
        _within(GW[k], a.T @ c, (len(a) + 3) * U * (np.abs(a).T @ np.abs(c)), ("gw", k))
        if len(a) == 0:
            assert (GW[k] == 0).all()
    assert (Y[rows:] == -3).all() and (GX[rows:] == -4).all()
    want = np.concatenate([x[r].astype(np.float64) @ w[k] for k, r in _spans(sizes)])
    _norm_within(Y[:rows], want, inner, "y")
    # the same from a list, and each gradient by itself
    again = cl.ClTensor(total, outer).fill(-3.0).groupedmm(X, W, sizes).float()
    assert np.array_equal(again.view(np.uint32), Y.view(np.uint32))
    gx2, gw2 = cl.ClTensor(total, inner).fill(-4.0), cl.ClTensor()
    cl.groupedmmBackward(gx2, None, GY, X, W, sizes)
    cl.groupedmmBackward(None, gw2, GY, X, W, sizes)
    assert np.array_equal(gx2.float(), GX) and np.array_equal(gw2.float(), GW)


@pytest.mark.parametrize("inner,outer", [(30, 70), (129, 260)])
def test_groupedmm_views(cl, inner, outer):
    g = _rng("grouped views", inner, outer)
    sizes, G, T = [30, 0, 41, 9], 4, 85
    x, w, gy = _normal(g, T, inner), _normal(g, G, inner, outer), _normal(g, T, outer)
    want = np.concatenate([x[r].astype(np.float64) @ w[k] for k, r in _spans(sizes)])
    tol = np.concatenate([(inner + 3) * U * (np.abs(x[r]).astype(np.float64) @ np.abs(w[k])) for k, r in _spans(sizes)])
    xv, _ = _padded(cl, x)
    gv, _ = _padded(cl, gy)
    S = cl.ClTensor(np.repeat(np.array(sizes, dtype=F), 2)).strided([G], [2], 1)
    for name, W in {"transposed": cl.ClTensor(np.ascontiguousarray(w.transpose(0, 2, 1))).transpose(2, 3),
                    "groups inside": cl.ClTensor(np.ascontiguousarray(w.transpose(1, 0, 2))).transpose(1, 2),
                    "groups last": cl.ClTensor(np.ascontiguousarray(w.transpose(1, 2, 0))).permute(3, 1, 2)}.items():
        yv, ybuf = _padded(cl, np.zeros((T, outer), dtype=F))
        yv.groupedmm(xv, W, S)
        _within(yv.float()[:80], want, tol, name)
        assert (yv.float()[80:] == 0).all()
        out = ybuf.float()
        assert (out[:, :3] == -77).all() and (out[:, outer + 3:] == -77).all()
        yt = cl.ClTensor(outer, T).fill(6.0).t()
        yt.groupedmm(xv, W, S)
        assert np.array_equal(yt.float()[:80], yv.float()[:80]) and (yt.float()[80:] == 6).all()
        gw = cl.ClTensor(np.zeros((inner, G, outer), dtype=F)).transpose(1, 2)
        gx = cl.ClTensor()
        cl.groupedmmBackward(gx, gw, gv, xv, W, S)
        for k, r in _spans(sizes):
            a, c = x[r].astype(np.float64), gy[r].astype(np.float64)
            _within(gw.float()[k], a.T @ c, (len(a) + 3) * U * (np.abs(a).T @ np.abs(c)), (name, "gw"))
            _within(gx.float()[r], c @ w[k].T.astype(np.float64), (outer + 3) * U * (np.abs(c) @ np.abs(w[k]).T), (name, "gx"))
        gwt = cl.ClTensor(np.zeros((G, outer, inner), dtype=F)).transpose(2, 3)
        cl.groupedmmBackward(None, gwt, gv, xv, W, S)
        assert np.array_equal(gwt.float(), gw.float())
    # one matrix for every group
    shared = cl.ClTensor(w[:1]).expand(G, inner, outer)
    y = cl.ClTensor().groupedmm(xv, shared, S).float()[:80]
    plain = x[:80].astype(np.float64) @ w[0]
    _within(y, plain, (inner + 3) * U * (np.abs(x[:80]).astype(np.float64) @ np.abs(w[0])), "shared")


def test_groupedmm_keeps_what_is_not_finite_in_its_group_and_row(cl):
    g = _rng("grouped nan")
    sizes, inner, outer = [37, 3, 60], 90, 140
    x, w = _normal(g, 105, inner), _normal(g, 3, inner, outer)
    clean = cl.ClTensor(105, outer).fill(0.0).groupedmm(cl.ClTensor(x), cl.ClTensor(w), sizes).float()
    x[36], x[100:], w[1] = np.nan, np.inf, np.inf
    got = cl.ClTensor(105, outer).fill(0.0).groupedmm(cl.ClTensor(x), cl.ClTensor(w), sizes).float()
    assert np.isnan(got[36]).all() and not np.isfinite(got[37:40]).any() and (got[100:] == 0).all()
    keep = [i for i in range(100) if i not in (36, 37, 38, 39)]
    assert np.array_equal(got[keep], clean[keep])
    gw = cl.ClTensor()
    gy = _normal(g, 105, outer)
    cl.groupedmmBackward(None, gw, cl.ClTensor(gy), cl.ClTensor(x), cl.ClTensor(w), sizes)
    GW = gw.float()
    assert np.isnan(GW[0]).all()
    for k, r in ((1, slice(37, 40)), (2, slice(40, 100))):
        a, c = x[r].astype(np.float64), gy[r].astype(np.float64)
        _within(GW[k], a.T @ c, (len(a) + 3) * U * (np.abs(a).T @ np.abs(c)), ("gw", k))


@pytest.mark.parametrize("sizes", [[3, -1, 2], [5, 6, 0], [1.5, 2, 1], [np.nan, 1, 1], [np.inf, 0, 0], [11, 0, 0], [1e30, 1e30, 1e30]])
def test_groupedmm_sizes_that_do_not_fit_write_nothing_and_are_reported(cl, sizes):
    X, W = cl.ClTensor(np.ones((10, 4), dtype=F)), cl.ClTensor(np.ones((3, 4, 5), dtype=F))
    y, gx, gw = cl.ClTensor(10, 5).fill(2.0), cl.ClTensor(10, 4).fill(2.0), cl.ClTensor(3, 4, 5).fill(2.0)
    S = cl.ClTensor(np.array(sizes, dtype=F))
    y.groupedmm(X, W, S)
    with pytest.raises(cl.ClError, match="group sizes"):
        cl.synchronize()
    assert (y.float() == 2).all()
    cl.groupedmmBackward(gx, None, y, X, W, S)
    with pytest.raises(cl.ClError, match="group sizes"):
        cl.synchronize()
    cl.groupedmmBackward(None, gw, y, X, W, S)
    with pytest.raises(cl.ClError, match="group sizes"):
        cl.synchronize()
    assert (gx.float() == 2).all() and (gw.float() == 2).all()
    cl.synchronize()                       # reported once
    assert (y.groupedmm(X, W, [3, 3, 4]).float() == 4).all()


# ------------------------------------------------------- the operators together ---
def test_feed_forward_block_forward_and_backward(cl):
    """x + W2 act(W1 norm(x)) and its gradients, as one pre-norm block of a network runs them."""
    g = _rng("block")
    T, D, H = 70, 96, 200
    x, gy = _normal(g, 2, T // 2, D), _normal(g, 2, T // 2, D)
    nw, nb = _normal(g, D, scale=0.2, mean=1.0), _normal(g, D, scale=0.1)
    w1, b1 = _normal(g, H, D, scale=D ** -0.5), _normal(g, H, scale=0.1)
    w2, b2 = _normal(g, D, H, scale=H ** -0.5), _normal(g, D, scale=0.1)
    X, GY, NW, NB, W1, B1, W2, B2 = (cl.ClTensor(a) for a in (x, gy, nw, nb, w1, b1, w2, b2))
    h, mean, rstd, z, a, y = (cl.ClTensor() for _ in range(6))
    h.layerNorm(X, NW, NB, EPS, mean=mean, rstd=rstd)
    a.linear(h, W1, B1, activation="gelu", preact=z)
    y.linear(a, W2, B2, residual=X)
    ga, gw2, gb2, gh, gw1, gb1, gx, gnw, gnb = (cl.ClTensor() for _ in range(9))
    cl.linearBackward(ga, gw2, gb2, GY, a, W2)
    cl.linearBackward(gh, gw1, gb1, ga, h, W1, preact=z, activation="gelu")
    cl.layerNormBackward(gx, gnw, gnb, gh, X, NW, mean, rstd)
    gx.add(GY)
    import torch
    t = {k: torch.tensor(v, dtype=torch.float64, requires_grad=True) for k, v in
         dict(x=x, nw=nw, nb=nb, w1=w1, b1=b1, w2=w2, b2=b2).items()}
    away = t["x"] - t["x"].mean(-1, keepdim=True)
    hh = away / torch.sqrt((away ** 2).mean(-1, keepdim=True) + EPS) * t["nw"] + t["nb"]
    zz = hh @ t["w1"].t() + t["b1"]
    yy = (0.5 * zz * torch.erfc(-zz / math.sqrt(2))) @ t["w2"].t() + t["b2"] + t["x"]
    yy.backward(torch.tensor(gy, dtype=torch.float64))
    # three chained stages, each off by its own sums' sqrt(K) u and by the input's error, in the norm
    tol = 6 * math.sqrt(H) * U
    for name, got, want in (("y", y, yy), ("gx", gx, t["x"].grad), ("gnw", gnw, t["nw"].grad), ("gnb", gnb, t["nb"].grad),
                            ("gw1", gw1, t["w1"].grad), ("gb1", gb1, t["b1"].grad), ("gw2", gw2, t["w2"].grad), ("gb2", gb2, t["b2"].grad)):
        want = want.detach().numpy()
        assert got.size() == want.shape
        rel = np.linalg.norm(got.float() - want) / np.linalg.norm(want)
        assert rel <= tol, (name, rel)


def test_expert_block_with_routing_by_index(cl):
    """Tokens sorted by expert with index, through two grouped products with a gate between, and back by indexCopy."""
    g = _rng("experts")
    T, D, H, G = 50, 64, 90, 6
    x, w1, w2 = _normal(g, T, D), _normal(g, G, D, 2 * H, scale=D ** -0.5), _normal(g, G, H, D, scale=H ** -0.5)
    expert = g.randint(0, G - 1, T)                      # the last expert gets nothing
    order = np.argsort(expert, kind="stable")
    sizes = cl.ClTensor(np.bincount(expert, minlength=G).astype(F))
    xs = cl.ClTensor(x).index(1, list(order + 1))
    h = cl.ClTensor().groupedmm(xs, cl.ClTensor(w1), sizes)
    gate, up = h.narrow(2, 1, H), h.narrow(2, H + 1, H)
    a = up.clone().map_on_gpu(gate, "x = x * y / (1.0 + exp(-y))")
    ys = cl.ClTensor().groupedmm(a, cl.ClTensor(w2), sizes)
    y = cl.ClTensor(T, D).fill(0.0).indexCopy(1, list(order + 1), ys).float()
    want = np.empty((T, D))
    for t in range(T):
        u = x[t].astype(np.float64) @ w1[expert[t]]
        want[t] = (u[H:] * u[:H] / (1 + np.exp(-u[:H]))) @ w2[expert[t]]
    assert np.linalg.norm(y - want) / np.linalg.norm(want) <= 4 * math.sqrt(H) * U


# -------------------------------------------------------------------- refusals ---
def test_refusals(cl):
    t = lambda *s: cl.ClTensor(*s).fill(1.0)  # noqa: E731
    x, w, b = t(6, 8), t(5, 8), t(5)
    E = cl.ClError
    for call in (lambda: t(6, 5).linear(x, t(5, 7)), lambda: t(6, 5).linear(x, t(8)), lambda: t(6, 5).linear(x, w, t(6)),
                 lambda: t(6, 5).linear(x, w, b, residual=t(5, 6)), lambda: t(6, 5).linear(x, w, b, activation="tanh"),
                 lambda: x.linear(x, t(8, 8)), lambda: b.linear(t(8), w, b), lambda: t(6, 5).linear(cl.ClTensor(), w),
                 lambda: cl.linearBackward(t(6, 8), None, None, t(6, 5), x, w, activation="gelu"),
                 lambda: cl.linearBackward(t(6, 8), None, None, t(6, 4), x, w),
                 lambda: cl.linearBackward(x, None, None, t(6, 5), x, w), lambda: cl.linearBackward(None, w, None, t(6, 5), x, w),
                 lambda: t(6, 8).layerNorm(x, t(7)), lambda: t(6, 8).layerNorm(x, None, t(9)), lambda: t(6, 8).layerNorm(x, eps=-1.0),
                 lambda: t(6, 8).layerNorm(cl.ClTensor()), lambda: cl.layerNormBackward(t(6, 8), None, None, t(6, 7), x, None, t(6), t(6)),
                 lambda: cl.layerNormBackward(t(6, 8), None, None, t(6, 8), x, None, t(5), t(6)),
                 lambda: cl.layerNormBackward(t(6, 8), None, None, t(6, 8), x, None, t(6), cl.ClTensor()),
                 lambda: t(6, 5).groupedmm(x, w, [6]), lambda: t(6, 5).groupedmm(x, t(2, 7, 5), [3, 3]),
                 lambda: t(6, 5).groupedmm(x, t(2, 8, 5), [6]), lambda: t(6, 5).groupedmm(t(8), t(2, 8, 5), [3, 3]),
                 lambda: x.groupedmm(x, t(2, 8, 8), [3, 3]),
                 lambda: cl.groupedmmBackward(t(6, 8), None, t(5, 5), x, t(2, 8, 5), [3, 3])):
        with pytest.raises(E):
            call()
    # results inside an operand's memory, at other places than its own
    whole = t(12, 8)
    for call in (lambda: whole.narrow(1, 2, 6).layerNorm(whole.narrow(1, 1, 6)), lambda: whole.narrow(1, 2, 6).linear(whole.narrow(1, 1, 6), t(8, 8)),
                 lambda: whole.narrow(1, 2, 6).linear(x, t(8, 8), residual=whole.narrow(1, 1, 6)),
                 lambda: whole.narrow(1, 2, 6).linear(x, t(8, 8), preact=whole.narrow(1, 1, 6))):
        with pytest.raises(E, match="share memory"):
            call()
    assert (whole.float() == 1).all()
    # column ranges of one buffer are apart
    wide = t(6, 13)
    got = wide.narrow(2, 9, 5).linear(wide.narrow(2, 1, 8), w, b)
    assert (got.float() == 9).all() and (wide.narrow(2, 1, 8).float() == 1).all()
