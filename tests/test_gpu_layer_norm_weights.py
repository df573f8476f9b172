"""Layer norm with weight and bias that are views at odd offsets, of widths that are read four values at a time: the same
bits as with weight and bias of their own."""
import zlib

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
F = np.float32


@pytest.mark.parametrize("rows", [3, 600, 1100])
@pytest.mark.parametrize("width", [4, 60, 128, 256, 512, 1024, 2048, 4096, 8192, 8196, 16384])
def test_weight_and_bias_at_odd_offsets(cl, rows, width):
    g = np.random.RandomState(zlib.crc32(repr((rows, width)).encode()) & 0x7FFFFFFF)
    x, gy = g.standard_normal((rows, width)).astype(F), g.standard_normal((rows, width)).astype(F)
    w, b = g.standard_normal(width).astype(F), g.standard_normal(width).astype(F)
    X, GY = cl.ClTensor(x), cl.ClTensor(gy)
    results = []
    for offset in (0, 1, 2, 3):
        both = cl.ClTensor(2 * width + 8).fill(9.0)
        W, B = both.narrow(1, offset + 1, width), both.narrow(1, width + 2 * offset + 1, width)
        W.copy(cl.ClTensor(w))
        B.copy(cl.ClTensor(b))
        y, mean, rstd, gx, gw, gb = (cl.ClTensor() for _ in range(6))
        y.layerNorm(X, W, B, 1e-5, mean=mean, rstd=rstd)
        cl.layerNormBackward(gx, gw, gb, GY, X, W, mean, rstd)
        results.append([t.float() for t in (y, gx, gw, gb)])
    x64 = x.astype(np.float64)
    h = (x64 - x64.mean(1, keepdims=True)) / np.sqrt(x64.var(1, keepdims=True) + 1e-5)
    # x - mean rounds twice, rstd three times, the product and the sum once
    assert (np.abs(results[0][0] - (h * w + b)) <= 2.0 ** -24 * (7 * np.abs(h * w) + 2 * np.abs(h * w + b)) + 2.0 ** -24).all()
    for other in results[1:]:
        for a, c in zip(results[0], other):
            assert np.array_equal(a, c)
