"""Lists of group sizes on their way to the device, where they are fp32."""
import numpy as np
import pytest

import cltorch_amd.tensor as T


@pytest.fixture
def held(monkeypatch):
    """what a list is handed on as, without a device"""
    class Held:
        def __init__(self, values):
            self.values = values
    monkeypatch.setattr(T, "ClTensor", Held)
    return lambda sizes: T._sizes_of(sizes).values


@pytest.mark.parametrize("size", [2 ** 24 + 1, 2 ** 25 + 2, 2 ** 31 - 1, 1.7e38 * 3, 123456789])
def test_sizes_that_would_be_rounded_are_refused(held, size):
    for sizes in ([size], [3, size], (0, size, 1), np.array([size], dtype=np.float64)):
        with pytest.raises(T.ClError, match="group sizes"):
            held(sizes)


def test_sizes_that_fp32_holds_are_handed_on(held):
    for sizes in ([0, 5, 2 ** 24], [2 ** 24 + 2, 2 ** 30], (1, 2), np.array([[1, 2], [3, 4]])):
        got = held(sizes)
        assert got.dtype == np.float32 and np.array_equal(got, np.asarray(sizes).reshape(-1))
    # what the device reports: no whole numbers, negative, not a number
    got = held([1.5, 0.1, -1, np.nan, np.inf, -np.inf])
    assert np.array_equal(got, np.array([1.5, 0.1, -1, np.nan, np.inf, -np.inf], dtype=np.float32), equal_nan=True)
