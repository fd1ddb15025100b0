"""Host data that u32 does not hold is refused before it is uploaded, and does not wrap."""
import numpy as np
import pytest


@pytest.mark.parametrize("bad", [[-1], [1.5], [np.nan], [2 ** 32], [np.inf], [-2 ** 31], [2 ** 63]])
@pytest.mark.parametrize("make", [list, np.array, lambda x: np.array(x, np.float64)])
def test_positions_that_32_bits_do_not_hold(bad, make):
    from floneum_b200.tensor import _whole_numbers
    with pytest.raises(AssertionError, match="u32"):
        _whole_numbers(make(bad))


def test_positions_that_they_hold():
    from floneum_b200.tensor import _whole_numbers
    for x in ([0, 1, 2 ** 32 - 1], np.array([0.0, 7.0, 2.0 ** 31]), np.zeros(3, np.float32), np.array([[5]], np.uint32), [], np.array([3], np.uint64),
              np.array([True, False])):
        got = _whole_numbers(x)
        assert got.dtype == np.uint32 and np.array_equal(got, np.asarray(x))
