"""Axes that the positions do not have are refused before anything is launched, and do not wrap."""
import ctypes

import numpy as np
import pytest


def _fb():
    import floneum_b200 as fb
    return fb


def _bytes(p, n):
    """What the C call reads (the field itself ends at its first zero)."""
    return ctypes.string_at(ctypes.c_void_p.from_buffer(p, type(p).axis_of_pair.offset).value, n)


def _ids(*shape):
    return _fb().Tensor(None, 4096, shape, _fb().U32)


@pytest.mark.parametrize("bad", [[0, 0, 0, 256], [0, 0, 0, -1], [0, 0, 0, 2], [0, 0, 0, 1.5], [0, 0, 0, 257], [0, 0, 0, np.nan], [0, 0, 0, 2 ** 40], [0, 0, 0, -256]])
@pytest.mark.parametrize("make", [list, np.array, lambda x: np.array(x, np.float64), lambda x: np.array(x, np.float32)])
def test_an_axis_that_the_positions_do_not_have(bad, make):
    from floneum_b200.rope import _positions
    with pytest.raises(AssertionError, match="ax"):
        _positions(_ids(2, 3), make(bad), 1, 3, 8)


@pytest.mark.parametrize("dtype", [np.uint8, np.int8, np.int32, np.int64, np.uint64, np.float32, bool])
def test_axes_of_any_type_of_whole_numbers(dtype):
    from floneum_b200.rope import _positions
    p = _positions(_ids(2, 3), np.array([0, 1, 1, 0], dtype), 1, 3, 8)
    assert _bytes(p, 4) == bytes([0, 1, 1, 0])
    p = _positions(_ids(2, 3), (0, 1, 1, 0), 1, 3, 8)
    assert _bytes(p, 4) == bytes([0, 1, 1, 0])
    p = _positions(_ids(2, 3), np.array([0, 9, 1, 9, 1, 9, 0, 9], dtype)[::2], 1, 3, 8)
    assert _bytes(p, 4) == bytes([0, 1, 1, 0])
