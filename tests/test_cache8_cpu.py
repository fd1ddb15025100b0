"""The 8-bit cache and rotary positions with several axes without a GPU: argument checks of the host mirrors and of the C ABI."""
import ctypes

import numpy as np
import pytest


def _fb():
    import floneum_b200 as fb
    return fb


def test_axes_of_sections():
    fb = _fb()
    assert fb.axes_of_sections([2, 3, 1]).tolist() == [0, 0, 1, 1, 1, 2]
    assert fb.axes_of_sections([4]).tolist() == [0] * 4
    assert fb.axes_of_sections([0, 2]).tolist() == [1, 1]
    assert fb.axes_of_sections([3, 2, 2], alternating=True).tolist() == [0, 1, 2, 0, 1, 2, 0]
    assert fb.axes_of_sections([4, 1, 1], alternating=True).tolist() == [0, 1, 2, 0, 0, 0]
    for bad in ([], [-1, 3], [1] * 257):
        with pytest.raises(AssertionError):
            fb.axes_of_sections(bad)
    with pytest.raises(AssertionError):
        fb.axes_of_sections([1, 3], alternating=True)  # axis 0 would have to give up its pairs


def test_positions_are_checked_before_the_call():
    fb = _fb()
    from floneum_b200.rope import _positions
    ids = lambda *shape, **kw: fb.Tensor(None, 4096, shape, kw.pop("dtype", fb.U32), **kw)
    axes = fb.axes_of_sections([2, 2])
    p = _positions(ids(2, 3, 5), axes, 3, 5, 8)
    assert (p.ids, p.axis_stride, p.batch_stride, p.n_axes) == (4096, 15, 5, 2)
    p = _positions(ids(2, 5), axes, 3, 5, 8)
    assert (p.axis_stride, p.batch_stride) == (5, 0)
    p = _positions(ids(2, 3, 5, strides=(40, 8, 1)), axes, 3, 5, 8)
    assert (p.axis_stride, p.batch_stride) == (40, 8)
    for bad in (ids(2, 3, 5, dtype=fb.F32), ids(2, 3, 4), ids(2, 2, 5), ids(5), ids(2, 3, 5, strides=(30, 10, 2))):
        with pytest.raises(AssertionError):
            _positions(bad, axes, 3, 5, 8)
    with pytest.raises(AssertionError):
        _positions(ids(2, 3, 5), axes, 3, 5, 16)  # the axis of each of 8 pairs


def test_a_cache_has_bf16_or_8_bit_pages():
    fb = _fb()
    assert fb.KvCache.new(2, 64).dtype == fb.BF16 and fb.KvCache.new(2, 64, fb.I8).dtype == fb.I8
    assert [b.dtype for b in fb.LlamaCache(2, 64, dtype=fb.I8).blocks] == [fb.I8] * 2
    for dtype in (fb.F32, fb.F16, fb.U32, 7):
        with pytest.raises(fb.FusorCudaError):
            fb.KvCache.new(2, 64, dtype)


def test_the_c_view_of_a_tensor():
    fb = _fb()
    from floneum_b200 import _lib
    assert ctypes.sizeof(_lib.Tensor4) == 80
    for t in (fb.Tensor(None, 2 ** 47 + 16, (2, 3, 5, 64), fb.BF16), fb.Tensor(None, 4096, (1, 2, 3, 4), fb.F32, (2 ** 40, 7, 0, 1))):
        c = t._c4()
        assert (c.data, c.dtype, tuple(c.shape), tuple(c.stride)) == (t.ptr, t.dtype, t.shape(), tuple(t.strides))
    assert fb.Tensor(None, 0, (2, 3, 5, 64)).strides == (960, 320, 64, 1) and fb.Tensor(None, 0, (4, 3, 2)).strides == (6, 2, 1)


def test_null_arguments_are_status_codes():
    from floneum_b200 import _lib
    L = _lib.load()
    null = ctypes.c_void_p()
    pos = _lib.RopePositions()
    assert L.fusor_cuda_kvcache_create_dtype(None, 1, 1, 64, 16, 1, 1, _lib.I8, ctypes.byref(null)) == _lib.INVALID_ARGUMENT
    assert L.fusor_cuda_kvcache_scales(None, ctypes.byref(null)) == _lib.INVALID_ARGUMENT
    assert L.fusor_cuda_kvcache_write_scales(None, 0, 0, None) == _lib.INVALID_ARGUMENT
    assert L.fusor_cuda_kvcache_read_scales(None, 0, 0, None) == _lib.INVALID_ARGUMENT
    assert L.fusor_cuda_rope_axes(None, None, None, None, 1, ctypes.byref(pos), 0, None) == _lib.INVALID_ARGUMENT
    assert L.fusor_cuda_kvcache_rope_axes_append(None, None, None, None, None, None, 1, ctypes.byref(pos), 0, None) == _lib.INVALID_ARGUMENT


def test_plain_rows_have_the_properties_the_format_promises():
    """The oracle of the GPU tests: codes within +-127, the smallest step that allows it, values exact in bf16, and the same
    codes for a row that is written again."""
    from cache8_oracle import quantise, values
    rng = np.random.default_rng(8)
    rows = np.concatenate([rng.standard_normal((300, 64)) * 2.0 ** rng.integers(-120, 120, (300, 1)), np.zeros((1, 64)),
                           np.full((1, 64), 1e-44)]).astype(np.float32)
    codes, byte = quantise(rows)
    assert np.abs(codes.astype(int)).max() == 127 and byte.min() == 1 and byte.max() < 255
    big = byte > 1
    assert np.abs(codes[big].astype(int)).max(1).min() >= 64  # else the step could be halved
    v = values(codes, byte)
    assert np.array_equal(v.view(np.uint32) & 0xffff, np.zeros_like(v.view(np.uint32)))
    assert np.all(np.abs(v - rows) <= np.ldexp(0.5, byte.astype(int) - 127)[:, None])
    again = quantise(v)
    assert np.array_equal(again[0], codes) and np.array_equal(again[1][big], byte[big])
