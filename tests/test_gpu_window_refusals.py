"""An append that is refused leaves a full window, and its oldest rows, as they were."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _fb():
    import floneum_b200 as fb
    return fb


def _T(device, a, dtype=0):
    return _fb().Tensor.from_slice(device, a.shape, a, dtype)


def _full(device, dtype, B=2, window=20, D=64):
    fb = _fb()
    rng = np.random.default_rng(window)
    x = lambda n, h=2, b=B, d=D: _T(device, rng.standard_normal((b, h, n, d)).astype(np.float32))
    cache = fb.KvCache(2, window, dtype=dtype)
    cache.append(device, x(window), x(window))
    return fb, cache, x


def _rows(cache):
    k, v = cache.k().as_slice(), cache.v().as_slice()
    return k, v


def _as_before(cache, before, what):
    assert cache.k() is not None, what
    for a, b in zip(before, _rows(cache)):
        assert np.array_equal(a, b), what


DTYPES = pytest.mark.parametrize("pages", ["bf16", "i8"])


def _dtype(pages):
    return _fb().I8 if pages == "i8" else _fb().BF16


@DTYPES
@pytest.mark.parametrize("n", [3, 20, 27])
def test_rotated_appends(device, pages, n):
    fb, cache, x = _full(device, _dtype(pages))
    rope, axes = fb.RopeCache.new(64, 64, 10000.0, device), fb.axes_of_sections([16, 16])
    narrow = fb.RopeCache.new(32, 64, 10000.0, device)
    ids = _T(device, np.zeros((2, n), np.uint32), fb.U32)
    before = _rows(cache)
    third = axes.copy()
    third[31] = 2
    refused = (AssertionError, fb.FusorCudaError, KeyError)
    calls = {
        "an axis that the positions do not have": lambda: rope.forward_append(x(n, 4), x(n), x(n), cache, positions=ids, axes=third),
        "tables of another width": lambda: narrow.forward_append(x(n, 4), x(n), x(n), cache, positions=ids, axes=axes),
        "tables of another width, one axis": lambda: narrow.forward_append(x(n, 4), x(n), x(n), cache, start_pos=0),
        "rows past the tables": lambda: rope.forward_append(x(n, 4), x(n), x(n), cache, start_pos=64 - n + 1),
        "a type that is not one": lambda: rope.forward_append(x(n, 4), x(n), x(n), cache, start_pos=0, out_dtype=fb.U32),
        "a type that is not one, axes": lambda: rope.forward_append(x(n, 4), x(n), x(n), cache, positions=ids, axes=axes, out_dtype=9),
        "q and k of different lengths": lambda: rope.forward_append(x(n + 1, 4), x(n), x(n), cache, start_pos=0),
        "q of another batch": lambda: rope.forward_append(x(n, 4, 1), x(n), x(n), cache, start_pos=0),
    }
    if n < 20:
        calls["another batch"] = lambda: rope.forward_append(x(n, 4, 1), x(n, 2, 1), x(n, 2, 1), cache, start_pos=0)
    for what, call in calls.items():
        with pytest.raises(refused):
            call()
        _as_before(cache, before, what)
    q, k, _ = rope.forward_append(x(n, 4), x(n), x(n), cache, positions=ids, axes=axes)  # and it goes on
    assert q.shape()[2] == n and cache.current_seq_len() == 20
    assert np.array_equal(k.as_slice()[:, :, :20 - min(n, 20)], before[0][:, :, min(n, 20):])


def test_the_default_position_of_a_full_window_is_past_tables_of_its_length(device):
    fb, cache, x = _full(device, fb_i8())
    rope = fb.RopeCache.new(64, 20, 10000.0, device)  # context == window
    before = _rows(cache)
    for _ in range(3):
        with pytest.raises(fb.FusorCudaError):
            rope.forward_append(x(1, 4), x(1), x(1), cache)
        _as_before(cache, before, "one more token")


def fb_i8():
    return _fb().I8


@DTYPES
@pytest.mark.parametrize("n", [1, 20, 30])
def test_plain_appends(device, pages, n):
    import torch
    fb, cache, x = _full(device, _dtype(pages))
    before = _rows(cache)
    wide = torch.zeros((2, 2, n, 128), device="cuda")
    ints = torch.zeros((2, 2, n, 64), device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    apart = fb.Tensor.from_torch(device, wide[..., ::2])
    calls = {"elements apart": lambda: cache.append(device, apart, apart),
             "values apart": lambda: cache.append(device, x(n), apart),
             "whole numbers": lambda: cache.append(device, *(fb.Tensor.from_torch(device, ints),) * 2),
             "other heads, elements apart": lambda: cache.append(device, *(fb.Tensor.from_torch(device, wide[:, :1, :, ::2]),) * 2),
             "a head_dim without kernels": lambda: cache.append(device, x(n, 2, 2, 32), x(n, 2, 2, 32)),
             "a larger batch, elements apart": lambda: cache.append(device, *(fb.Tensor.from_torch(device, torch.zeros((3, 2, n, 128), device="cuda")[..., ::2]),) * 2)}
    if n < 20:
        calls["another batch"] = lambda: cache.append(device, x(n, 2, 1), x(n, 2, 1))
    for what, call in calls.items():
        with pytest.raises(fb.FusorCudaError):
            call()
        _as_before(cache, before, what)
    k, v = x(n), x(n)
    cache.append(device, k, v)
    assert cache.current_seq_len() == 20


@DTYPES
@pytest.mark.parametrize("window,D", [(1, 64), (16, 128), (21, 64), (37, 128)])
def test_a_window_of_a_paged_cache(device, pages, window, D):
    """Appends of every length up to the window, on a pool with one page a sequence to spare, against the newest rows; what does not fit or is
    refused changes nothing."""
    from cache8_oracle import held
    from oracle import oracle as O
    fb = _fb()
    rng = np.random.default_rng(window + D)
    keep = held if pages == "i8" else O.bf16_round
    B, Hkv, most = 2, 3, (window + 15) // 16 + 1
    cache = fb.PagedKvCache(device, B, Hkv, D, B * most, most, dtype=_dtype(pages))
    cache.set_window(window)
    want = np.zeros((B, Hkv, 0, D), np.float32)
    for n in [1, 1] + [int(x) for x in rng.integers(1, window + 1, 25)] + [window]:
        x = rng.standard_normal((B, Hkv, n, D)).astype(np.float32)
        with pytest.raises(fb.FusorCudaError):
            cache.append(_T(device, np.zeros((B, Hkv, window + 1, D), np.float32)), _T(device, np.zeros((B, Hkv, window + 1, D), np.float32)))
        cache.append(_T(device, x), _T(device, -x))
        want = np.concatenate([want, keep(x)], 2)[:, :, -window:]
        gk, gv = cache.gather(B, want.shape[2])
        assert np.array_equal(gk.as_slice(), want) and np.array_equal(gv.as_slice(), -want)
        assert cache.seq_len(0) == cache.seq_len(1) == want.shape[2]
    one = rng.standard_normal((1, Hkv, window, D)).astype(np.float32)  # the place of all that was there, in another batch
    cache.append(_T(device, one), _T(device, one))
    assert np.array_equal(cache.gather(1, window)[0].as_slice(), keep(one))
    cache.set_window(0)
    more = rng.standard_normal((1, Hkv, 1, D)).astype(np.float32)
    cache.append(_T(device, more), _T(device, more))
    assert np.array_equal(cache.gather(1, window + 1)[0].as_slice(), np.concatenate([keep(one), keep(more)], 2))
    with pytest.raises(fb.FusorCudaError):
        cache.set_window(-1)


@DTYPES
def test_own_positions_in_a_window(device, pages):
    """start_pos < 0: every sequence's length without the rows that give way, so tables as long as the window are enough."""
    from cache8_oracle import held
    from oracle import oracle as O
    fb = _fb()
    rng = np.random.default_rng(4)
    keep, D, window = held if pages == "i8" else O.bf16_round, 64, 21
    rope = fb.RopeCache.new(D, window, 10000.0, device)
    cos, sin = rope.cos.as_slice(), rope.sin.as_slice()
    cache = fb.PagedKvCache(device, 2, 2, D, 2 * 3, 3, dtype=_dtype(pages))
    cache.set_window(window)
    want, at = np.zeros((2, 2, 0, D), np.float32), 0
    for n in (5, 16, 1, 1, 7, 21, 3):
        q, k = (rng.standard_normal((2, h, n, D)).astype(np.float32) for h in (4, 2))
        at = min(at, window - n)
        got = rope.forward_append(_T(device, q), _T(device, k), _T(device, k), cache)
        assert np.array_equal(got.as_slice(), O.rope(q, cos, sin, at, False))
        want = np.concatenate([want, keep(O.rope(k, cos, sin, at, False))], 2)[:, :, -window:]
        at += n
        assert np.array_equal(cache.gather(2, at)[0].as_slice(), want)


@DTYPES
def test_a_window_when_the_pool_is_short(device, pages):
    """An append that finds no page is refused before the window drops a row; pages that the drop frees are counted."""
    fb = _fb()
    rng = np.random.default_rng(3)
    x = lambda n: _T(device, rng.standard_normal((2, 2, n, 64)).astype(np.float32))
    cache = fb.PagedKvCache(device, 2, 2, 64, 5, 4, dtype=_dtype(pages))
    cache.set_window(40)
    cache.append(x(32), x(32))  # four of five pages
    before = [t.as_slice() for t in cache.gather(2, 32)]
    with pytest.raises(fb.FusorCudaError) as e:
        cache.append(x(9), x(9))  # 40 rows a sequence: six pages
    assert e.value.code == fb._lib.OUT_OF_PAGES
    for a, b in zip(before, cache.gather(2, 32)):
        assert np.array_equal(a, b.as_slice())
    cache.set_window(32)
    k = x(16)
    cache.append(k, x(16))  # sixteen rows, a page, of each give way
    assert np.array_equal(cache.gather(2, 32)[0].as_slice()[:, :, :16], before[0][:, :, 16:])
