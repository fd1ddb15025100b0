"""8-bit decode: what the merges of partial records make of rows that are not finite."""
import numpy as np
import pytest

from cache8_oracle import attention, attention_bound, held

pytestmark = pytest.mark.gpu


def _fb():
    import floneum_b200 as fb
    return fb


def _T(device, a, dtype=0):
    return _fb().Tensor.from_slice(device, a.shape, a, dtype)


def _far(rng, D, n, far_at, where, bad):
    """q of four heads on one kv head; key `far_at` scores 150 (natural log) for heads 0 and 2, the others about 1: next to it every other
    weight is below the smallest float.  Row `bad` of K or V is not finite."""
    q = rng.standard_normal((1, 4, 1, D)).astype(np.float32)
    k, v = (rng.standard_normal((1, 1, n, D)).astype(np.float32) for _ in range(2))
    q[0, 2] = q[0, 0]
    k[0, 0, far_at] = q[0, 0, 0] * np.float32(150 * D ** 0.5 / np.square(q[0, 0, 0]).sum())
    if where:
        (k if where == "k" else v)[0, 0, bad, 7] = np.nan
    return q, k, v


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ctas", [0, 1, 2, 9, 148])
@pytest.mark.parametrize("where,bad,far_at", [("k", 100, 3900), ("v", 100, 3900), ("k", 3900, 100), ("v", 3990, 5), ("k", 2000, 2017), ("v", 2000, 2001)])
def test_a_row_that_is_not_finite_reaches_the_result_from_any_share(device, D, ctas, where, bad, far_at):
    """Its weight next to the largest score is zero in f32, and 0 * NaN is NaN: on every path, however the pages are shared out."""
    fb = _fb()
    rng = np.random.default_rng(D + bad)
    q, k, v = _far(rng, D, 4000, far_at, where, bad)
    cache = fb.PagedKvCache(device, 1, 1, D, 250, 250, dtype=fb.I8)
    cache.append(_T(device, k), _T(device, v))
    cache.set_decode_ctas(ctas)
    tq, scale = _T(device, q), float(D ** -0.5)
    assert np.isnan(cache.decode(tq, scale).as_slice()).all()
    part = cache.decode_partial(tq, scale).as_slice()
    assert np.isnan(part[..., 2:]).all()
    cache.drop_front(0, 4000 - max(bad, far_at) - 1)  # both rows gone
    lo = max(bad, far_at) + 1
    got, want = cache.decode(tq, scale).as_slice()[0, :, 0], attention(q[0, :, 0], held(k)[0, :, lo:], held(v)[0, :, lo:], scale)[0]
    assert np.abs(got - want).max() <= attention_bound(q[0, :, 0], held(k)[0, :, lo:], held(v)[0, :, lo:], scale)


@pytest.mark.parametrize("D", [64, 128])
def test_a_finite_cache_with_a_far_key(device, D):
    """The same rows without the NaN: the far key's value for the heads it belongs to."""
    fb = _fb()
    rng = np.random.default_rng(D)
    q, k, v = _far(rng, D, 4000, 3900, "", 0)
    cache = fb.PagedKvCache(device, 1, 1, D, 250, 250, dtype=fb.I8)
    cache.append(_T(device, k), _T(device, v))
    scale = float(D ** -0.5)
    want = attention(q[0, :, 0], held(k)[0], held(v)[0], scale)[0]
    for ctas in (0, 1, 2, 9, 148):
        cache.set_decode_ctas(ctas)
        got = cache.decode(_T(device, q), scale).as_slice()[0, :, 0]
        assert np.abs(got - want).max() <= attention_bound(q[0, :, 0], held(k)[0], held(v)[0], scale), ctas
