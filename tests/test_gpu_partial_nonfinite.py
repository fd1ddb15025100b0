"""Partial records with a sum that is not finite, merged: NaN, not the zeros of a row without keys."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _fb():
    import floneum_b200 as fb
    return fb


def _T(device, a, dtype=0):
    return _fb().Tensor.from_slice(device, a.shape, a, dtype)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("m", [0.0, -200.0, 200.0])
def test_a_record_of_nan_makes_nan_of_its_row(device, D, m):
    from floneum_b200.cache import lse_combine
    rng = np.random.default_rng(D)
    parts = rng.standard_normal((3, 2, 4, D + 2)).astype(np.float32)  # {m, l, O}
    parts[..., 1] = np.abs(parts[..., 1]) + 0.5
    parts[1, 0, 2, 0], parts[1, 0, 2, 1:] = m, np.nan
    parts[:, 1, 3, 0], parts[:, 1, 3, 1:] = -np.inf, 0.0  # a row without keys
    got = lse_combine(device, _T(device, parts)).as_slice()
    p = parts.astype(np.float64)
    with np.errstate(invalid="ignore"):
        w = np.exp(p[..., 0] - p[..., 0].max(0))
        want = (w[..., None] * p[..., 2:]).sum(0) / (w * p[..., 1]).sum(0)[..., None]
    want[1, 3] = 0.0
    assert np.isnan(got[0, 2]).all()
    rest = np.ones((2, 4), bool)
    rest[0, 2] = False
    # each of three weighted terms: weight 2^-21 (exp of a difference of a few units), product and sum 2^-23
    size = (w[..., None] * np.abs(p[..., 2:])).sum(0) / (w * p[..., 1]).sum(0)[..., None]
    assert (np.abs(got - want)[rest] <= 2.0 ** -19 * size[rest] + 1e-30)[~np.isnan(size[rest])].all() and not got[1, 3].any()


@pytest.mark.parametrize("pages", ["i8", "bf16"])
@pytest.mark.parametrize("ctas", [1, 9, 148])
def test_a_key_of_nan_through_partial_records_and_the_exchange(device, pages, ctas):
    fb = _fb()
    from floneum_b200.cache import lse_combine
    from floneum_b200.sharding import PeerExchange
    rng = np.random.default_rng(ctas)
    D, n, scale = 128, 2500, 0.09
    k, v = (rng.standard_normal((2, 2, n, D)).astype(np.float32) for _ in range(2))
    k[0, 1, 70, 3] = np.nan
    q = _T(device, rng.standard_normal((2, 8, 1, D)).astype(np.float32))
    cache = fb.PagedKvCache(device, 2, 2, D, 2 * 157, 157, dtype=fb.I8 if pages == "i8" else fb.BF16)
    cache.append(_T(device, k), _T(device, v))
    cache.set_decode_ctas(ctas)
    bad = np.zeros((2, 8), bool)
    bad[0, 4:] = True
    whole = cache.decode(q, scale).as_slice()[:, :, 0]
    joined = lse_combine(device, _T(device, cache.decode_partial(q, scale).as_slice()[None])).as_slice()
    ex = PeerExchange(device, 0, 1, 2 * 8 * (D + 2))
    out = fb.Tensor.zeros(device, (2, 8, D))
    ex.decode(cache, q, scale, out)
    for got in (whole, joined.reshape(2, 8, D), out.as_slice()):
        assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
    ex.close()
