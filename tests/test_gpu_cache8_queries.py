"""8-bit decode of queries whose elements lie far apart, and how near f32 results are to 64 bits."""
import numpy as np
import pytest

from cache8_oracle import attention, attention_bound, held
from oracle import oracle as O

pytestmark = pytest.mark.gpu

# A weight's relative error is that of five roundings of its score (the sum of digits times codes in two, the factor, the product, the
# difference to the reference; |s| is about 2, in log2 units), of the exponential (2^-22.5) and of two f16 terms (2^-23), each
# independent: rms 0.7 * 2 * sqrt(5) * 2^-24 / sqrt(3) = 1.1e-7, 1e-7 and 0.7e-7, together 1.7e-7.  The result's error, relative to the
# result, is the same (its terms and their errors add up alike), and the sums' roundings over the pages come on top, another 2e-7.  Three times
# that is allowed.
NORM = 1e-6


def _fb():
    import floneum_b200 as fb
    return fb


def _T(device, a, dtype=0):
    return _fb().Tensor.from_slice(device, a.shape, a, dtype)


def _off(device, q, k, v, scale, ctas):
    fb = _fb()
    B, Hkv, n, D = k.shape
    cache = fb.PagedKvCache(device, B, Hkv, D, B * ((n + 15) // 16), (n + 15) // 16, dtype=fb.I8)
    cache.append(_T(device, k), _T(device, v))
    wk, wv = held(k), held(v)
    want = np.stack([attention(q[b, :, 0], wk[b], wv[b], scale)[0] for b in range(B)])
    offs = []
    for c in ctas:
        cache.set_decode_ctas(c)
        got = cache.decode(_T(device, q), scale).as_slice()[:, :, 0]
        assert np.isfinite(got).all()
        offs.append(np.linalg.norm(got - want) / np.linalg.norm(want))
    return offs


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("r", [1, 30, 100, 1000, 30000, 1e6, 2.0 ** 22])
def test_one_dimension_far_above_the_others(device, D, r):
    """q has an element r times as large as the others where the keys are zero: the scores are those of the others, in f32 as in 64 bits."""
    rng = np.random.default_rng(D)
    q = rng.standard_normal((2, 8, 1, D)).astype(np.float32)
    k, v = (rng.standard_normal((2, 2, 1411, D)).astype(np.float32) for _ in range(2))
    q[..., 5], k[..., 5] = r, 0.0
    q[:, 3, 0, 9] = -r  # a head with two of them
    k[..., 9] = 0.0
    for off in _off(device, q, k, v, float(D ** -0.5), (0, 1, 148)):
        assert off <= NORM


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("g,Hkv,n", [(1, 3, 700), (5, 2, 333), (8, 1, 5000), (3, 4, 17)])
def test_f32_queries_of_any_spread(device, D, g, Hkv, n):
    """Elements spread over 2^-20 .. 1, and keys that are zero where the query's are large: the small ones make the scores."""
    rng = np.random.default_rng(D * g + n)
    up = rng.integers(0, 21, D)
    q = (rng.standard_normal((2, g * Hkv, 1, D)) * np.exp2(-up)).astype(np.float32)
    k = (rng.standard_normal((2, Hkv, n, D)) * np.exp2(rng.integers(-3, 3, (2, Hkv, n, 1)) / 2)).astype(np.float32)
    small = up > np.median(up)
    k[..., ~small] = 0.0
    v = rng.standard_normal((2, Hkv, n, D)).astype(np.float32)
    q /= np.abs(q[..., small]).max(-1, keepdims=True) * np.float32(0.5)  # scores of a few units
    for off in _off(device, q, k, v, float(D ** -0.5), (0, 7)):
        assert off <= NORM


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", [17, 1411, 9000])
def test_f32_results_of_ordinary_queries(device, D, lens):
    """Nearer to 64 bits than a looser test could tell from a query cut to 16 bits (1.4e-5)."""
    rng = np.random.default_rng(lens + D)
    q = rng.standard_normal((1, 8, 1, D)).astype(np.float32)
    k, v = (rng.standard_normal((1, 2, lens, D)).astype(np.float32) for _ in range(2))
    for off in _off(device, q, k, v, float(D ** -0.5), (0, 1, 40)):
        assert off <= NORM


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [1, 2])
@pytest.mark.parametrize("r", [1, 100, 8000, 60000])
def test_16_bit_queries_of_any_spread(device, D, dtype, r):
    """Elements from 2^-14 (f16: 2^-11) of the largest on are exact, the others off by up to 2^-23 of it: what that makes of a score, and twice
    that of a result, on top of the bound of exact queries."""
    fb = _fb()
    rng = np.random.default_rng(D + dtype)
    q = rng.standard_normal((1, 4, 1, D)).astype(np.float32)
    k, v = (rng.standard_normal((1, 1, 700, D)).astype(np.float32) for _ in range(2))
    q[..., 5], k[..., 5] = r, 0.0
    q = O.bf16_round(q) if dtype == 1 else q.astype(np.float16).astype(np.float32)
    wk, wv, scale = held(k)[0], held(v)[0], float(D ** -0.5)
    want = attention(q[0, :, 0], wk, wv, scale)[0]
    a = np.abs(q[0, :, 0].astype(np.float64))
    off = np.where(a >= a.max(-1, keepdims=True) * 2.0 ** (-14 if dtype == 1 else -11), 0.0, 2.0 ** -23 * a.max(-1, keepdims=True))  # [heads, D]
    score = (off @ np.abs(wk[0].astype(np.float64)).T).max(-1) * scale
    bound = attention_bound(q[0, :, 0], wk, wv, scale) + 2.1 * score[:, None] * np.abs(wv).max()
    cache = fb.PagedKvCache(device, 1, 1, D, 44, 44, dtype=fb.I8)
    cache.append(_T(device, k), _T(device, v))
    for ctas in (0, 9):
        cache.set_decode_ctas(ctas)
        got = cache.decode(_T(device, q, dtype), scale).as_slice()[0, :, 0]
        assert (np.abs(got - want) <= bound).all(), (ctas, (np.abs(got - want) / bound).max())
