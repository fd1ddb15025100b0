"""8-bit decode: values whose rows have hardly any weight, alone in their dims."""
import numpy as np
import pytest

from cache8_oracle import attention, held, quantise

pytestmark = pytest.mark.gpu


def _fb():
    import floneum_b200 as fb
    return fb


def _T(device, a, dtype=0):
    return _fb().Tensor.from_slice(device, a.shape, a, dtype)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [40, 4000])
@pytest.mark.parametrize("lift", [0, 12, -12])
def test_many_light_rows_that_carry_dims_of_their_own(device, D, n, lift):
    """One row with nearly all the weight and zeros in half the dims; the others weigh 2^-20 to 2^-28 of it and have those dims to themselves.
    A weight is held in two f16 terms with a factor of 2^6: off by 2^-22 of itself or by 2^-31 of the largest weight, that of exp(s) times
    the row's step (the reference may lie below it, not above).  The exponential adds 2^-22, five roundings of a score of up to 30 in log2
    units 30 * 5 * 2^-24 ln 2 = 2^-17.3, and the same again in the sum the result is divided by; 2^-16 with the sums' own roundings."""
    fb = _fb()
    rng = np.random.default_rng(D + n)
    q = np.zeros((1, 2, 1, D), np.float32)
    q[..., 0] = 1.0
    k, v = np.zeros((1, 1, n, D), np.float32), rng.standard_normal((1, 1, n, D)).astype(np.float32)
    heavy = n // 3
    k[0, 0, :, 0] = -rng.integers(56, 78, n) * 0.25  # scores of -14 to -19.5, exact in 8 bits
    k[0, 0, heavy, 0] = 0.0
    v[0, 0, heavy, D // 2:] = 0.0
    v[0, 0, heavy] *= np.float32(2.0 ** lift)  # steps apart
    wk, wv = held(k)[0], held(v)[0]
    want = attention(q[0, :, 0], wk, wv, 1.0)[0]
    s = wk[0, :, 0].astype(np.float64)
    p = np.exp(s) / np.exp(s).sum()
    codes, byte = quantise(v[0, 0])
    step = np.ldexp(1.0, byte.astype(int) - 127)
    bound = 2.0 ** -31 * (p * step).max() * np.abs(codes.astype(np.float64)).sum(0) + 2.0 ** -16 * (p[:, None] * np.abs(wv[0].astype(np.float64))).sum(0)
    cache = fb.PagedKvCache(device, 1, 1, D, (n + 15) // 16, (n + 15) // 16, dtype=fb.I8)
    cache.append(_T(device, k), _T(device, v))
    for ctas in (0, 1, 9):
        cache.set_decode_ctas(ctas)
        got = cache.decode(_T(device, q), 1.0).as_slice()[0, :, 0]
        assert (np.abs(got - want) <= bound).all(), (ctas, (np.abs(got - want) / bound).max())
