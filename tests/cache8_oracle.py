"""What an 8-bit cache holds, and attention over it, restated in numpy (64 bits) from the definition."""
import numpy as np


def quantise(x):
    """f32 rows [..., D] -> int8 codes [..., D] and scale bytes uint8 [...]."""
    x = np.asarray(x, np.float32).astype(np.float64)
    fine = np.isfinite(x).all(-1)
    top = np.where(fine, np.abs(x).max(-1), 0.0)
    m, e = np.frexp(top / 127.5)  # top / 127.5 = m 2^e, m in [1/2, 1): the smallest whole exponent above it is e
    e = np.where(top > 0, np.clip(e, -126, 121), -126)  # 64 * 2^122 would be infinite: there codes end at 127
    codes = np.clip(np.rint(np.where(fine[..., None], x, 0.0) * np.ldexp(1.0, -e)[..., None]), -127, 127)
    return codes.astype(np.int8), np.where(fine, e + 127, 255).astype(np.uint8)


def values(codes, byte):
    """The f32 values that codes and bytes stand for."""
    step = np.where(byte == 255, np.nan, np.ldexp(1.0, byte.astype(int) - 127))
    return (codes.astype(np.float64) * step[..., None]).astype(np.float32)


def held(x):
    return values(*quantise(x))


def attention(q, k, v, scale):
    """q [Hq, D], k and v [Hkv, n, D] -> (out [Hq, D], m [Hq], l [Hq]) in 64 bits; m and l in natural-log units."""
    Hq, Hkv = q.shape[0], k.shape[0]
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    k, v = np.repeat(k, Hq // Hkv, 0), np.repeat(v, Hq // Hkv, 0)
    s = np.einsum("hd,hnd->hn", q, k) * scale
    m = s.max(-1)
    p = np.exp(s - m[:, None])
    l = p.sum(-1)
    return np.einsum("hn,hnd->hd", p, v) / l[:, None], m, l


def attention_bound(q, k, v, scale):
    """How far an f32 result may be off, from roundings alone: a score's products and sums (D + 8 of 2^-24 of sum |q k| scale; the
    query in two 11-bit terms adds 2^-21), which the exponential turns into the same error relative to each weight, for the
    weight and for the sum; exponentials, two-term weights and the sums themselves 2^-19 on top, of the largest |v|."""
    D = q.shape[-1]
    s = np.einsum("hd,hnd->hn", np.abs(np.asarray(q, np.float64)), np.repeat(np.abs(np.asarray(k, np.float64)), q.shape[0] // k.shape[0], 0)) * abs(scale)
    return (2 * s.max() * ((D + 8) * 2.0 ** -24 + 2.0 ** -21) + 2.0 ** -19) * np.abs(np.asarray(v, np.float64)).max()
