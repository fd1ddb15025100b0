"""The 8-bit KV cache: rows written, read back, evicted and attended over, against numpy in 64 bits."""
import numpy as np
import pytest

from cache8_oracle import attention, attention_bound, held, quantise, values
from oracle import oracle as O

pytestmark = pytest.mark.gpu


def _fb():
    import floneum_b200 as fb
    return fb


def _T(device, a, dtype=0):
    return _fb().Tensor.from_slice(device, a.shape, a, dtype)


def _as(a, dtype):
    """f32 values as a tensor of `dtype` holds them."""
    return a if dtype == 0 else O.bf16_round(a) if dtype == 1 else a.astype(np.float16).astype(np.float32)


def _cache(device, B, Hkv, D, tokens, spare=0):
    fb = _fb()
    pages = (tokens + 15) // 16
    return fb.PagedKvCache(device, B, Hkv, D, B * pages + spare, pages + spare, dtype=fb.I8)


# ------------------------------------------------------------------------------------------------------------ writing
@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("B,Hkv,D,steps", [(1, 1, 64, [1]), (2, 3, 64, [5, 1, 11, 30]), (3, 2, 128, [16, 16, 1]), (1, 8, 128, [257]), (20, 1, 128, [15, 2]),
                                            (40, 2, 64, [1, 1, 31])])
def test_appended_rows_read_back_as_the_format_says(device, B, Hkv, D, steps, dtype):
    fb = _fb()
    rng = np.random.default_rng(B * D + len(steps))
    n = sum(steps)
    k, v = (_as(rng.standard_normal((B, Hkv, n, D), dtype=np.float32) * np.exp2(rng.integers(-6, 6, (B, Hkv, n, 1))).astype(np.float32), dtype)
            for _ in range(2))
    cache, at = _cache(device, B, Hkv, D, n), 0
    for s in steps:
        cache.append(_T(device, k[:, :, at:at + s], dtype), _T(device, v[:, :, at:at + s], dtype))
        at += s
    for out in (0, 1, 2):
        got = cache.gather(B, n, out)
        for g, x in zip(got, (k, v)):
            assert np.array_equal(g.as_slice(), held(x)), out  # f16 holds them too: 7 bits of a few units
    # the codes and bytes themselves, wherever the pages are
    codes, scales = cache.read_pages(0, cache.num_pages), cache.read_scales(0, cache.num_pages)
    for which, x in enumerate((k, v)):
        c, b = quantise(x)
        rows = {(c[i].tobytes(), int(b[i])) for i in np.ndindex(b.shape)}
        pool = {(codes[which][p, h, t].tobytes(), int(scales[p, h, which, t])) for p in range(cache.num_pages) for h in range(Hkv) for t in range(16)}
        assert rows <= pool and len(pool - rows) <= 1  # the rest was never written: zeros


def test_appends_of_strided_and_unaligned_views(device):
    import torch
    fb = _fb()
    gen = torch.Generator().manual_seed(4)
    for dt, D in ((torch.float32, 64), (torch.bfloat16, 128), (torch.float16, 64)):
        B, Hkv, n = 2, 3, 21
        whole = torch.randn((B, n, 2 * Hkv, D + 1), generator=gen).to(dt).cuda()
        k, v = (whole[:, :, h:h + Hkv, 1:].transpose(1, 2) for h in (0, Hkv))  # rows start one element off
        cache = _cache(device, B, Hkv, D, n)
        torch.cuda.synchronize()
        cache.append(fb.Tensor.from_torch(device, k), fb.Tensor.from_torch(device, v))
        for g, x in zip(cache.gather(B, n, 0), (k, v)):
            assert np.array_equal(g.as_slice(), held(x.float().cpu().numpy()))


def test_rows_of_mixed_types(device):
    rng = np.random.default_rng(6)
    k, v = (rng.standard_normal((1, 2, 19, 64), dtype=np.float32) for _ in range(2))
    cache = _cache(device, 1, 2, 64, 19)
    cache.append(_T(device, k, 1), _T(device, v, 0))
    gk, gv = cache.gather(1, 19, 0)
    assert np.array_equal(gk.as_slice(), held(O.bf16_round(k))) and np.array_equal(gv.as_slice(), held(v))


@pytest.mark.parametrize("D", [64, 128])
def test_rows_at_the_edges_of_the_format(device, D):
    """Zeros, ties, steps about to change, the largest and the smallest values, and rows that are not finite."""
    f = np.float32
    base = np.zeros(D, f)
    rows = [base]
    for top in (f(127.5), np.nextafter(f(127.5), f(0)), f(63.75), np.nextafter(f(63.75), f(1000)), f(127), f(64), f(1)):
        for e in (-120, 0, 100):
            r = np.linspace(-1, 1, D, dtype=f) * f(50)
            r[3] = -top
            rows.append(np.ldexp(r, e).astype(f))
    ties = np.arange(D, dtype=f) - f(0.5)  # every value half way between two codes: to the even one
    rows += [ties, -ties, np.full(D, np.finfo(f).max, f), np.full(D, np.finfo(f).tiny, f), np.full(D, 1e-45, f), np.full(D, 2.0 ** -127, f)]
    for bad in (np.nan, np.inf, -np.inf):
        r = np.ones(D, f)
        r[D - 1] = bad
        rows.append(r)
    x = np.stack(rows)[None, None]
    n = x.shape[2]
    cache = _cache(device, 1, 1, D, n)
    cache.append(_T(device, x), _T(device, x[:, :, ::-1].copy()))
    gk, gv = cache.gather(1, n, 0)
    assert np.array_equal(gk.as_slice(), held(x), equal_nan=True) and np.array_equal(gv.as_slice(), held(x[:, :, ::-1]), equal_nan=True)
    assert np.isnan(gk.as_slice()[0, 0, -3:]).all() and np.isfinite(gk.as_slice()[0, 0, :-3]).all()
    # a row that is read back and written again: the same codes, except that a row of nothing but zeros may have any step
    second = _cache(device, 1, 1, D, n)
    second.append(gk, gv)
    assert np.array_equal(second.read_pages(0, second.num_pages)[0], cache.read_pages(0, cache.num_pages)[0])
    assert np.array_equal(second.gather(1, n, 0)[0].as_slice(), held(x), equal_nan=True)


def test_a_row_does_not_depend_on_how_it_came(device):
    """One call or many, short or long, with or without neighbours: the same codes and bytes in the same places."""
    rng = np.random.default_rng(5)
    k, v = (rng.standard_normal((2, 2, 70, 128), dtype=np.float32) for _ in range(2))
    pages = []
    for steps in ([70], [1] * 70, [33, 4, 33]):
        cache, at = _cache(device, 2, 2, 128, 80), 0
        table = np.arange(10, dtype=np.int32).reshape(2, 5)[:, ::-1].copy()
        cache.set_page_table(table, np.zeros(2, np.int32))
        for s in steps:
            cache.append(_T(device, k[:, :, at:at + s]), _T(device, v[:, :, at:at + s]))
            at += s
        g = cache.gather(2, 70, 1)
        pages.append([x.as_slice() for x in g])
    for p in pages[1:]:
        assert np.array_equal(p[0], pages[0][0]) and np.array_equal(p[1], pages[0][1])


def test_raw_pages_and_scales_travel(device):
    fb = _fb()
    rng = np.random.default_rng(11)
    cache = fb.PagedKvCache(device, 1, 2, 64, 5, 5, dtype=fb.I8)
    k, v = (rng.integers(-127, 128, (3, 2, 16, 64)).astype(np.int8) for _ in range(2))
    s = rng.integers(110, 140, (3, 2, 2, 16)).astype(np.uint8)
    cache.write_pages(1, k, v)
    cache.write_scales(1, s)
    got = cache.read_pages(1, 3)
    assert np.array_equal(got[0], k) and np.array_equal(got[1], v) and np.array_equal(cache.read_scales(1, 3), s)
    cache.set_page_table(np.array([[3, 1, 2, 0, 0]], np.int32), np.array([40], np.int32))
    order = [2, 0, 1]
    want = np.concatenate([values(k[p], s[p][:, 0]) for p in order], 1)[:, :40]
    assert np.array_equal(cache.gather(1, 40)[0].as_slice()[0], want)


# ------------------------------------------------------------------------------------------------------------ eviction
@pytest.mark.parametrize("D,window,first", [(128, 1, 1), (64, 17, 9), (128, 40, 40), (64, 300, 300)])
def test_a_full_window(device, D, window, first):
    fb = _fb()
    rng = np.random.default_rng(window)
    B, Hq, Hkv = 2, 4, 2
    steps = [first] + [1] * 18 + [3, 1]
    n = sum(steps)
    k, v = (rng.standard_normal((B, Hkv, n, D), dtype=np.float32) for _ in range(2))
    q = rng.standard_normal((B, Hq, n, D), dtype=np.float32)
    cache, at, scale = fb.KvCache.new(2, window, fb.I8), 0, float(D ** -0.5)
    for s in steps:
        ck, cv = cache.append(device, _T(device, k[:, :, at:at + s].copy()), _T(device, v[:, :, at:at + s].copy()))
        at += s
        lo = max(0, at - window)
        wk, wv = held(k[:, :, lo:at]), held(v[:, :, lo:at])
        assert cache.current_seq_len() == at - lo
        assert np.array_equal(ck.as_slice(), wk) and np.array_equal(cv.as_slice(), wv)
        got = _T(device, q[:, :, at - 1:at].copy()).flash_attention(ck, cv, scale).as_slice()
        for b in range(B):
            want = attention(q[b, :, at - 1], wk[b], wv[b], scale)[0]
            assert np.abs(got[b, :, 0] - want).max() <= attention_bound(q[b, :, at - 1], wk[b], wv[b], scale), f"{at} tokens"


@pytest.mark.parametrize("keep", [0, 20, 33, 38, 1000])
def test_truncate_moves_rows_with_their_steps(device, keep):
    rng = np.random.default_rng(keep)
    k, v = (rng.standard_normal((2, 3, 41, 64), dtype=np.float32) * np.exp2(rng.integers(-9, 9, (2, 3, 41, 1))).astype(np.float32) for _ in range(2))
    cache = _cache(device, 2, 3, 64, 48)
    cache.append(_T(device, k), _T(device, v))
    cache.drop_front(1, 38)
    cache.truncate_front(1, keep)
    left = min(keep, 38)
    gk, gv = (x.as_slice() for x in cache.gather(2, 41))
    for g, x in ((gk, k), (gv, v)):
        assert np.array_equal(g[0], held(x[0])) and np.array_equal(g[1, :, :left], held(x[1, :, 41 - left:])) and not g[1, :, left:].any()


def test_a_session_goes_out_and_comes_back(device):
    fb = _fb()
    rng = np.random.default_rng(21)
    k, v = (rng.standard_normal((2, 2, 50, 64), dtype=np.float32) for _ in range(2))
    cache = fb.KvCache.new(2, 40, fb.I8)
    cache.append(device, _T(device, k[:, :, :35].copy()), _T(device, v[:, :, :35].copy()))
    cache.append(device, _T(device, k[:, :, 35:].copy()), _T(device, v[:, :, 35:].copy()))
    session = cache.export_session()
    assert np.array_equal(session["k"], held(k[:, :, 10:])) and session["dtype"] == fb.I8
    back = fb.KvCache.import_session(device, session)
    assert back.dtype == fb.I8
    q = _T(device, rng.standard_normal((2, 4, 1, 64), dtype=np.float32))
    assert np.array_equal(q.flash_attention(back.k(), back.v(), 0.125).as_slice(), q.flash_attention(cache.k(), cache.v(), 0.125).as_slice())
    assert fb.KvCache.import_session(device, {x: session[x] for x in ("k", "v", "max_sequence_len")}).dtype == fb.BF16  # as before there was a choice


# ------------------------------------------------------------------------------------------------------------ decode
def _filled(device, rng, lens, Hkv, D, k_scale=1.0, v_scale=1.0):
    """A cache with permuted pages, every byte of the pools something, and what its rows stand for."""
    fb = _fb()
    pages = [(n + 15) // 16 for n in lens]
    total, widest = sum(pages) + 3, max(pages)
    cache = fb.PagedKvCache(device, len(lens), Hkv, D, total, widest, dtype=fb.I8)
    k, v = (rng.standard_normal((total, Hkv, 16, D)).astype(np.float32) * np.float32(s) for s in (k_scale, v_scale))
    (kc, kb), (vc, vb) = quantise(k), quantise(v)
    order, table, at = rng.permutation(total), np.zeros((len(lens), widest), np.int32), 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    used = np.zeros((total, 16), bool)
    for b, n in enumerate(lens):
        for p in range(pages[b]):
            used[table[b, p], :min(16, n - 16 * p)] = True
    kb, vb = (np.where(used[:, None], x, 255).astype(np.uint8) for x in (kb, vb))  # rows that belong to nobody stand for NaN
    cache.write_pages(0, kc, vc)
    cache.write_scales(0, np.stack([kb, vb], 2))
    cache.set_page_table(table, np.asarray(lens, np.int32))

    def dense(codes, bytes_, b):
        x = values(codes, bytes_)[table[b, :pages[b]]]
        return x.transpose(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :lens[b]]

    cache.table = table
    return cache, [(dense(kc, kb, b), dense(vc, vb, b)) for b in range(len(lens))]


def _check(got, q, rows, scale, out):
    half = {0: 0.0, 1: 2.0 ** -8, 2: 2.0 ** -11}[out]  # the rounding of the result, half a step
    off = norm = 0.0
    for b, (k, v) in enumerate(rows):
        want = attention(q[b, :, 0], k, v, scale)[0]
        bound = attention_bound(q[b, :, 0], k, v, scale)
        assert np.isfinite(got[b]).all()
        assert (np.abs(got[b, :, 0] - want) <= bound + half * (np.abs(want) + bound)).all(), (b, np.abs(got[b, :, 0] - want).max(), bound)
        off += np.square(got[b, :, 0] - want).sum()
        norm += np.square(want).sum()
    # over all values the roundings do not all point one way: 2e-5 of the norm and the result's own rounding
    assert np.sqrt(off / norm) <= 2e-5 + half, np.sqrt(off / norm)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv,lens", [(1, 1, [1]), (4, 1, [2, 15, 16, 17]), (8, 8, [33, 1, 100]), (14, 2, [5, 700, 31, 64, 1]), (64, 8, [1411]),
                                         (6, 2, [3000, 40, 1500]), (32, 4, [130] * 9), (10, 2, [17] * 50), (5, 1, [9000, 16])])
def test_decode(device, D, Hq, Hkv, lens):
    rng = np.random.default_rng(D + Hq + sum(lens))
    cache, rows = _filled(device, rng, lens, Hkv, D)
    scale = float(D ** -0.5)
    for dtype in (0, 1, 2):
        q = _as(rng.standard_normal((len(lens), Hq, 1, D)).astype(np.float32), dtype)
        for out in (0, 1, 2):
            _check(cache.decode(_T(device, q, dtype), scale, out_dtype=out).as_slice(), q, rows, scale, out)
        assert np.array_equal(cache.decode_host(q, scale), cache.decode(_T(device, q, 0), scale).as_slice())


@pytest.mark.parametrize("ctas", [1, 2, 5, 37, 148])
def test_decode_at_any_grid(device, ctas):
    """Shares of the pages that begin and end anywhere, sequences of one page among long ones."""
    rng = np.random.default_rng(ctas)
    lens = [1, 700, 16, 31, 2000, 1, 1, 333]
    for D, Hq, Hkv in ((64, 8, 2), (128, 12, 3)):
        cache, rows = _filled(device, rng, lens, Hkv, D)
        cache.set_decode_ctas(ctas)
        q = rng.standard_normal((len(lens), Hq, 1, D)).astype(np.float32)
        _check(cache.decode(_T(device, q), float(D ** -0.5)).as_slice(), q, rows, float(D ** -0.5), 0)


@pytest.mark.parametrize("D,lens", [(128, [200, 1, 77]), (64, [4000])])
def test_decode_partial_records(device, D, lens):
    from floneum_b200.cache import lse_combine
    rng = np.random.default_rng(D)
    cache, rows = _filled(device, rng, lens, 2, D)
    q = rng.standard_normal((len(lens), 8, 1, D)).astype(np.float32)
    part = cache.decode_partial(_T(device, q), 0.1).as_slice()
    for b, (k, v) in enumerate(rows):
        want, m, l = attention(q[b, :, 0], k, v, 0.1)
        bound = attention_bound(q[b, :, 0], k, v, 0.1)
        # m may be any reference near the maximum: what the record says is l e^m and O / l
        lse = part[b, :, 0].astype(np.float64) + np.log(part[b, :, 1].astype(np.float64))
        assert np.abs(lse - (m + np.log(l))).max() <= 1e-5
        assert np.abs(part[b, :, 2:] / part[b, :, 1:2] - want).max() <= bound + 2.0 ** -22 * np.abs(want).max()
    whole = lse_combine(device, _T(device, part[None])).as_slice()
    assert np.abs(whole - cache.decode(_T(device, q), 0.1).as_slice()[:, :, 0]).max() <= 2.0 ** -20 * np.abs(whole).max()


def test_partial_records_of_an_empty_sequence(device):
    fb = _fb()
    rng = np.random.default_rng(31)
    cache, rows = _filled(device, rng, [40, 16, 90], 2, 64)
    table = np.zeros((3, cache.max_pages_per_seq), np.int32)
    table[0, :3], table[2, :6] = [0, 1, 2], [3, 4, 5, 6, 7, 8]
    cache.write_scales(0, np.full((cache.num_pages, 2, 2, 16), 127, np.uint8))
    q = _T(device, rng.standard_normal((3, 4, 1, 64)).astype(np.float32))
    for lens in ([40, 0, 90], [0, 0, 0], [0, 0, 7]):
        cache.set_page_table(table, np.asarray(lens, np.int32))
        part = cache.decode_partial(q, 0.125).as_slice()
        for b, n in enumerate(lens):
            if n == 0:
                assert np.isneginf(part[b, :, 0]).all() and not part[b, :, 1:].any()
            else:
                assert np.isfinite(part[b]).all() and (part[b, :, 1] > 0).all()
        with pytest.raises(fb.FusorCudaError):
            cache.decode(q, 0.125)


def test_decode_of_peaked_and_very_different_rows(device):
    """One key far above the others, values whose steps lie 2^60 apart, zero rows of large weight, large and tiny queries."""
    fb = _fb()
    rng = np.random.default_rng(77)
    D, Hkv, n = 128, 1, 500
    scale = float(D ** -0.5)
    for name in ("peak", "steps", "zeros", "large q", "small q", "large v", "large k"):
        k, v = (rng.standard_normal((1, Hkv, n, D)).astype(np.float32) for _ in range(2))
        q = rng.standard_normal((1, 4, 1, D)).astype(np.float32)
        if name == "peak":
            k[0, 0, 333] = q[0, 1, 0] * 3
        if name == "steps":  # the rows with the weight have the small values
            v *= np.exp2(rng.integers(-30, 30, (1, Hkv, n, 1))).astype(np.float32)
            k[0, 0, 10] = q[0, 0, 0] * 2
            v[0, 0, 10] *= np.float32(2.0 ** -60)
        if name == "zeros":
            k[0, 0, 100:120] = q[0, :, 0].mean(0) * 3
            v[0, 0, 100:120] = 0
        if name == "large q":
            q, k = q * np.float32(2.0 ** 60), k * np.float32(2.0 ** -60)
        if name == "small q":
            q, k = q * np.float32(2.0 ** -70), k * np.float32(2.0 ** 70)
        if name == "large v":
            v *= np.float32(2.0 ** 100)
        if name == "large k":
            q, k = q * np.float32(2.0 ** -60), k * np.float32(2.0 ** 60)
        cache = _cache(device, 1, Hkv, D, n)
        cache.append(_T(device, k), _T(device, v))
        got = cache.decode(_T(device, q), scale).as_slice()
        wk, wv = held(k)[0], held(v)[0]
        want = attention(q[0, :, 0], wk, wv, scale)[0]
        assert np.isfinite(got).all(), name
        assert np.abs(got[0, :, 0] - want).max() <= attention_bound(q[0, :, 0], wk, wv, scale), name


def test_values_that_are_not_finite_stay_with_their_sequence(device):
    """A row of NaN makes NaN of the sequence and head it belongs to, K or V, and of nothing else; evicted, it is gone."""
    rng = np.random.default_rng(9)
    B, Hkv, n, D = 3, 2, 40, 64
    k, v = (rng.standard_normal((B, Hkv, n, D)).astype(np.float32) for _ in range(2))
    k[0, 0, 7, 3], v[1, 1, 5, 0] = np.nan, np.inf
    q = rng.standard_normal((B, 8, 1, D)).astype(np.float32)
    cache = _cache(device, B, Hkv, D, n)
    cache.append(_T(device, k), _T(device, v))
    got = cache.decode(_T(device, q), 0.125).as_slice()[:, :, 0]
    bad = np.zeros((B, 8), bool)
    bad[0, :4], bad[1, 4:] = True, True
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
    for b in range(2):
        cache.drop_front(b, n - 9)
    got = cache.decode(_T(device, q), 0.125).as_slice()
    for b in range(B):
        lo = 9 if b < 2 else 0
        wk, wv = held(k)[b, :, lo:], held(v)[b, :, lo:]
        assert np.abs(got[b, :, 0] - attention(q[b, :, 0], wk, wv, 0.125)[0]).max() <= attention_bound(q[b, :, 0], wk, wv, 0.125)
    q[2, 5, 0, 11] = np.inf  # a query that is not finite: its own row
    got = cache.decode(_T(device, q), 0.125).as_slice()[:, :, 0]
    assert np.isnan(got[2, 5]).all() and np.isfinite(np.delete(got.reshape(-1, D), 2 * 8 + 5, 0)).all()


@pytest.mark.parametrize("n", [1, 16, 300, 5000])
def test_a_head_whose_values_are_all_not_finite(device, n):
    rng = np.random.default_rng(n)
    k, v = (rng.standard_normal((2, 2, n, 128)).astype(np.float32) for _ in range(2))
    v[1, 0, :, 7] = np.inf
    q = rng.standard_normal((2, 4, 1, 128)).astype(np.float32)
    cache = _cache(device, 2, 2, 128, n)
    cache.append(_T(device, k), _T(device, v))
    got = cache.decode(_T(device, q), 0.1).as_slice()
    assert np.isnan(got[1, :2]).all() and np.isfinite(got[1, 2:]).all()
    _check(got[:1], q[:1], [(held(k)[0], held(v)[0])], 0.1, 0)


def test_decode_of_strided_queries_and_results(device):
    import torch
    fb = _fb()
    rng = np.random.default_rng(15)
    cache, rows = _filled(device, rng, [100, 33], 2, 64)
    for dt, code in ((torch.float32, 0), (torch.bfloat16, 1)):
        wide = torch.tensor(rng.standard_normal((2, 3, 8, 2 * 64)).astype(np.float32)).to(dt).cuda()
        q = wide[:, 1:2, :, 64:].transpose(1, 2)
        out = torch.full((2, 3, 8, 64), 7.0, device="cuda", dtype=dt)
        torch.cuda.synchronize()
        cache.decode(fb.Tensor.from_torch(device, q), 0.125, out=fb.Tensor.from_torch(device, out[:, 1:2].transpose(1, 2)))
        device.synchronize()
        _check(out[:, 1].float().cpu().numpy()[:, :, None], q.float().cpu().numpy(), rows, 0.125, code)
        assert (out[:, 0] == 7).all() and (out[:, 2] == 7).all()


def test_two_decodes_at_once_and_a_replayed_one(device):
    """Two contexts with caches of their own on streams of their own, and a decode captured into a graph and replayed with other
    queries in the same memory."""
    import torch
    fb = _fb()
    rng = np.random.default_rng(3)
    other = fb.Device.gpu(0)
    sides = []
    for dev in (device, other):
        cache, rows = _filled(dev, rng, [3000, 40, 1200], 2, 128)
        q = rng.standard_normal((3, 8, 1, 128)).astype(np.float32)
        sides.append((dev, cache, rows, q, _T(dev, q)))
    outs = [[s[1].decode(s[4], 0.1) for s in sides] for _ in range(10)]
    for pair in outs:
        for s, out in zip(sides, pair):
            _check(out.as_slice(), s[3], s[2], 0.1, 0)
            assert np.array_equal(out.as_slice(), outs[0][sides.index(s)].as_slice())  # no order of atomics in it
    stream = torch.cuda.Stream()
    dev3 = fb.Device.gpu(0, stream.cuda_stream)
    cache, rows = _filled(dev3, rng, [3000, 40, 1200], 2, 128)
    q = torch.zeros((3, 8, 1, 128), device="cuda")
    out = torch.zeros_like(q)
    tq, to = fb.Tensor.from_torch(dev3, q), fb.Tensor.from_torch(dev3, out)
    torch.cuda.synchronize()
    cache.decode(tq, 0.1, out=to)  # the tables are on the device before the capture
    dev3.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        cache.decode(tq, 0.1, out=to)
    for _ in range(3):
        host = rng.standard_normal((3, 8, 1, 128)).astype(np.float32)
        q.copy_(torch.tensor(host))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _check(out.cpu().numpy(), host, rows, 0.1, 0)
    del graph


@pytest.mark.parametrize("D", [64, 128])
def test_more_sequences_than_warps(device, D):
    """Hundreds of sequences of a token to three pages: shares that hold many of them whole."""
    rng = np.random.default_rng(300 + D)
    lens = [int(x) for x in rng.integers(1, 41, 300)]
    cache, rows = _filled(device, rng, lens, 4, D)
    q = rng.standard_normal((300, 8, 1, D)).astype(np.float32)
    for ctas in (0, 3, 148, 0):
        cache.set_decode_ctas(ctas)
        _check(cache.decode(_T(device, q), float(D ** -0.5)).as_slice(), q, rows, float(D ** -0.5), 0)


def test_one_cache_at_one_grid_after_another(device):
    """What a launch leaves behind for the next: the same result from every grid, again and again, and as captured."""
    import torch
    fb = _fb()
    stream = torch.cuda.Stream()
    dev = fb.Device.gpu(0, stream.cuda_stream)
    rng = np.random.default_rng(41)
    cache, rows = _filled(dev, rng, [5000, 7, 900, 16, 3100], 3, 128)
    q = rng.standard_normal((5, 12, 1, 128)).astype(np.float32)
    tq = _T(dev, q)
    first = {}
    for ctas in (148, 1, 40, 148, 9, 0, 40, 1, 9, 0):
        cache.set_decode_ctas(ctas)
        got = cache.decode(tq, 0.09).as_slice()
        _check(got, q, rows, 0.09, 0)
        assert np.array_equal(got, first.setdefault(ctas, got))
    for ctas in (40, 0):
        cache.set_decode_ctas(ctas)
        out = fb.Tensor.zeros(dev, q.shape)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
            for _ in range(3):
                cache.decode(tq, 0.09, out=out)
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out.as_slice(), first[ctas])
        del graph


@pytest.mark.parametrize("B,past", [(1, 3), (2, 40), (40, 100)])
def test_each_launch_sees_what_the_one_before_wrote(device, B, past):
    """Rows rotated and written, attended over and read back, with nothing between the launches: what comes of it when each is waited for.
    40 sequences: their lengths come from the device's tables, and do not travel with the launch."""
    fb = _fb()
    rng = np.random.default_rng(B)
    steps, Hq, Hkv, D = 24, 8, 2, 128
    x = [rng.standard_normal((B, h, past + steps, D)).astype(np.float32) for h in (Hq, Hkv, Hkv)]

    def run(wait):
        rope, cache, outs = fb.RopeCache.new(D, past + steps, 10000.0, device), _cache(device, B, Hkv, D, past + steps), []
        parts = [[_T(device, np.ascontiguousarray(t[:, :, at:end])) for t in x] for at, end in [(0, past)] + [(past + i, past + i + 1) for i in range(steps)]]
        for i, (q, k, v) in enumerate(parts):
            q = rope.forward_append(q, k, v, cache)
            wait()
            if i:
                outs.append(cache.decode(q, 0.09))
                wait()
            outs += cache.gather(B, past + i, 1)
            wait()
        return [t.as_slice() for t in outs]

    alone = run(device.synchronize)
    for _ in range(3):
        for got, want in zip(run(lambda: None), alone):
            assert np.array_equal(got, want)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("exchange", [False, True])
def test_a_captured_decode_meets_other_lengths(device, D, exchange):
    """Captured at one set of lengths, replayed at shorter ones (fewer pages than warps, to a page in all) and at the first ones again."""
    import torch
    fb = _fb()
    from floneum_b200.sharding import PeerExchange
    stream = torch.cuda.Stream()
    dev = fb.Device.gpu(0, stream.cuda_stream)
    rng = np.random.default_rng(D)
    lens = [6000, 33, 2500]
    cache, rows = _filled(dev, rng, lens, 2, D)
    cache.set_decode_ctas(148)  # not the cluster
    q = rng.standard_normal((3, 8, 1, D)).astype(np.float32)
    tq = _T(dev, q)
    ex = PeerExchange(dev, 0, 1, 3 * 8 * (D + 2)) if exchange else None
    there = torch.zeros((3, 8, D) if exchange else q.shape, device="cuda")
    torch.cuda.synchronize()
    out = fb.Tensor.from_torch(dev, there)
    decode = (lambda: ex.decode(cache, tq, 0.09, out)) if exchange else (lambda: cache.decode(tq, 0.09, out=out))
    decode()
    dev.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
        decode()
    for now in ([6000, 33, 2500], [400, 33, 100], [17, 1, 16], [6000, 1, 40], [1, 33, 1], [6000, 33, 2500]):
        cache.set_page_table(cache.table, np.asarray(now, np.int32))
        decode()  # the tables to the device
        dev.synchronize()
        there.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = there.cpu().numpy()
        _check(got[:, :, None] if exchange else got, q, [tuple(x[:, :n] for x in r) for r, n in zip(rows, now)], 0.09, 0)
    del graph
    if ex:
        ex.close()


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_any_scale_and_a_query_of_zeros(device, scale):
    rng = np.random.default_rng(2)
    cache, rows = _filled(device, rng, [300, 5], 2, 64)
    q = rng.standard_normal((2, 6, 1, 64)).astype(np.float32)
    q[0, 1] = 0
    _check(cache.decode(_T(device, q), scale).as_slice(), q, rows, scale, 0)


def test_exchange_decode_of_one_rank(device):
    """The KV-chunk decode's merge and exchange over 8-bit pages, with a sequence of which this rank has no key."""
    fb = _fb()
    from floneum_b200.sharding import PeerExchange
    rng = np.random.default_rng(19)
    lens = [3000, 20, 700]
    cache, rows = _filled(device, rng, lens, 2, 128)
    q = rng.standard_normal((3, 8, 1, 128)).astype(np.float32)
    ex = PeerExchange(device, 0, 1, 3 * 8 * 130)
    for ctas in (0, 5, 148, 0):
        cache.set_decode_ctas(ctas)
        out = fb.Tensor.zeros(device, (3, 8, 128))
        ex.decode(cache, _T(device, q), 0.09, out)
        _check(out.as_slice()[:, :, None], q, rows, 0.09, 0)
    empty = fb.PagedKvCache(device, 3, 2, 128, 4, 2, dtype=fb.I8)
    empty.set_page_table(np.array([[0, 1], [0, 0], [2, 0]], np.int32), np.array([20, 0, 3], np.int32))
    for _ in range(2):
        out = fb.Tensor.from_slice(device, (3, 8, 128), np.full((3, 8, 128), 7.0))
        ex.decode(empty, _T(device, q), 0.09, out)
        assert not out.as_slice().any()  # rows of zeros, and no rows
    ex.close()


def test_pools_of_more_than_four_gigabytes(device):
    """Pages behind byte 2^32 of a pool: written, rotated into, read back, moved and attended over."""
    fb = _fb()
    rng = np.random.default_rng(44)
    pages, Hkv, D = 270000, 8, 128  # 4.4 GB a pool
    assert pages * Hkv * 16 * D > 2 ** 32
    cache = fb.PagedKvCache(device, 1, Hkv, D, pages, 4, dtype=fb.I8)
    rope = fb.RopeCache.new(D, 64, 10000.0, device)
    k, v = (rng.standard_normal((1, Hkv, 33, D)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((1, 8, 12, D)).astype(np.float32)
    cache.set_page_table(np.array([[pages - 1, 0, 0, 0]], np.int32), np.array([1], np.int32))
    cache.append(_T(device, k[:, :, :15].copy()), _T(device, v[:, :, :15].copy()))
    cache.set_page_table(np.array([[pages - 1, 3, pages - 2, 0]], np.int32), np.array([33], np.int32))
    cache.append(_T(device, k[:, :, 15:18].copy()), _T(device, v[:, :, 15:18].copy()))
    cache.rope_append(_T(device, q), _T(device, k[:, :, 21:33].copy()), _T(device, v[:, :, 21:33].copy()), rope.cos, rope.sin, 5)
    gk, gv = (x.as_slice() for x in cache.gather(1, 48))
    zero = np.zeros_like(k[:, :, :1])
    want_k = np.concatenate([zero, held(k[:, :, :15]), np.repeat(zero, 17, 2), held(k[:, :, 15:18]),
                             held(O.rope(k[:, :, 21:33], rope.cos.as_slice(), rope.sin.as_slice(), 5, False))], 2)
    want_v = np.concatenate([zero, held(v[:, :, :15]), np.repeat(zero, 17, 2), held(v[:, :, 15:18]), held(v[:, :, 21:33])], 2)
    assert np.array_equal(gk, want_k) and np.array_equal(gv, want_v)
    one = q[:, :, :1].copy()
    for ctas in (0, 2):
        cache.set_decode_ctas(ctas)
        _check(cache.decode(_T(device, one), 0.09).as_slice(), one, [(want_k[0], want_v[0])], 0.09, 0)
    cache.truncate_front(0, 30)
    assert np.array_equal(cache.gather(1, 30)[0].as_slice(), want_k[:, :, 18:])
    cache.close()


def test_refusals(device):
    fb = _fb()
    UN, SH, IN = fb._lib.UNSUPPORTED, fb._lib.SHAPE_MISMATCH, fb._lib.INVALID_ARGUMENT

    def refused(code, call):
        with pytest.raises(fb.FusorCudaError) as e:
            call()
        assert e.value.code == code

    for dtype in (0, 2, 4, 9):
        refused(UN, lambda: fb.PagedKvCache(device, 1, 1, 64, 4, 4, dtype=dtype))
    refused(UN, lambda: fb.PagedKvCache(device, 1, 1, 96, 4, 4, dtype=fb.I8))
    refused(UN, lambda: fb.PagedKvCache(device, 1, 1, 64, 4, 4, page_tokens=32, dtype=fb.I8))
    cache = fb.PagedKvCache(device, 2, 2, 64, 8, 4, dtype=fb.I8)
    z = lambda *s, dtype=0: _T(device, np.zeros(s, np.float32), dtype)
    refused(IN, lambda: cache.decode(z(2, 4, 1, 64), 1.0))  # nothing in it
    refused(SH, lambda: cache.append(z(2, 2, 3, 128), z(2, 2, 3, 128)))
    refused(SH, lambda: cache.append(z(2, 2, 3, 64), z(2, 2, 4, 64)))
    refused(IN, lambda: cache.append(z(3, 2, 3, 64), z(3, 2, 3, 64)))
    refused(fb._lib.OUT_OF_PAGES, lambda: cache.append(z(2, 2, 65, 64), z(2, 2, 65, 64)))
    cache.append(z(2, 2, 20, 64), z(2, 2, 20, 64))
    refused(UN, lambda: cache.decode(z(2, 4, 2, 64), 1.0))
    refused(SH, lambda: cache.decode(z(2, 3, 1, 64), 1.0))
    refused(UN, lambda: cache.decode(z(2, 18, 1, 64), 1.0))  # nine query heads a kv head
    refused(SH, lambda: cache.gather(2, 21))
    plain = fb.PagedKvCache(device, 1, 1, 64, 4, 4)
    refused(UN, plain.scales)
    refused(UN, lambda: plain.read_scales(0, 1))
    refused(UN, lambda: plain.write_scales(0, np.zeros((1, 1, 2, 16), np.uint8)))
    refused(IN, lambda: cache.read_scales(7, 2))
    assert np.array_equal(cache.gather(2, 20)[0].as_slice(), np.zeros((2, 2, 20, 64)))  # as it was


# ------------------------------------------------------------------------------------------------------------ a run
@pytest.mark.parametrize("interleaved,pages", [(False, "i8"), (True, "i8"), (False, "bf16")])
def test_a_chat_with_a_picture_in_it(device, interleaved, pages):
    """A layer's part of a chat: a prompt with an image's tokens on three axes, a follow-up, single tokens; rotation with the
    append, attention over the cache each time.  Every step against 64 bits on the rows the cache must hold."""
    fb = _fb()
    rng = np.random.default_rng(12)
    B, Hq, Hkv, D = 2, 8, 2, 64
    scale = float(D ** -0.5)
    axes = fb.axes_of_sections([8, 12, 12])
    rope = fb.RopeCache.new(D, 128, 10000.0, device)
    cos, sin = rope.cos.as_slice(), rope.sin.as_slice()
    cache, masks = fb.KvCache.new(2, 200, fb.I8 if pages == "i8" else fb.BF16), fb.MaskCache()
    keep = held if pages == "i8" else O.bf16_round
    wk, wv = np.zeros((B, Hkv, 0, D), np.float32), np.zeros((B, Hkv, 0, D), np.float32)
    grid = np.stack(np.meshgrid(np.arange(5), np.arange(7), indexing="ij")).reshape(2, -1)
    picture = np.concatenate([np.full((3, 6), 0) + np.arange(6), np.concatenate([np.zeros((1, 35), int), grid]) + 6, np.arange(9)[None] + np.full((3, 1), 13)], 1)
    past = 0
    for pos in (picture, np.arange(20)[None] + np.full((3, 1), 22), *[np.full((3, 1), 42 + i) for i in range(4)]):
        n = pos.shape[1]
        ids = np.stack([pos, pos + 5], 1)  # [axis, B, n]: the second sequence stands five further on
        q, k, v = (rng.standard_normal((B, h, n, D)).astype(np.float32) for h in (Hq, Hkv, Hkv))
        q_rot, ck, cv = rope.forward_append(*(_T(device, x) for x in (q, k, v)), cache, interleaved=interleaved,
                                            positions=_T(device, ids, fb.U32), axes=axes)
        row = ids[axes].transpose(1, 2, 0)  # [B, n, D / 2]
        c, s = (t[row, np.arange(D // 2)][:, None] for t in (cos, sin))
        turned = []
        for x in (q, k):
            a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :D // 2], x[..., D // 2:])
            re, im = a * c - b * s, a * s + b * c
            turned.append(np.stack([re, im], -1).reshape(x.shape) if interleaved else np.concatenate([re, im], -1))
        assert np.array_equal(q_rot.as_slice(), turned[0])
        wk, wv = np.concatenate([wk, keep(turned[1])], 2), np.concatenate([wv, keep(v)], 2)
        assert np.array_equal(ck.as_slice(), wk) and np.array_equal(cv.as_slice(), wv)
        got = q_rot.flash_attention(ck, cv, scale, (masks.get_mask(n, past, None, device), fb.MaskKind.QKMask)).as_slice()
        past += n
        for b in range(B):
            for t in range(n):
                upto = past - n + t + 1
                # several tokens, and any token over a bf16 cache: queries rounded to bf16, a score off by 2^-8 of |q| |k|
                rounded = n > 1 or pages == "bf16"
                qt = O.bf16_round(turned[0][b, :, t]) if rounded else turned[0][b, :, t]
                want = attention(qt, wk[b, :, :upto], wv[b, :, :upto], scale)[0]
                tol = attention_bound(qt, wk[b, :, :upto], wv[b, :, :upto], scale)
                assert np.abs(got[b, :, t] - want).max() <= (max(tol, 2e-3) if rounded else tol), (past, b, t)
