"""A captured decode over 8-bit pages whose sequences became empty after the capture."""
import numpy as np
import pytest

from cache8_oracle import attention, attention_bound, held, quantise

pytestmark = pytest.mark.gpu


def _fb():
    import floneum_b200 as fb
    return fb


def _T(device, a, dtype=0):
    return _fb().Tensor.from_slice(device, a.shape, a, dtype)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ctas", [0, 148])
@pytest.mark.parametrize("out", [0, 1, 2])
def test_a_sequence_without_keys_gives_zeros(device, D, ctas, out):
    """A batch with idle places, replayed: what a place without keys gives is zeros on every path, not what lay in the result."""
    import torch
    fb = _fb()
    stream = torch.cuda.Stream()
    dev = fb.Device.gpu(0, stream.cuda_stream)
    rng = np.random.default_rng(D + ctas)
    lens, Hq, Hkv, scale = [3000, 40, 1200], 6, 2, 0.1
    widest = (3000 + 15) // 16
    cache = fb.PagedKvCache(dev, 3, Hkv, D, 3 * widest, widest, dtype=fb.I8)
    k, v = (rng.standard_normal((3, Hkv, 16 * widest, D)).astype(np.float32) for _ in range(2))
    table = rng.permutation(3 * widest).reshape(3, widest).astype(np.int32)
    codes, scales = [np.zeros((3 * widest, Hkv, 16, D), np.int8) for _ in range(2)], np.zeros((3 * widest, Hkv, 2, 16), np.uint8)
    for which, x in enumerate((k, v)):
        c, e = quantise(x)
        codes[which][table] = c.reshape(3, Hkv, widest, 16, D).swapaxes(1, 2)
        scales[table, :, which] = e.reshape(3, Hkv, widest, 16).swapaxes(1, 2)
    cache.write_pages(0, *codes)
    cache.write_scales(0, scales)
    cache.set_page_table(table, np.asarray(lens, np.int32))
    cache.set_decode_ctas(ctas)
    tt = {0: torch.float32, 1: torch.bfloat16, 2: torch.float16}[out]
    wide = torch.full((3, 2, Hq, D), 7.0, device="cuda", dtype=tt)  # the result's rows lie among others
    q = rng.standard_normal((3, Hq, 1, D)).astype(np.float32)
    tq = _T(dev, q)
    torch.cuda.synchronize()
    res = fb.Tensor.from_torch(dev, wide[:, :1].transpose(1, 2))
    cache.decode(tq, scale, out=res)
    dev.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
        cache.decode(tq, scale, out=res)
    half = {0: 0.0, 1: 2.0 ** -8, 2: 2.0 ** -11}[out]
    for now in ([3000, 0, 1200], [0, 40, 0], [0, 0, 1], [0, 0, 0], [3000, 40, 1200]):
        cache.set_page_table(table, np.asarray(now, np.int32))
        dev.synchronize()
        wide.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = wide.float().cpu().numpy()
        assert (got[:, 1] == 7).all()
        for b, n in enumerate(now):
            if n == 0:
                assert not got[b, 0].any(), (now, b)
                continue
            rows = [held(x)[b, :, :n] for x in (k, v)]
            want, bound = attention(q[b, :, 0], *rows, scale)[0], attention_bound(q[b, :, 0], *rows, scale)
            assert (np.abs(got[b, 0] - want) <= bound + half * (np.abs(want) + bound)).all(), (now, b)
    del graph


@pytest.mark.parametrize("window", [0, 900])
def test_a_cache_that_was_reset(device, window):
    """Decodes from many shares, eager and captured, between resets: each as from a cache of its own."""
    import torch
    fb = _fb()
    stream = torch.cuda.Stream()
    dev = fb.Device.gpu(0, stream.cuda_stream)
    rng = np.random.default_rng(window)
    D, scale = 64, 0.125
    cache = fb.PagedKvCache(dev, 2, 2, D, 2 * 60, 60, dtype=fb.I8)
    cache.set_window(window)
    cache.set_decode_ctas(40)
    for n in (900, 900, 33, 900):
        k, v = (rng.standard_normal((2, 2, n, D)).astype(np.float32) for _ in range(2))
        q = rng.standard_normal((2, 4, 1, D)).astype(np.float32)
        if window == 0 or n < window:
            cache.reset()
        cache.append(_T(dev, k), _T(dev, v))
        tq, out = _T(dev, q), fb.Tensor.zeros(dev, q.shape)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
            cache.decode(tq, scale, out=out)
        got = []
        for _ in range(2):
            got.append(cache.decode(tq, scale).as_slice())
            graph.replay()
            torch.cuda.synchronize()
            got.append(out.as_slice())
        for g in got:
            assert np.array_equal(g, got[0])
            for b in range(2):
                want, bound = attention(q[b, :, 0], held(k)[b], held(v)[b], scale)[0], attention_bound(q[b, :, 0], held(k)[b], held(v)[b], scale)
                assert (np.abs(g[b, :, 0] - want) <= bound).all()
        del graph
