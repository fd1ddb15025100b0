"""Rotary positions with several axes: alone and fused with the append, against the rotation in f32 with each product rounded."""
import numpy as np
import pytest

from cache8_oracle import held
from oracle import oracle as O

pytestmark = pytest.mark.gpu


def _fb():
    import floneum_b200 as fb
    return fb


def _T(device, a, dtype=0):
    return _fb().Tensor.from_slice(device, a.shape, a, dtype)


def _as(a, dtype):
    return a if dtype == 0 else O.bf16_round(a) if dtype == 1 else a.astype(np.float16).astype(np.float32)


def _turn(x, cos, sin, ids, axes, interleaved):
    """x [B, H, n, D]; ids [axes, B, n]; numpy rounds every product and every sum to f32."""
    half = x.shape[-1] // 2
    row = ids[np.asarray(axes)].transpose(1, 2, 0)
    c, s = (t[row, np.arange(half)][:, None] for t in (cos, sin))
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    re, im = a * c - b * s, a * s + b * c
    return np.stack([re, im], -1).reshape(x.shape) if interleaved else np.concatenate([re, im], -1)


CASES = [(1, 1, 1, 2, [1]), (2, 3, 5, 6, [1, 2]), (1, 16, 70, 80, [20, 20]), (2, 2, 33, 96, [16, 16, 16]), (3, 8, 40, 128, [16, 24, 24]),
         (1, 5, 19, 64, [11, 10, 11]), (1, 2, 9, 512, [100, 156]), (1, 32, 257, 128, [64]), (2, 4, 8, 32, [3, 3, 5, 5]), (1, 2, 3, 48, [0, 24])]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,H,n,D,sections", CASES)
def test_rope_axes(device, B, H, n, D, sections, interleaved):
    fb = _fb()
    rng = np.random.default_rng(n + D)
    rows = 300
    cos, sin = (rng.uniform(-1, 1, (rows, D // 2)).astype(np.float32) for _ in range(2))
    tc, ts = _T(device, cos), _T(device, sin)
    orders = [fb.axes_of_sections(sections), rng.integers(0, len(sections), D // 2).astype(np.uint8)]
    for dtype, out in ((0, None), (1, None), (2, None), (1, 0), (0, 1)):
        x = _as(rng.standard_normal((B, H, n, D)).astype(np.float32), dtype)
        ids = rng.integers(0, rows, (len(sections), B, n)).astype(np.uint32)
        ids[0, 0, 0], ids[-1, -1, -1] = rows - 1, 0
        for axes in orders:
            got = fb.rope_axes(_T(device, x, dtype), tc, ts, _T(device, ids, fb.U32), axes, interleaved, out_dtype=out).as_slice()
            assert np.array_equal(got, _as(_turn(x, cos, sin, ids, axes, interleaved), dtype if out is None else out))
        # the same positions for every sequence
        got = fb.rope_axes(_T(device, x, dtype), tc, ts, _T(device, ids[:, 0], fb.U32), axes, interleaved, out_dtype=out).as_slice()
        assert np.array_equal(got, _as(_turn(x, cos, sin, np.repeat(ids[:, :1], B, 1), axes, interleaved), dtype if out is None else out))


def test_one_position_on_every_axis_is_rope(device):
    fb = _fb()
    rng = np.random.default_rng(3)
    rope = fb.RopeCache.new(128, 64, 10000.0, device)
    q, k = (_T(device, rng.standard_normal((2, h, 30, 128)).astype(np.float32), 1) for h in (8, 2))
    ids = _T(device, np.broadcast_to(np.arange(30) + 11, (3, 30)).astype(np.uint32), fb.U32)
    for interleaved in (False, True):
        a = rope.forward_axes(q, k, ids, fb.axes_of_sections([16, 24, 24]), interleaved)
        b = (rope.forward_interleaved if interleaved else rope.forward)(q, k, 11)
        assert all(np.array_equal(x.as_slice(), y.as_slice()) for x, y in zip(a, b))


@pytest.mark.parametrize("B,Hq,Hkv,n,D,sections", [(1, 16, 16, 70, 80, [20, 20]), (2, 14, 2, 33, 128, [16, 24, 24]), (3, 3, 1, 1, 64, [32]), (2, 4, 2, 9, 6, [1, 2]),
                                                   (1, 1, 9, 300, 96, [24, 24])])
def test_q_and_k_in_one_call(device, B, Hq, Hkv, n, D, sections):
    fb = _fb()
    rng = np.random.default_rng(D * n)
    cos, sin = (rng.uniform(-1, 1, (90, D // 2)).astype(np.float32) for _ in range(2))
    rope, axes = fb.RopeCache.from_parts(_T(device, cos), _T(device, sin)), fb.axes_of_sections(sections)
    ids = rng.integers(0, 90, (len(sections), B, n)).astype(np.uint32)
    for dtypes in ((0, 0), (1, 1), (2, 2), (0, 1)):
        q, k = (_as(rng.standard_normal((B, h, n, D)).astype(np.float32), t) for h, t in zip((Hq, Hkv), dtypes))
        for interleaved in (False, True):
            got = rope.forward_axes(_T(device, q, dtypes[0]), _T(device, k, dtypes[1]), _T(device, ids, fb.U32), axes, interleaved)
            for g, x, t in zip(got, (q, k), dtypes):
                assert np.array_equal(g.as_slice(), _as(_turn(x, cos, sin, ids, axes, interleaved), t))
    with pytest.raises(AssertionError):
        rope.forward_axes(_T(device, q), _T(device, np.zeros((B, Hkv, n + 1, D), np.float32)), _T(device, ids, fb.U32), axes)


def test_strided_views(device):
    """Heads behind tokens in memory, rows that start one element off, positions cut out of longer ones; nothing else is written."""
    import torch
    fb = _fb()
    gen = torch.Generator().manual_seed(8)
    B, H, n, D, rows = 2, 3, 17, 64, 50
    cos, sin = (torch.rand((rows, D // 2), generator=gen).cuda() for _ in range(2))
    axes = fb.axes_of_sections([10, 22])
    ids = torch.randint(0, rows, (2, B, 40), generator=gen).to(torch.int32).cuda()
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        for off in (0, 1, 8):
            wide = torch.randn((B, n, H, D + 16), generator=gen).to(dt).cuda()
            x = wide[..., off:off + D].transpose(1, 2)
            out = torch.full((B, H, n, D + 16), 7.0, device="cuda", dtype=dt)
            view = out[..., off:off + D]
            torch.cuda.synchronize()
            co, x4, o4 = [fb.Tensor.from_torch(device, t) for t in (cos, sin)], fb.Tensor.from_torch(device, x), fb.Tensor.from_torch(device, view)
            import ctypes
            from floneum_b200.rope import _positions
            pos = _positions(fb.Tensor.from_torch(device, ids[:, :, 5:5 + n]), axes, B, n, D)
            cx, c_o = x4._c4(), o4._c4()
            L = fb._lib.load()
            fb._lib.check(L.fusor_cuda_rope_axes(device.handle, ctypes.byref(cx), co[0].ptr, co[1].ptr, rows, ctypes.byref(pos), 0, ctypes.byref(c_o)),
                          device.handle)
            device.synchronize()
            want = _turn(x.float().cpu().numpy(), cos.cpu().numpy(), sin.cpu().numpy(), ids[:, :, 5:5 + n].cpu().numpy(), axes, False)
            assert torch.equal(view.cpu(), torch.tensor(want).to(dt))
            assert (out[..., :off] == 7).all() and (out[..., off + D:] == 7).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("pages", ["bf16", "i8"])
@pytest.mark.parametrize("B,Hq,Hkv,D,steps", [(1, 1, 1, 64, [1, 1]), (2, 14, 2, 64, [19, 1, 30]), (3, 8, 8, 128, [16, 33]), (1, 32, 4, 128, [300]), (40, 4, 2, 128, [3, 14])])
def test_rope_axes_append(device, B, Hq, Hkv, D, steps, pages, interleaved):
    fb = _fb()
    rng = np.random.default_rng(D + Hq)
    keep = held if pages == "i8" else O.bf16_round
    rows, n_all = 90, sum(steps)
    cos, sin = (rng.uniform(-1, 1, (rows, D // 2)).astype(np.float32) for _ in range(2))
    rope = fb.RopeCache.from_parts(_T(device, cos), _T(device, sin))
    axes = fb.axes_of_sections([D // 8, D // 2 - D // 8 - 5, 5])
    for dtype in (0, 1, 2):
        per_seq = (n_all + 15) // 16
        cache = fb.PagedKvCache(device, B, Hkv, D, B * per_seq, per_seq, dtype=fb.I8 if pages == "i8" else fb.BF16)
        wk, wv = [], []
        for n in steps:
            q, k, v = (_as(rng.standard_normal((B, h, n, D)).astype(np.float32), dtype) for h in (Hq, Hkv, Hkv))
            ids = rng.integers(0, rows, (3, B, n)).astype(np.uint32)
            got = rope.forward_append(*(_T(device, x, dtype) for x in (q, k, v)), cache, interleaved=interleaved, positions=_T(device, ids, fb.U32), axes=axes)
            assert np.array_equal(got.as_slice(), _as(_turn(q, cos, sin, ids, axes, interleaved), dtype))
            wk.append(keep(_turn(k, cos, sin, ids, axes, interleaved)))
            wv.append(keep(v))
        gk, gv = cache.gather(B, n_all)
        assert np.array_equal(gk.as_slice(), np.concatenate(wk, 2)) and np.array_equal(gv.as_slice(), np.concatenate(wv, 2))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_rope_append_to_8_bit_pages(device, D, interleaved):
    """The one-axis form: from a given row of the tables on, and from each sequence's own length, evicted rows aside."""
    fb = _fb()
    rng = np.random.default_rng(D)
    B, Hq, Hkv = 2, 6, 2
    rope = fb.RopeCache.new(D, 128, 10000.0, device)
    cos, sin = rope.cos.as_slice(), rope.sin.as_slice()
    for dtype in (0, 1, 2):
        cache, wk, wv = fb.PagedKvCache(device, B, Hkv, D, 16, 8, dtype=fb.I8), [], []
        for n, start in ((37, 50), (1, -1), (20, -1)):
            q, k, v = (_as(rng.standard_normal((B, h, n, D)).astype(np.float32), dtype) for h in (Hq, Hkv, Hkv))
            at = start if start >= 0 else cache.seq_len(0)
            got = rope.forward_append(*(_T(device, x, dtype) for x in (q, k, v)), cache, start, interleaved)
            assert np.array_equal(got.as_slice(), _as(O.rope(q, cos, sin, at, interleaved), dtype))
            wk.append(held(O.rope(k, cos, sin, at, interleaved)))
            wv.append(held(v))
            if n == 1:  # both sequences lose eleven rows at the front: positions count from the length that is left
                for b in range(B):
                    cache.drop_front(b, 27)
        gk, gv = cache.gather(B, 47)
        assert np.array_equal(gk.as_slice(), np.concatenate(wk, 2)[:, :, 11:]) and np.array_equal(gv.as_slice(), np.concatenate(wv, 2)[:, :, 11:])


def test_a_window_that_a_prompt_overruns(device):
    """More tokens than the window holds: all of q is rotated, the newest rows stay."""
    fb = _fb()
    rng = np.random.default_rng(5)
    B, Hq, Hkv, n, D, w = 2, 4, 2, 50, 64, 20
    rope = fb.RopeCache.new(D, 64, 10000.0, device)
    cos, sin = rope.cos.as_slice(), rope.sin.as_slice()
    axes, ids = fb.axes_of_sections([16, 16]), rng.integers(0, 64, (2, B, n)).astype(np.uint32)
    for dtype in (fb.I8, fb.BF16):
        cache = fb.KvCache.new(2, w, dtype)
        q, k, v = (rng.standard_normal((B, h, n, D)).astype(np.float32) for h in (Hq, Hkv, Hkv))
        got, ck, cv = rope.forward_append(*(_T(device, x) for x in (q, k, v)), cache, positions=_T(device, ids, fb.U32), axes=axes)
        keep = held if dtype == fb.I8 else O.bf16_round
        assert np.array_equal(got.as_slice(), _turn(q, cos, sin, ids, axes, False))
        assert np.array_equal(ck.as_slice(), keep(_turn(k, cos, sin, ids, axes, False)[:, :, -w:])) and np.array_equal(cv.as_slice(), keep(v[:, :, -w:]))


@pytest.mark.parametrize("D,off", [(128, 0), (80, 0), (64, 1), (6, 0)])
def test_a_tensor_rotated_where_it_lies(device, D, off):
    import ctypes
    import torch
    fb = _fb()
    from floneum_b200.rope import _positions
    rng = np.random.default_rng(D + off)
    cos, sin = (rng.uniform(-1, 1, (40, D // 2)).astype(np.float32) for _ in range(2))
    tc, ts = _T(device, cos), _T(device, sin)
    ids, axes = rng.integers(0, 40, (2, 2, 21)).astype(np.uint32), fb.axes_of_sections([D // 4, D // 2 - D // 4])
    for interleaved in (0, 1):
        wide = torch.tensor(rng.standard_normal((2, 3, 21, D + 8)).astype(np.float32)).cuda()
        x = wide[..., off:off + D]
        before = x.cpu().numpy().copy()
        torch.cuda.synchronize()
        tid = _T(device, ids, fb.U32)
        pos, cx = _positions(tid, axes, 2, 21, D), fb.Tensor.from_torch(device, x)._c4()
        fb._lib.check(fb._lib.load().fusor_cuda_rope_axes(device.handle, ctypes.byref(cx), tc.ptr, ts.ptr, 40, ctypes.byref(pos), interleaved,
                                                          ctypes.byref(cx)), device.handle)
        device.synchronize()
        assert np.array_equal(x.cpu().numpy(), _turn(before, cos, sin, ids, axes, interleaved))


def test_a_position_outside_the_tables_is_reported(device):
    """Read as row 0 and reported at the next wait; the context stays usable."""
    fb = _fb()
    rng = np.random.default_rng(6)
    rope = fb.RopeCache.new(64, 32, 10000.0, device)
    x = rng.standard_normal((1, 2, 4, 64)).astype(np.float32)
    for bad in (32, 2 ** 31, 2 ** 32 - 1):
        ids = np.array([[1, 2, 3, 4], [5, bad, 7, 8]], np.uint32)
        out = fb.rope_axes(_T(device, x), rope.cos, rope.sin, _T(device, ids, fb.U32), fb.axes_of_sections([16, 16]))
        with pytest.raises(fb.FusorCudaError, match="rope position"):
            device.synchronize()
        ids[1, 1] = 0
        assert np.array_equal(out.as_slice(), _turn(x, rope.cos.as_slice(), rope.sin.as_slice(), ids[:, None], fb.axes_of_sections([16, 16]), False))
    device.synchronize()


def test_a_captured_rotation_reads_new_positions(device):
    import torch
    fb = _fb()
    rng = np.random.default_rng(16)
    stream = torch.cuda.Stream()
    dev = fb.Device.gpu(0, stream.cuda_stream)
    x = rng.standard_normal((2, 3, 10, 80)).astype(np.float32)
    cos, sin = (rng.uniform(-1, 1, (30, 40)).astype(np.float32) for _ in range(2))
    tx, tc, ts = (fb.Tensor.from_torch(dev, torch.tensor(a).cuda()) for a in (x, cos, sin))
    ids = torch.zeros((2, 2, 10), dtype=torch.int32, device="cuda")
    axes = fb.axes_of_sections([20, 20])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
        out = fb.rope_axes(tx, tc, ts, fb.Tensor.from_torch(dev, ids), axes)
    for _ in range(2):
        host = rng.integers(0, 30, (2, 2, 10))
        ids.copy_(torch.tensor(host, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out.as_slice(), _turn(x, cos, sin, host, axes, False))
    del graph


def test_refusals(device):
    import ctypes
    fb = _fb()
    L = fb._lib.load()
    UN, IN = fb._lib.UNSUPPORTED, fb._lib.INVALID_ARGUMENT
    rope = fb.RopeCache.new(64, 32, 10000.0, device)
    x = _T(device, np.zeros((1, 2, 4, 64), np.float32))
    ids = _T(device, np.zeros((2, 4), np.uint32), fb.U32)
    axes = np.zeros(32, np.uint8)

    def rc(**kw):
        p = fb._lib.RopePositions()
        p.ids, p.axis_stride, p.batch_stride, p.n_axes, p.axis_of_pair = ids.ptr, 4, 0, 2, axes.tobytes()
        for k, v in kw.items():
            setattr(p, k, v)
        cx, co = x._c4(), x._c4()
        return L.fusor_cuda_rope_axes(device.handle, ctypes.byref(cx), rope.cos.ptr, rope.sin.ptr, 32, ctypes.byref(p), 0, ctypes.byref(co))

    assert rc() == 0
    assert rc(ids=None) == IN and rc(axis_of_pair=None) == IN and rc(n_axes=0) == IN and rc(axis_stride=-4) == IN and rc(batch_stride=-1) == IN
    assert rc(ids=ids.ptr + 2) == UN
    axes[31] = 2
    assert rc() == IN
    with pytest.raises(fb.FusorCudaError):  # more pairs than the call carries
        fb.rope_axes(_T(device, np.zeros((1, 1, 1, 514), np.float32)), _T(device, np.zeros((4, 257), np.float32)), _T(device, np.zeros((4, 257), np.float32)),
                     _T(device, np.zeros((1, 1), np.uint32), fb.U32), np.zeros(257, np.uint8))
    cache = fb.PagedKvCache(device, 1, 2, 64, 4, 4, dtype=fb.I8)
    for kw in (dict(positions=ids), dict(axes=axes)):
        with pytest.raises(AssertionError):
            rope.forward_append(x, x, x, cache, **kw)
    with pytest.raises(fb.FusorCudaError):  # q and k_new differ in tokens
        rope.forward_append(_T(device, np.zeros((1, 2, 3, 64), np.float32)), x, x, cache, positions=_T(device, np.zeros((2, 3), np.uint32), fb.U32),
                            axes=np.zeros(32, np.uint8))
    assert cache.seq_len(0) == 0
    device.synchronize()


def test_a_refused_append_leaves_a_full_window_as_it_was(device):
    """Positions that do not fit are refused before the oldest rows give way to the new ones."""
    fb = _fb()
    rng = np.random.default_rng(8)
    rope, axes = fb.RopeCache.new(64, 64, 10000.0, device), fb.axes_of_sections([16, 16])
    x = lambda n, h=2: _T(device, rng.standard_normal((1, h, n, 64)).astype(np.float32))
    ids = lambda n, a=2: _T(device, np.zeros((a, n), np.uint32), fb.U32)
    cache = fb.KvCache(2, 20, dtype=fb.I8)
    cache.append(device, x(20), x(20))
    before = [t.copy() for t in (lambda s: (s["k"], s["v"]))(cache.export_session())]
    for kw in (dict(positions=ids(4), axes=axes), dict(positions=ids(3), axes=axes[:-1]), dict(positions=ids(3)), dict(axes=axes)):
        with pytest.raises(AssertionError):
            rope.forward_append(x(3, 4), x(3), x(3), cache, **kw)
    with pytest.raises(AssertionError):
        rope.forward_append(x(2, 4), x(3), x(3), cache, positions=ids(3), axes=axes)
    after = cache.export_session()
    assert all(np.array_equal(a, after[name]) for a, name in zip(before, ("k", "v")))
