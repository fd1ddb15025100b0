"""Positions and tables that the launch just before a rotation wrote on the same stream, with nothing waited for between."""
import numpy as np
import pytest

from cache8_oracle import held
from oracle import oracle as O

pytestmark = pytest.mark.gpu


def _fb():
    import floneum_b200 as fb
    return fb


def _turn(x, cos, sin, ids, axes):
    half = x.shape[-1] // 2
    row = ids[np.asarray(axes)].transpose(1, 2, 0)
    c, s = (t[row, np.arange(half)][:, None] for t in (cos, sin))
    a, b = x[..., :half], x[..., half:]
    return np.concatenate([a * c - b * s, a * s + b * c], -1)


class _Steps:
    """`steps` single steps of a decoder: positions advanced (and the tables replaced) on the device by the launch before each rotation."""

    def __init__(self, B, n, D, dtype, steps, alternating):
        import torch
        fb = _fb()
        self.stream = torch.cuda.Stream()
        self.dev = fb.Device.gpu(0, self.stream.cuda_stream)
        rng = np.random.default_rng(n + D)
        self.n, self.rows, self.steps = n, 64, steps
        self.axes = (np.arange(D // 2) % 3).astype(np.uint8) if alternating else fb.axes_of_sections([D // 8, D // 8, D // 2 - 2 * (D // 8)])
        self.cos, self.sin = (rng.uniform(-1, 1, (steps, self.rows, D // 2)).astype(np.float32) for _ in range(2))
        self.ids = rng.integers(0, self.rows, (steps, 3, B, n))
        self.x = [rng.standard_normal((B, h, n, D)).astype(np.float32) for h in (4, 2, 2)]
        if dtype == 1:
            self.x = [O.bf16_round(x) for x in self.x]
        tt = torch.bfloat16 if dtype == 1 else torch.float32
        self.src = [torch.tensor(a).cuda() for a in (self.cos, self.sin)] + [torch.tensor(self.ids, dtype=torch.int32).cuda()]
        self.now = [torch.zeros_like(t[0]) for t in self.src]
        self.qkv = [torch.tensor(x).to(tt).cuda() for x in self.x]
        torch.cuda.synchronize()
        T = lambda t: fb.Tensor.from_torch(self.dev, t)
        self.rope, self.pos, self.t = fb.RopeCache.from_parts(T(self.now[0]), T(self.now[1])), T(self.now[2]), [T(t) for t in self.qkv]
        self.dtype = dtype

    def write(self, i):
        for to, src in zip(self.now, self.src):
            to.copy_(src[i])

    def want(self, i, which):
        y = _turn(self.x[which], self.cos[i], self.sin[i], self.ids[i], self.axes)
        return O.bf16_round(y) if self.dtype == 1 else y


@pytest.mark.parametrize("alternating", [False, True])
@pytest.mark.parametrize("B,n,D,dtype", [(2, 1, 64, 0), (1, 5, 128, 1), (3, 300, 128, 0), (2, 7, 80, 1)])
def test_rotations_of_q_and_k(B, n, D, dtype, alternating):
    import torch
    S = _Steps(B, n, D, dtype, 40, alternating)
    outs = []
    with torch.cuda.stream(S.stream):
        for i in range(S.steps):
            S.write(i)
            outs.append(S.rope.forward_axes(S.t[0], S.t[1], S.pos, S.axes))
    for i, out in enumerate(outs):
        for which in range(2):
            assert np.array_equal(out[which].as_slice(), S.want(i, which)), i


@pytest.mark.parametrize("pages", ["bf16", "i8"])
@pytest.mark.parametrize("alternating", [False, True])
@pytest.mark.parametrize("B,n,D,dtype", [(2, 1, 64, 0), (40, 1, 128, 1), (1, 60, 128, 0)])
def test_rotations_with_the_append(B, n, D, dtype, alternating, pages):
    import torch
    fb = _fb()
    S = _Steps(B, n, D, dtype, 24, alternating)
    most = (S.steps * n + 15) // 16
    cache, outs = fb.PagedKvCache(S.dev, B, 2, D, B * most, most, dtype=fb.I8 if pages == "i8" else fb.BF16), []
    with torch.cuda.stream(S.stream):
        for i in range(S.steps):
            S.write(i)
            outs.append(S.rope.forward_append(S.t[0], S.t[1], S.t[2], cache, positions=S.pos, axes=S.axes))
    for i, out in enumerate(outs):
        assert np.array_equal(out.as_slice(), S.want(i, 0)), i
    keep = held if pages == "i8" else O.bf16_round
    got = cache.gather(B, S.steps * n)[0].as_slice()
    turned = [_turn(S.x[1], S.cos[i], S.sin[i], S.ids[i], S.axes) for i in range(S.steps)]
    assert np.array_equal(got, keep(np.concatenate(turned, 2)))


def test_one_axis_with_tables_just_written():
    """The one-axis rotation with the append to 8-bit pages, its tables replaced before every step."""
    import torch
    fb = _fb()
    S = _Steps(2, 3, 128, 0, 24, False)
    cache, outs = fb.PagedKvCache(S.dev, 2, 2, 128, 2 * 5, 5, dtype=fb.I8), []
    with torch.cuda.stream(S.stream):
        for i in range(S.steps):
            S.write(i)
            outs.append(S.rope.forward_append(S.t[0], S.t[1], S.t[2], cache, start_pos=i))
    for i, out in enumerate(outs):
        assert np.array_equal(out.as_slice(), O.rope(S.x[0], S.cos[i], S.sin[i], i, False)), i
    want = np.concatenate([held(O.rope(S.x[1], S.cos[i], S.sin[i], i, False)) for i in range(S.steps)], 2)
    assert np.array_equal(cache.gather(2, 72)[0].as_slice(), want)


def test_a_captured_run_of_steps():
    """Positions advanced by a kernel inside the graph, right before each rotation."""
    import torch
    fb = _fb()
    S = _Steps(2, 2, 64, 0, 12, True)
    graph, outs = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph, stream=S.stream, capture_error_mode="relaxed"):
        for i in range(S.steps):
            S.write(i)
            outs.append(S.rope.forward_axes(S.t[0], S.t[1], S.pos, S.axes))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for i, out in enumerate(outs):
            for which in range(2):
                assert np.array_equal(out[which].as_slice(), S.want(i, which)), i
    del graph
