"""Rotary position embedding behind fusor's names: `RopeCache` and the `Tensor` rope ops.

Reference: fusor-ml/fusor/src/composite/rope.rs — `Tensor::rope` (:38-68), `rope_interleaved` (:70-118),
`RopeCache::new / from_parts / forward / forward_interleaved` (:186-265) — and the llama call site
models/kalosm-llama/src/raw/rope.rs:86-111.  `RopeCache.forward_append` is the fused form of
"rope(q, k) then KvCache.append(k, v)": one kernel rotates q, rotates k into the bf16 pages and copies v there.
All arithmetic runs in libfusor_cuda.so.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple

import numpy as np

from . import _lib
from .device import Device
from .tensor import F32, U32, Tensor


def base_inverse_frequency(dim: int, rope_theta: float) -> np.ndarray:
    """`1 / theta^(i/dim)` for i = 0, 2, .. dim-2 in f32 (rope.rs:189-194)."""
    theta = np.float32(rope_theta)
    return np.array([np.float32(1.0) / theta ** (np.float32(i) / np.float32(dim)) for i in range(0, dim, 2)],
                    dtype=np.float32)


def _check_tables(cos: Tensor, sin: Tensor, head_dim: int):
    cs, ss = cos.shape(), sin.shape()
    assert tuple(cs) == tuple(ss) and len(cs) == 2 and cs[1] == head_dim // 2, (
        f"cos/sin shape {list(cs)} / {list(ss)} does not match [context, {head_dim // 2}]")
    assert cos.dtype == F32 and sin.dtype == F32 and cos.is_contiguous() and sin.is_contiguous()


def rope(x: Tensor, cos: Tensor, sin: Tensor, start_pos: int = 0, interleaved: bool = False,
         out_dtype: int | None = None) -> Tensor:
    """x [B,H,n,D] rotated with rows start_pos .. start_pos+n of cos/sin [context, D/2] (f32 device tensors)."""
    shape = x.shape()
    assert len(shape) == 4, "rope expects [batch, heads, sequence, head_dim]"
    assert shape[3] % 2 == 0, "head_dim must be even"
    _check_tables(cos, sin, shape[3])
    cs = cos.shape()
    dev = x.device
    out = Tensor.empty(dev, shape, x.dtype if out_dtype is None else out_dtype)
    cx, co = x._c4(), out._c4()
    _lib.check(_lib.load().fusor_cuda_rope(dev.handle, ctypes.byref(cx), cos.ptr, sin.ptr, cs[0], int(start_pos),
                                           int(bool(interleaved)), ctypes.byref(co)), dev.handle)
    return out


def axes_of_sections(sections: Sequence[int], alternating: bool = False) -> np.ndarray:
    """The axis of each pair (uint8 [head_dim / 2]) from the number of pairs of each axis.

    In order: the first sections[0] pairs are axis 0, the next sections[1] axis 1 and so on.  `alternating`: pair i is axis
    i % len(sections) while that axis has pairs left, else axis 0."""
    counts = [int(n) for n in sections]
    assert counts and min(counts) >= 0 and len(counts) <= 256, f"sections {counts} must be 1 to 256 counts of pairs"
    if not alternating:
        return np.repeat(np.arange(len(counts), dtype=np.uint8), counts)
    half, left = sum(counts), list(counts)
    out = np.zeros(half, np.uint8)
    for i in range(half):
        a = i % len(counts)
        out[i] = a if a == 0 or left[a] > 0 else 0
        left[out[i]] -= 1
    assert left[0] == 0, f"sections {counts} cannot alternate: axis 0 would get {counts[0] - left[0]} pairs"
    return out


_BYTE = np.dtype(np.uint8)


def _positions(positions: Tensor, axes, batch: int, n: int, head_dim: int):
    """The C view of positions (u32 [n_axes, n], the same for every sequence, or [n_axes, batch, n])."""
    assert positions.dtype == U32, "positions must be a u32 tensor"
    shape, strides = positions.shape(), positions.strides
    assert len(shape) in (2, 3) and shape[-1] == n and (len(shape) == 2 or shape[1] == batch), (
        f"positions shape {list(shape)} does not match [axes, {batch}, {n}] or [axes, {n}]")
    assert n == 1 or strides[-1] == 1, "the token axis of the positions must be contiguous"
    given = np.asarray(axes)
    assert given.shape == (head_dim // 2,), f"axes must name the axis of each of {head_dim // 2} pairs, got {list(given.shape)}"
    if given.dtype is not _BYTE:  # (bytes travel as they are, and the call looks at them)
        assert given.min() >= 0 and given.max() < min(shape[0], 256) and (given.dtype.kind in "uib" or not (given % 1).any()), (
            f"axes {given.tolist()} must be whole numbers from 0 to {shape[0] - 1}, the axes of the positions")
        given = given.astype(np.uint8)
    p = _lib.RopePositions()
    p.ids, p.axis_stride, p.batch_stride = positions.ptr, strides[0], strides[1] if len(shape) == 3 else 0
    p.n_axes, p.axis_of_pair = shape[0], given.tobytes()  # (the structure keeps the bytes)
    return p


def rope_axes(x: Tensor, cos: Tensor, sin: Tensor, positions: Tensor, axes, interleaved: bool = False,
              out_dtype: Optional[int] = None) -> Tensor:
    """x [B,H,n,D] rotated with several axes: pair i of token t takes row positions[axes[i], (b,) t] of cos / sin [context, D/2].

    positions: u32 [n_axes, n] or [n_axes, B, n]; axes: the axis of each pair (see `axes_of_sections`).  A position outside the
    tables is read as row 0 and raises at the next `Device.synchronize`."""
    shape = x.shape()
    assert len(shape) == 4, "rope expects [batch, heads, sequence, head_dim]"
    assert shape[3] % 2 == 0, "head_dim must be even"
    _check_tables(cos, sin, shape[3])
    pos = _positions(positions, axes, shape[0], shape[2], shape[3])
    dev = x.device
    out = Tensor.empty(dev, shape, x.dtype if out_dtype is None else out_dtype)
    cx, co = x._c4(), out._c4()
    _lib.check(_lib.load().fusor_cuda_rope_axes(dev.handle, ctypes.byref(cx), cos.ptr, sin.ptr, cos.shape()[0], ctypes.byref(pos),
                                                int(bool(interleaved)), ctypes.byref(co)), dev.handle)
    return out


class RopeCache:
    """cos / sin tables [context_length, head_dim/2] on the device (rope.rs:180-265)."""

    def __init__(self, cos: Tensor, sin: Tensor):
        assert tuple(cos.shape()) == tuple(sin.shape()) and len(cos.shape()) == 2
        self.cos, self.sin = cos, sin

    @classmethod
    def new(cls, head_dim: int, context_length: int, rope_theta: float, device: Device) -> "RopeCache":
        inv = base_inverse_frequency(head_dim, rope_theta)
        outer = np.arange(context_length, dtype=np.float32)[:, None] * inv[None, :]
        shape = (context_length, head_dim // 2)
        return cls(Tensor.from_slice(device, shape, np.cos(outer).astype(np.float32)),
                   Tensor.from_slice(device, shape, np.sin(outer).astype(np.float32)))

    @classmethod
    def from_parts(cls, cos: Tensor, sin: Tensor) -> "RopeCache":
        return cls(cos, sin)

    def forward(self, q: Tensor, k: Tensor, start_pos: int) -> Tuple[Tensor, Tensor]:
        return (rope(q, self.cos, self.sin, start_pos, False), rope(k, self.cos, self.sin, start_pos, False))

    def forward_interleaved(self, q: Tensor, k: Tensor, start_pos: int) -> Tuple[Tensor, Tensor]:
        return (rope(q, self.cos, self.sin, start_pos, True), rope(k, self.cos, self.sin, start_pos, True))

    def forward_axes(self, q: Tensor, k: Tensor, positions: Tensor, axes, interleaved: bool = False) -> Tuple[Tensor, Tensor]:
        """`forward` for tokens with a position on each of several axes (time, row, column), in one launch: see `rope_axes`."""
        B, _, n, D = q.shape()
        kB, _, kn, kD = k.shape()
        assert (kB, kn, kD) == (B, n, D), f"q {list(q.shape())} and k {list(k.shape())} differ in batch, tokens or head_dim"
        assert D % 2 == 0, "head_dim must be even"
        _check_tables(self.cos, self.sin, D)
        pos = _positions(positions, axes, B, n, D)
        dev = q.device
        q_out, k_out = Tensor.empty(dev, q.shape(), q.dtype), Tensor.empty(dev, k.shape(), k.dtype)
        cq, ck, cqo, cko = q._c4(), k._c4(), q_out._c4(), k_out._c4()
        _lib.check(_lib.load().fusor_cuda_rope_axes_qk(dev.handle, ctypes.byref(cq), ctypes.byref(ck), self.cos.ptr, self.sin.ptr,
                                                       self.cos.shape()[0], ctypes.byref(pos), int(bool(interleaved)),
                                                       ctypes.byref(cqo), ctypes.byref(cko)), dev.handle)
        return q_out, k_out

    def forward_append(self, q: Tensor, k: Tensor, v: Tensor, cache, start_pos: int = -1, interleaved: bool = False,
                       out_dtype: int | None = None, positions: Optional[Tensor] = None, axes=None):
        """Rotates q, rotates k into `cache` and appends v, in one launch.

        `cache` is a `KvCache` (returns `(q_rotated, cached_k, cached_v)`) or a `PagedKvCache` (returns q_rotated).
        start_pos < 0 positions every sequence at its own cache length.  `positions` with `axes` take its place for tokens
        with a position on each of several axes (see `rope_axes`)."""
        from .cache import KvCache

        if isinstance(cache, KvCache):
            return cache._append_rotated(self, q, k, v, start_pos, interleaved, out_dtype, positions, axes)
        return cache.rope_append(q, k, v, self.cos, self.sin, start_pos, interleaved, out_dtype, positions, axes)
