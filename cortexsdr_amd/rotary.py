"""Rotary positions beside the cache's own (adjacent pairs over a whole head at theta's frequencies,
apply_rope_inplace, api/cortex_sdk.cpp:1363-1423): halves, the first dims of a head, frequencies scaled
for long contexts. csdr_rotary of include/cortexsdr_hip.h, before an append without rotation:

    rot = Rotary(head_dim, theta=5e5, layout="halves", scaling="parts", factor=8.0, original=8192)
    q, k = rot.apply(q, positions, k=k)
    batch.append(None, k, v)          # paged.PagedBatch: keys as they are
    out = batch.attend(q)
"""
from __future__ import annotations

import math

from . import _lib
from .hsdr import _check, _torch
from .paged import _dtype, _empty, _int, _on_device, _stream_of

LAYOUTS = {"adjacent": 0, "halves": 1}
SCALINGS = ("none", "linear", "base", "parts")


def frequencies(dims: int, theta: float = 1e6, scaling: str = "none", factor: float = 1.0,
                original: int = 0, low: float = 1.0, high: float = 4.0) -> list:
    """Radians per position of the dims / 2 pairs, theta ** (-2 j / dims), scaled by
    "linear" (all divided by factor), "base" (theta times factor ** (dims / (dims - 2)): the slowest
    divided by factor, the fastest kept) or "parts" (by the turns of a pair over `original`
    positions: kept from `high` turns up, divided by factor up to `low`, between by a share that
    grows with the turns)."""
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}")
    if dims < 2 or dims % 2:
        raise ValueError("dims must be even and positive")
    if not (0 < theta < math.inf and 0 < factor < math.inf):
        raise ValueError("theta and factor must be positive and finite")
    if scaling == "base":
        if dims == 2:
            raise ValueError("scaling 'base' needs more than one pair")
        theta = theta * factor ** (dims / (dims - 2))
    f = [theta ** (-2.0 * j / dims) for j in range(dims // 2)]
    if scaling == "linear":
        return [w / factor for w in f]
    if scaling == "parts":
        if original <= 0 or not 0 <= low < high:
            raise ValueError("scaling 'parts' needs original positions and low < high turns")
        keep = [min(max((original * w / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for w in f]
        return [w * (s + (1 - s) / factor) for w, s in zip(f, keep)]
    return f


class Rotary:
    """The rotation of heads of head_dim: of their first `dims` dims (0: all), as "adjacent" pairs
    (2 j, 2 j + 1) or "halves" (j, j + dims / 2). The frequencies are those of frequencies(), or
    given: dims / 2 numbers, radians per position. Sine and cosine are multiplied by magnitude."""

    def __init__(self, head_dim: int, theta: float = 1e6, dims: int = 0, layout: str = "adjacent",
                 scaling: str = "none", factor: float = 1.0, original: int = 0, low: float = 1.0,
                 high: float = 4.0, magnitude: float = 1.0, freqs=None):
        torch = _torch()
        dims = dims or head_dim
        if layout not in LAYOUTS:
            raise ValueError("layout must be 'adjacent' or 'halves'")
        if not 0 < head_dim <= 1024 or not 0 < dims <= head_dim or dims % 2:
            raise ValueError("dims must be even and up to head_dim, head_dim up to 1024")
        if freqs is None:
            freqs = frequencies(dims, theta, scaling, factor, original, low, high)
        freqs = [float(f) for f in freqs]
        if len(freqs) != dims // 2 or not all(math.isfinite(f) for f in freqs):
            raise ValueError("freqs must be dims / 2 finite numbers")
        self.head_dim, self.dims, self.magnitude = int(head_dim), int(dims), float(magnitude)
        self._layout = LAYOUTS[layout]
        self._turns = torch.tensor([f / (2 * math.pi) for f in freqs], dtype=torch.float64,
                                   device="cuda")

    def _side(self, torch, what, x, out, n, stream):
        """Heads and strides of x and of its output, which is made if there is none."""
        hd = self.head_dim
        strides = []
        for name, t in ((what, x), (what + "_out", out)):
            if t is None:
                t = out = _empty(torch, tuple(x.shape), x.dtype, x.device, stream)
            if t.dim() != 3 or t.shape[2] != hd or t.stride(2) != 1 or \
                    (t.shape[1] > 1 and t.stride(1) != hd) or t.shape[1] < 1:
                raise ValueError(f"{name} must be (tokens, heads, {hd}) with a token's values side "
                                 "by side")
            if t.shape[0] != n or t.dtype != x.dtype or t.shape[1] != x.shape[1]:
                raise ValueError(f"{name}: other tokens, heads or type")
            if n > 1 and t.stride(0) < t.shape[1] * hd:
                raise ValueError(f"{name}: its tokens overlap")
            strides.append(t.stride(0) if n > 1 else 0)
        return out, x.shape[1], strides[0], strides[1]

    def apply(self, q, positions, k=None, q_out=None, k_out=None, stream=None):
        """q and k (tokens, heads, head_dim), float32 or float16 with tokens any stride apart, turned
        at positions, (tokens,) int32; returns q, or q and k where k is given. q_out may be q
        (in place). A token with a negative position is none: its rows are not written."""
        torch = _torch()
        dt, n = _dtype(q), q.shape[0]
        if positions.dtype != torch.int32 or tuple(positions.shape) != (n,) or \
                not positions.is_contiguous():
            raise ValueError("positions must be a contiguous int32 tensor, one per token")
        q_out, hq, qs, qos = self._side(torch, "q", q, q_out, n, stream)
        hk = ks = kos = 0
        if k is not None:
            if k.dtype != q.dtype:
                raise ValueError("q and k must have the same type")
            k_out, hk, ks, kos = self._side(torch, "k", k, k_out, n, stream)
        elif k_out is not None:
            raise ValueError("k_out without k")
        dev = _on_device(torch, "tensors", q, k, q_out, k_out, positions, self._turns)
        if n:
            _check(_lib.load().csdr_rotary(
                q.data_ptr(), q_out.data_ptr(), _int(hq), qs, qos,
                k.data_ptr() if k is not None else None,
                k_out.data_ptr() if k is not None else None, _int(hk), ks, kos, dt, _int(n), self.head_dim,
                self.dims, self._layout, positions.data_ptr(), self._turns.data_ptr(),
                self.magnitude, _stream_of(torch, dev, stream)))
        return q_out if k is None else (q_out, k_out)
