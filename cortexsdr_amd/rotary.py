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
    given: dims / 2 numbers, radians per position. Sine and cosine are multiplied by magnitude. It may
    be dropped while its calls are queued, on any stream; a captured one needs it until its graph's
    last replay."""

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
        self._at = self._turns.data_ptr()
        # the streams that the table's memory waits for before it is given to another tensor
        self._streams = {_stream_of(torch, self._turns.get_device(), None)}
        self._call = _lib.load().csdr_rotary

    def _stride(self, what: str, x, n: int) -> int:
        """The token stride of (n, heads, head_dim) with a token's values side by side (0: one token)."""
        shape, hd = x.shape, self.head_dim
        if len(shape) == 3 and shape[0] == n and shape[2] == hd and shape[1] > 0:
            s = x.stride()
            if s[2] == 1 and (s[1] == hd or shape[1] == 1):
                if n < 2:
                    return 0
                if s[0] >= shape[1] * hd:
                    return s[0]
                raise ValueError(f"{what}: its tokens overlap")
        raise ValueError(f"{what} must be ({n}, heads, {hd}) with a token's values side by side")

    def _out(self, torch, what, x, out, n, stream):
        """Where x's heads go, and its token stride."""
        if out is None:
            return (x.new_empty(x.shape) if stream is None else
                    _empty(torch, x.shape, x.dtype, x.device, stream)), 0
        if out.dtype != x.dtype or out.shape != x.shape:
            raise ValueError(f"{what}: other tokens, heads or type")
        return out, self._stride(what, out, n)

    def apply(self, q, positions, k=None, q_out=None, k_out=None, stream=None):
        """q and k (tokens, heads, head_dim), float32 or float16 with tokens any stride apart, turned
        at positions, (tokens,) int32; returns q, or q and k where k is given. q_out may be q
        (in place). A token with a negative position is none: its rows are not written."""
        torch = _torch()
        dt, n = _dtype(q), q.shape[0]
        if positions.dtype != torch.int32 or positions.shape != (n,) or \
                not positions.is_contiguous():
            raise ValueError("positions must be a contiguous int32 tensor, one per token")
        qs = self._stride("q", q, n)
        q_out, qos = self._out(torch, "q_out", q, q_out, n, stream)
        hk = ks = kos = 0
        kp = kop = None
        if k is not None:
            if k.dtype != q.dtype:
                raise ValueError("q and k must have the same type")
            ks, hk = self._stride("k", k, n), k.shape[1]
            k_out, kos = self._out(torch, "k_out", k, k_out, n, stream)
            kp, kop = k.data_ptr(), k_out.data_ptr()
        elif k_out is not None:
            raise ValueError("k_out without k")
        dev = _on_device(torch, "tensors", q, k, q_out, k_out, positions, self._turns)
        if n:
            on = _stream_of(torch, dev, stream)
            if on not in self._streams:
                self._turns.record_stream(torch.cuda.current_stream() if stream is None else stream)
                self._streams.add(on)
            rc = self._call(q.data_ptr(), q_out.data_ptr(), _int(q.shape[1]), qs, qos, kp, kop, _int(hk),
                            ks, kos, dt, _int(n), self.head_dim, self.dims, self._layout,
                            positions.data_ptr(), self._at, self.magnitude, on)
            if rc:
                _check(rc)
        return q_out if k is None else (q_out, k_out)
