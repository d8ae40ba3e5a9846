"""A layer in 8 bits: rows of codes with a scale each, from a root-mean-square norm (with the residual's
addition), from values as they are or from silu(gate) * x, and their products on the integer matrix
cores. csdr_q8_* and csdr_add_rms_norm of include/cortexsdr_hip.h, in place of rms_norm, silu_mul
(api/cortex_sdk.cpp:1208-1256) and Kernels::linear_forward (kernels/blas_kernels.cpp:264-293):

    w = quantize(weights)                             # (R, C): a scale per output channel
    n = rms_norm(x, norm_w, 1e-5, residual=stream)    # n.residual = stream + x; n.rows its norm
    y = linear(w, n.rows, dtype="f16")                # (tokens, R)
    d = quantize(y[:, F:], gate=y[:, :F])             # silu(gate) * up for the down projection
    stream = linear(w_down, d, add=n.residual, dtype="f32")

With `stream`, a call runs on that stream, its outputs are allocated there, and the caller orders it
against the streams its tensors come from. A call of no rows does nothing.
"""
from __future__ import annotations

import typing

from . import _lib
from .hsdr import _check, _torch
from .paged import _dtype, _empty, _int, _on_device, _stream_of

PITCH = 128
MAX_WIDTH = (1 << 17) - 1


def _pitch(n: int) -> int:
    if not 0 < n <= MAX_WIDTH:
        raise ValueError("rows must have 1 to 131071 values")
    return (n + PITCH - 1) // PITCH * PITCH


def _rows(what: str, t, n=None) -> int:
    """The row stride of a (rows, n) tensor with a row's values side by side (0: one row)."""
    shape, s = t.shape, t.stride()
    if len(shape) != 2 or (n is not None and shape[1] != n) or (s[1] != 1 and shape[1] > 1):
        raise ValueError(f"{what} must be (rows, {n or 'n'}) with a row's values side by side")
    if shape[0] < 2:
        return 0
    if s[0] < shape[1]:  # an expanded tensor, or rows that overlap
        raise ValueError(f"the rows of {what} overlap")
    return s[0]


def _type(torch, dtype: str):
    if dtype == "f32":
        return torch.float32
    if dtype == "f16":
        return torch.float16
    raise ValueError("dtype must be 'f32' or 'f16'")


class Q8Rows:
    """Rows of n values as codes, (rows, n up to a whole number of 128) int8 with zeros behind the
    last, and scales, (rows,) float32: a value is scale * code."""

    __slots__ = ("codes", "scales", "n", "rows")

    def __init__(self, codes, scales, n: int):
        torch = _torch()
        n = int(n)
        if codes.dtype != torch.int8 or codes.dim() != 2 or codes.shape[1] != _pitch(n) or \
                not codes.is_contiguous():
            raise ValueError(f"codes must be a contiguous int8 tensor (rows, {_pitch(n)})")
        if scales.dtype != torch.float32 or scales.shape != (codes.shape[0],) or \
                not scales.is_contiguous():
            raise ValueError("scales must be a contiguous float32 tensor, one per row")
        _on_device(torch, "codes and scales", codes, scales)
        self.codes, self.scales, self.n, self.rows = codes, scales, n, int(codes.shape[0])

    @classmethod
    def pack(cls, codes, scales) -> "Q8Rows":
        """From (rows, n) int8 codes without a pitch, as other quantisers make them (a copy)."""
        torch = _torch()
        if codes.dtype != torch.int8 or codes.dim() != 2:
            raise ValueError("codes must be an int8 tensor (rows, n)")
        rows, n = codes.shape
        padded = torch.zeros((rows, _pitch(n)), dtype=torch.int8, device=codes.device)
        padded[:, :n] = codes
        return cls(padded, scales, n)

    def values(self, dtype: str = "f32", out=None, stream=None):
        """scale * code, (rows, n) of "f32" or "f16"."""
        torch = _torch()
        dt = _type(torch, dtype)
        if out is None:
            out = _empty(torch, (self.rows, self.n), dt, self.codes.device, stream)
        else:
            _out("out", out, dt, self.rows, self.n)
        dev = _on_device(torch, "tensors", self.codes, self.scales, out)
        if self.rows:
            rc = _lib.load().csdr_q8_dequantize(
                self.codes.data_ptr(), self.scales.data_ptr(), _int(self.rows), self.n, out.data_ptr(),
                int(dtype == "f16"), _stream_of(torch, dev, stream))
            if rc:
                _check(rc)
        return out


def _out(what: str, t, dt, rows, n) -> None:
    if t.dtype != dt or t.shape != (rows, n) or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dt} tensor ({rows}, {n})")


def _new_rows(torch, rows, n, device, stream) -> Q8Rows:
    r = Q8Rows.__new__(Q8Rows)
    r.n, r.rows = n, rows
    if stream is None:
        r.codes = torch.empty((rows, _pitch(n)), dtype=torch.int8, device=device)
        r.scales = torch.empty(rows, dtype=torch.float32, device=device)
    else:
        r.codes = _empty(torch, (rows, _pitch(n)), torch.int8, device, stream)
        r.scales = _empty(torch, (rows,), torch.float32, device, stream)
    return r


def quantize(x, gate=None, stream=None) -> Q8Rows:
    """8-bit rows of x, (rows, n) float32 or float16 with rows any stride apart (a weight matrix: a
    scale per output channel), or of silu(gate) * x. A row with a value that is not finite reads as
    NaN."""
    torch = _torch()
    dt, xs = _dtype(x), _rows("x", x)
    rows, n = x.shape
    gs = 0
    if gate is not None:
        gs = _rows("gate", gate, n)
        if gate.shape[0] != rows or gate.dtype != x.dtype:
            raise ValueError("gate and x must have the same rows and type")
    dev = _on_device(torch, "tensors", x, gate)
    r = _new_rows(torch, rows, n, x.device, stream)
    if rows:
        rc = _lib.load().csdr_q8_quantize(
            x.data_ptr(), gate.data_ptr() if gate is not None else None, dt, _int(rows), n, xs, gs,
            r.codes.data_ptr(), r.scales.data_ptr(), _stream_of(torch, dev, stream))
        if rc:
            _check(rc)
    return r


class Normed(typing.NamedTuple):
    rows: typing.Any      # Q8Rows, None without q8
    y: typing.Any         # (rows, n) of x's type, None unless asked for
    residual: typing.Any  # the stream with x added, (rows, n) of its type, None without one


def rms_norm(x, w, eps: float = 1e-5, residual=None, residual_out=None, q8: bool = True,
             y: bool = False, stream=None) -> Normed:
    """The norm of x (rows, n), or of residual + x as residual's type holds it: h / sqrt(mean(h^2) +
    eps) * w, as 8-bit rows and, with y, as values too. w: (n,) float32. residual_out: where the
    sum goes, residual itself (contiguous) for an update in place; else a new tensor."""
    torch = _torch()
    dt, xs = _dtype(x), _rows("x", x)
    rows, n = x.shape
    if w.dtype != torch.float32 or w.shape != (n,) or not w.is_contiguous():
        raise ValueError("w must be a contiguous float32 tensor, one per column")
    if not (q8 or y):
        raise ValueError("ask for q8, y or both")
    rs = rdt = 0
    if residual is not None:
        rs, rdt = _rows("residual", residual, n), _dtype(residual)
        if residual.shape[0] != rows:
            raise ValueError("residual and x must have the same rows")
        if residual_out is None:
            residual_out = _empty(torch, (rows, n), residual.dtype, x.device, stream)
        else:
            _out("residual_out", residual_out, residual.dtype, rows, n)
    elif residual_out is not None:
        raise ValueError("residual_out without residual")
    dev = _on_device(torch, "tensors", x, w, residual, residual_out)
    r = _new_rows(torch, rows, n, x.device, stream) if q8 else None
    yt = _empty(torch, (rows, n), x.dtype, x.device, stream) if y else None
    if rows:
        rc = _lib.load().csdr_add_rms_norm(
            x.data_ptr(), dt, xs, residual.data_ptr() if residual is not None else None, rdt, rs,
            residual_out.data_ptr() if residual is not None else None, w.data_ptr(), eps, _int(rows),
            _int(n), yt.data_ptr() if y else None, r.codes.data_ptr() if q8 else None,
            r.scales.data_ptr() if q8 else None, _stream_of(torch, dev, stream))
        if rc:
            _check(rc)
    return Normed(r, yt, residual_out)


def linear(w: Q8Rows, x: Q8Rows, bias=None, add=None, dtype: str = "f32", out=None, stream=None):
    """(x.rows, w.rows) = x . w^T of "f32" or "f16", plus bias, (w.rows,) float32, and add, (x.rows,
    w.rows) of the output's type (a residual; it may be out itself). out: rows any stride apart."""
    torch = _torch()
    M, R, n = x.rows, w.rows, x.n
    dt = _type(torch, dtype)
    if w.n != n:
        raise ValueError(f"w has rows of {w.n} values, x of {n}")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (R,) or
                             not bias.is_contiguous()):
        raise ValueError("bias must be a contiguous float32 tensor, one per row of w")
    ads = 0
    if add is not None:
        ads = _rows("add", add, R)
        if add.shape[0] != M or add.dtype != dt:
            raise ValueError("add must have x's rows and the output's type")
    if out is None:
        out, os = _empty(torch, (M, R), dt, x.codes.device, stream), 0
    else:
        os = _rows("out", out, R)
        if out.shape[0] != M or out.dtype != dt:
            raise ValueError(f"out must be ({M}, {R}) of {dtype}")
    dev = _on_device(torch, "tensors", w.codes, w.scales, x.codes, x.scales, bias, add, out)
    if M and R:
        rc = _lib.load().csdr_q8_linear(
            w.codes.data_ptr(), w.scales.data_ptr(), _int(R), x.codes.data_ptr(), x.scales.data_ptr(),
            _int(M), n,
            bias.data_ptr() if bias is not None else None,
            add.data_ptr() if add is not None else None, ads, out.data_ptr(), int(dtype == "f16"),
            os, _stream_of(torch, dev, stream))
        if rc:
            _check(rc)
    return out
