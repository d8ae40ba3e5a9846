"""Serving from a paged K/V cache: sequences of different lengths over shared pools of pages.

The cached attention that kernels/flash_attention.cpp:165-247 of the reference intends, in place
of its whole-context recompute (run_transformer_decode, api/cortex_sdk.cpp:1543-1696), for steps
and prompts of many sequences at once. csdr_paged_* of include/cortexsdr_hip.h: PagedCache holds
the pools, PagedBatch the sequences of a step (their page table and lengths, device tensors that
the caller's scheduler fills and may change between calls):

    cache = PagedCache(n_pages, 64, n_kv_heads, head_dim, "q4")
    batch = cache.batch(table, lens)          # int32: (n, pages per sequence), (n,)
    q = batch.append(q, k, v, theta=1e6)      # rotated queries; keys and values into the pages
    out = batch.attend(q)

With `stream`, a call runs on that stream, its outputs and workspace are allocated there, and the
caller orders it against the streams its tensors come from. Workspaces are allocated per call
(inside a graph capture, from that graph's pool), so calls on different streams and captured graphs
share none unless the caller passes one to both. A call of no tokens does nothing.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from .hsdr import _check, _torch

KV_DTYPES = {"f16": 1, "q4": 2}
_DTYPES = {}


def _dtype(t) -> int:
    if not _DTYPES:
        torch = _torch()
        _DTYPES.update({torch.float32: 0, torch.float16: 1})
    dt = _DTYPES.get(t.dtype)
    if dt is None:
        raise ValueError("tensors must be float32 or float16")
    return dt


_raw = None  # torch's raw accessor of a device's current stream, where it has one


def _on_device(torch, what: str, *ts) -> int:
    """Checks that the tensors are on the current device; its index."""
    dev = torch.cuda.current_device()
    for t in ts:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{what} must be on the current device")
    return dev


def _stream_on(stream, dev: int) -> None:
    if stream.device_index != dev:
        raise ValueError("stream must be one of the current device")


def _stream_of(torch, dev: int, stream) -> int:
    """The hipStream_t of `stream`, or of the device's current stream."""
    global _raw
    if stream is None:
        if _raw is None:
            _raw = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
                (lambda d: int(torch.cuda.current_stream(d).cuda_stream))
        return _raw(dev)
    _stream_on(stream, dev)
    return int(stream.cuda_stream)


def _empty(torch, shape, dtype, device, stream):
    """A tensor of the stream that will write it (the current one if None)."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    _stream_on(stream, torch.cuda.current_device())
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


_INT_MAX = 2 ** 31 - 1


def _int(v) -> int:
    """v as a C int holds it: past its ends the largest, or -1 (which the library refuses)."""
    return v if 0 <= v <= _INT_MAX else -1 if v < 0 else _INT_MAX


def _bytes(workspace) -> int:
    """What a caller's workspace holds: all of it has to be there (an expanded tensor's is not)."""
    if not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    return workspace.nbytes


def _ints(torch, what: str, t, shape) -> None:
    if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 tensor of shape {shape}")


class PagedCache:
    """Pools of n_pages K and V pages (page_size positions of every KV head each), in "f16" or
    "q4". k, v: existing pools as uint8 tensors of n_pages * page_bytes, else new ones."""

    def __init__(self, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int,
                 kv_dtype: str = "f16", k=None, v=None):
        torch = _torch()
        if kv_dtype not in KV_DTYPES:
            raise ValueError("kv_dtype must be 'f16' or 'q4'")
        self.page_bytes = int(_lib.load().csdr_paged_page_bytes(
            KV_DTYPES[kv_dtype], _int(page_size), _int(n_kv_heads), _int(head_dim)))
        if not self.page_bytes or not 0 < n_pages <= _INT_MAX:
            raise ValueError("page_size must be a power of two from 16 to 4096, head_dim 64 or "
                             "128, the numbers of pages and heads positive")
        self.n_pages, self.page_size = int(n_pages), int(page_size)
        self.n_kv_heads, self.head_dim, self.kv_dtype = int(n_kv_heads), int(head_dim), kv_dtype
        if (k is None) != (v is None):
            raise ValueError("give both pools or none")
        if k is None:
            k = torch.zeros((n_pages, self.page_bytes), dtype=torch.uint8, device="cuda")
            v = torch.zeros_like(k)
        for p in (k, v):
            if (p.dtype != torch.uint8 or not p.is_contiguous() or
                    p.numel() != n_pages * self.page_bytes):
                raise ValueError("a pool must be a contiguous uint8 tensor of n_pages * "
                                 "page_bytes")
        _on_device(torch, "pools", k, v)
        self.k, self.v = k, v

    def batch(self, table, lens) -> "PagedBatch":
        return PagedBatch(self, table, lens)


class PagedBatch:
    """Sequences over a PagedCache: row b of `table` holds the page ids of sequence b, lens[b] its
    positions with the tokens of the next call counted. Both are read when a call runs."""

    def __init__(self, cache: PagedCache, table, lens):
        torch = _torch()
        if table.dim() != 2:
            raise ValueError("table must be (sequences, pages)")
        _ints(torch, "table", table, tuple(table.shape))
        _ints(torch, "lens", lens, (table.shape[0],))
        self._device = _on_device(torch, "table, lens and pools", table, lens, cache.k)
        self.cache, self._table, self._lens = cache, table, lens
        self.n_seqs = int(table.shape[0])
        self._kv = _lib.PagedKV(cache.k.data_ptr(), cache.v.data_ptr(), table.data_ptr(),
                                lens.data_ptr(), KV_DTYPES[cache.kv_dtype], cache.page_size,
                                cache.n_pages, cache.n_kv_heads, cache.head_dim, self.n_seqs,
                                int(table.shape[1]))
        self._ref = C.byref(self._kv)
        self._lib = _lib.load()
        self._append, self._attn = self._lib.csdr_paged_append, self._lib.csdr_paged_attn
        self._need = {}  # workspace bytes by the call's sizes

    @property
    def table(self):
        """Page ids, to be changed in place: a batch keeps the tensor it was made with."""
        return self._table

    @property
    def lens(self):
        """Lengths, to be changed in place as `table` is."""
        return self._lens

    def _here(self, torch, *ts) -> int:
        """Checks that a call's tensors and the cache are on the current device; its index."""
        dev = _on_device(torch, "tensors", *ts)
        if dev != self._device:
            raise ValueError("the cache must be on the current device")
        return dev

    def _starts(self, torch, q_start, max_q):
        if q_start is None:
            return None, 0
        _ints(torch, "q_start", q_start, (self.n_seqs + 1,))
        if max_q is None:
            raise ValueError("q_start needs max_q, the most tokens of one sequence")
        return q_start.data_ptr(), _int(int(max_q))

    def _heads(self, what: str, t, n_heads=None):
        """The token stride of (tokens, heads, head_dim) or (tokens, heads * head_dim)."""
        hd, shape, stride = self.cache.head_dim, t.shape, t.stride()
        if len(shape) == 3:
            n = shape[1]
            ok = shape[2] == hd and stride[2] == 1 and (n == 1 or stride[1] == hd)
        else:
            ok = len(shape) == 2 and shape[1] % hd == 0 and stride[1] == 1
            n = shape[-1] // hd if ok else 0
        if not ok or n < 1 or (n_heads is not None and n != n_heads):
            raise ValueError(f"{what} must be (tokens, {n_heads or 'heads'}, {hd}) with a token's "
                             "values side by side")
        if shape[0] < 2:
            return n, 0
        if stride[0] < n * hd:  # an expanded tensor, or rows that overlap
            raise ValueError(f"{what}: its tokens overlap")
        return n, stride[0]

    def append(self, q, k, v, theta: float = 0.0, q_start=None, max_q=None, q_out=None,
               stream=None):
        """Write the tokens' keys, rotated with base theta (0: as they are), and values into the
        cache; returns the rotated queries, (tokens, heads, head_dim). q may be None."""
        torch = _torch()
        nkv, hd = self.cache.n_kv_heads, self.cache.head_dim
        n = k.shape[0]
        dt = _dtype(k)
        _, ks = self._heads("k", k, nkv)
        _, vs = self._heads("v", v, nkv)
        if v.shape[0] != n or v.dtype != k.dtype:
            raise ValueError("k and v must have the same tokens and type")
        nq = qs = 0
        if q is not None:
            nq, qs = self._heads("q", q)
            if q.shape[0] != n or q.dtype != k.dtype:
                raise ValueError("q and k must have the same tokens and type")
            if q_out is None:
                q_out = _empty(torch, (n, nq, hd), q.dtype, q.device, stream)
            elif q_out.dtype != q.dtype or q_out.numel() != n * nq * hd or \
                    not q_out.is_contiguous():
                raise ValueError("q_out must be contiguous (tokens, heads, head_dim) of q's type")
        elif q_out is not None:
            raise ValueError("q_out without q")
        starts, mq = self._starts(torch, q_start, max_q)
        dev = self._here(torch, q, k, v, q_out, q_start)
        if n == 0:
            return q_out
        rc = self._append(
            self._ref, q.data_ptr() if q is not None else None, k.data_ptr(), v.data_ptr(), dt, n,
            starts, mq, nq, qs, ks, vs, theta, q_out.data_ptr() if q_out is not None else None,
            _stream_of(torch, dev, stream))
        if rc:
            _check(rc)
        return q_out

    def attend(self, q, q_start=None, max_q=None, max_len: int = 0, scale: float = 0.0,
               softcap: float = 0.0, window: int = 0, slopes=None, prefix=None, out=None,
               workspace=None, stream=None):
        """Attention of the tokens (rotated queries) to what their sequences hold; (tokens, heads,
        head_dim) of q's type. scale 0: 1 / sqrt(head_dim). softcap, window, slopes (float32 per
        head), prefix (int32 per sequence): csdr_attn_options. max_len: a bound of lens that the
        caller knows, 0 for the table's capacity."""
        torch = _torch()
        dt = _dtype(q)
        n = q.shape[0]
        nq, qs = self._heads("q", q)
        if out is None:
            out = _empty(torch, (n, nq, self.cache.head_dim), q.dtype, q.device, stream)
        elif out.dtype != q.dtype or out.numel() != n * nq * self.cache.head_dim or \
                not out.is_contiguous():
            raise ValueError("out must be contiguous (tokens, heads, head_dim) of q's type")
        opt = None
        if softcap or window or slopes is not None or prefix is not None:
            if slopes is not None and (slopes.dtype != torch.float32 or slopes.numel() != nq or
                                       not slopes.is_contiguous()):
                raise ValueError("slopes must be a contiguous float32 tensor, one per head")
            if prefix is not None:
                _ints(torch, "prefix", prefix, (self.n_seqs,))
            opt = C.byref(_lib.AttnOptions(softcap, _int(window),
                                           slopes.data_ptr() if slopes is not None else None,
                                           prefix.data_ptr() if prefix is not None else None))
        starts, mq = self._starts(torch, q_start, max_q)
        max_len = _int(max_len)
        dev = self._here(torch, q, out, q_start, slopes, prefix, workspace)
        if n == 0:
            return out
        if workspace is None:
            key = (n, starts is None, mq, nq, max_len)
            need = self._need.get(key)
            if need is None:
                if len(self._need) >= 256:
                    self._need.clear()
                need = self._need[key] = self._lib.csdr_paged_attn_workspace_bytes(
                    self._ref, n, starts, mq, nq, max_len)
            if need:
                workspace = _empty(torch, need, torch.uint8, q.device, stream)
        rc = self._attn(
            self._ref, q.data_ptr(), dt, n, starts, mq, nq, qs, max_len, scale, opt,
            out.data_ptr(), workspace.data_ptr() if workspace is not None else None,
            _bytes(workspace) if workspace is not None else 0, _stream_of(torch, dev, stream))
        if rc:
            _check(rc)
        return out

    def workspace_bytes(self, n_tokens: int, n_heads: int, q_start=None, max_q=None,
                        max_len: int = 0) -> int:
        """Bytes of attend's workspace, for callers that keep one."""
        starts, mq = self._starts(_torch(), q_start, max_q)
        return int(self._lib.csdr_paged_attn_workspace_bytes(
            self._ref, _int(n_tokens), starts, mq, _int(n_heads), _int(max_len)))

    def read(self, n_tokens: int, q_start=None, max_q=None, dtype: str = "f32", stream=None):
        """The cached keys and values of the sequences' last n_tokens rows (laid out as append's
        tokens are), two (n_tokens, kv heads, head_dim) tensors of "f32" or "f16"."""
        torch = _torch()
        if dtype not in ("f32", "f16"):
            raise ValueError("dtype must be 'f32' or 'f16'")
        c = self.cache
        k, v = _empty(torch, (2, n_tokens, c.n_kv_heads, c.head_dim),
                      torch.float16 if dtype == "f16" else torch.float32, c.k.device,
                      stream).unbind(0)
        starts, mq = self._starts(torch, q_start, max_q)
        dev = self._here(torch, k, q_start)
        if n_tokens == 0:
            return k, v
        _check(self._lib.csdr_paged_read(self._ref, n_tokens, starts, mq, k.data_ptr(),
                                         v.data_ptr(), int(dtype == "f16"),
                                         _stream_of(torch, dev, stream)))
        return k, v
