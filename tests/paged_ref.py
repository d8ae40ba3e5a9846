"""The paged cache's operators in fp64 on the CPU: numpy, from their formulas, sequence by sequence,
with no pages."""
import numpy as np

GROUP = 32


def rotate(x, pos, theta):
    """x (n, heads, hd) at positions pos (n,), adjacent pairs."""
    x = x.astype(np.float64)
    if not theta:
        return x
    hd = x.shape[-1]
    ang = pos.astype(np.float64)[:, None, None] * theta ** (-np.arange(0, hd, 2) / hd)
    c, s = np.cos(ang), np.sin(ang)
    out = np.empty_like(x)
    out[..., 0::2] = x[..., 0::2] * c - x[..., 1::2] * s
    out[..., 1::2] = x[..., 0::2] * s + x[..., 1::2] * c
    return out


def quantised(x):
    """The values that a 4-bit cache holds for x (n, heads, hd)."""
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        g = x.astype(np.float32).reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
        m = g.min(-1, keepdims=True).astype(np.float16)
        s = np.maximum((g.max(-1, keepdims=True) - m.astype(np.float32)) / np.float32(15), 0)
        s = s.astype(np.float16)
        bad = ~np.isfinite(g).all(-1, keepdims=True) | ~np.isfinite(m) | ~np.isfinite(s)
        m64, s64 = m.astype(np.float64), s.astype(np.float64)
        c = np.where(s64 > 0, np.rint((g.astype(np.float64) - m64) / s64), 0)
        v = (m64 + s64 * np.clip(c, 0, 15)).astype(np.float32)
        return np.where(bad, np.float32(np.nan), v).reshape(x.shape)


def held(x, kv):
    """The values the cache holds for fp32 x."""
    if kv == "q4":
        return quantised(x.astype(np.float32))
    with np.errstate(over="ignore"):
        return x.astype(np.float16).astype(np.float32)


def attend(q, pos, k, v, scale=0.0, cap=0.0, window=0, slopes=None, prefix=0):
    """q (n, Hq, hd) at positions pos; k, v (len, Hkv, hd): (n, Hq, hd). What a token does not
    see takes no part; a token that sees nothing gets zeros."""
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    G = q.shape[1] // k.shape[1]
    out = np.zeros(q.shape)
    p = np.arange(len(k))
    for i, pq in enumerate(pos):
        if pq < 0:
            continue
        see = (p <= pq) & (pq - p < (window or 1 << 30)) | (p < prefix)
        if not see.any():
            continue
        for h in range(q.shape[1]):
            with np.errstate(invalid="ignore", over="ignore"):
                s = k[see, h // G] @ q[i, h] * (scale or q.shape[-1] ** -0.5)
                if cap:
                    s = cap * np.tanh(s / cap)
                if slopes is not None:
                    s = s - float(slopes[h]) * np.abs(pq - p[see])
                w = np.exp(s - s.max())
                out[i, h] = w @ v[see, h // G] / w.sum()
    return out
