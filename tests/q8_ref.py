"""8-bit rows, their products and rotary positions from the formulas, on the CPU: codes in exact
arithmetic (80-bit floats hold 255 times a product of two fp32 numbers), everything else in fp64."""
import numpy as np

LD = np.longdouble


def codes_of(t):
    """Codes of rows t (exact values of at most 56 bits, as longdouble) and their largest magnitudes."""
    t = t.astype(LD)
    top = np.abs(t).max(1, keepdims=True)
    a = np.abs(t)
    with np.errstate(invalid="ignore", divide="ignore"):
        k = np.floor(127 * a / top)
    k = np.where(top > 0, k, 0)
    # the quotient may be off by its last bit: k is the floor in exact arithmetic
    k = np.where(k * top > 127 * a, k - 1, k)
    k = np.where((k + 1) * top <= 127 * a, k + 1, k)
    twice = 254 * a - 2 * k * top  # 2 (127 a - k top), against top
    up = (twice > top) | ((twice == top) & (k % 2 == 1))
    k = np.where((top > 0) & up, k + 1, k)
    return (np.sign(t) * k).astype(np.int32), top[:, 0]


def silu_mul(gate, x):
    g, x = gate.astype(LD), x.astype(LD)
    return g / (1 + np.exp(-g)) * x


def sums(xc, wc):
    return xc.astype(np.float64) @ wc.astype(np.float64).T  # exact: below 2^53


def linear(sums, xs, ws, bias=None, add=None):
    """The product and the sum of its terms' magnitudes, fp64."""
    p = sums * xs.astype(np.float64)[:, None] * ws.astype(np.float64)
    mag = np.abs(p)
    if bias is not None:
        p, mag = p + bias.astype(np.float64), mag + np.abs(bias.astype(np.float64))
    if add is not None:
        p, mag = p + add.astype(np.float64), mag + np.abs(add.astype(np.float64))
    return p, mag


def rotary(x, positions, freqs, layout, magnitude=1.0):
    """x (tokens, heads, dims of a head), fp64."""
    x = x.astype(np.float64)
    half = len(freqs)
    ang = positions.astype(LD)[:, None, None] * np.asarray(freqs, np.float64).astype(LD)
    c = (np.cos(ang) * magnitude).astype(np.float64)
    s = (np.sin(ang) * magnitude).astype(np.float64)
    y = x.copy()
    if layout == "adjacent":
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half], y[..., half:2 * half] = a * c - b * s, a * s + b * c
    return y
