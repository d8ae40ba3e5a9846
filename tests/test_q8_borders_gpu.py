"""Norms whose values lie beside the border between two codes by less than fp64's quotient tells: the nearer code
all the same, against exact codes (tests/q8_ref.py)."""
import numpy as np
import pytest

import q8_ref
from test_q8_gpu import check_rows, dev, norm_parts

pytestmark = pytest.mark.gpu


def near_ties(count, seed):
    """(h1, w1, h2, w2) of 24 bits each with 254 h2 w2 = c h1 w1 +- 1, c odd: 127 t / top is c / 2 but for
    1 / (2 h1 w1), on either side, with h1 w1 the larger."""
    r = np.random.default_rng(seed)
    found = []
    while len(found) < count:
        h1, h2, c = (int(r.integers(2 ** 23, 2 ** 24)) | 1, int(r.integers(2 ** 23, 2 ** 24)) | 1,
                     int(r.integers(0, 127)) * 2 + 1)
        m, sign = c * h1, int(r.choice([-1, 1]))
        try:
            w2 = sign * pow(254 * h2, -1, m) % m
        except ValueError:  # not coprime
            continue
        w1 = (254 * h2 * w2 - sign) // m
        if not (2 ** 12 < w2 < 2 ** 24 and 2 ** 12 < w1 < 2 ** 24):
            continue
        assert 254 * h2 * w2 == c * h1 * w1 + sign and h2 * w2 < h1 * w1
        found.append((h1, w1, h2, w2))
    return found


# one found by hand: 78.5 and a little
PAIRS = [(11119041, 15325327, 8435770, 12485855)] + near_ties(99, seed=1)


@pytest.mark.parametrize("n", [200, 5003, 33000])
# (2^-70 each: rows formed in fp64 throughout)
@pytest.mark.parametrize("size", [1.0, 2.0 ** -70])
def test_beside_a_border(gpu, n, size):
    from cortexsdr_amd import q8

    rows = len(PAIRS)
    h, w = np.zeros((rows, n), np.float32), np.ones(n, np.float32)
    at = np.random.default_rng(n).permutation(n)
    for i, (h1, w1, h2, w2) in enumerate(PAIRS):
        a, b = at[2 * i], at[2 * i + 1]
        h[i, a], w[a] = (-1) ** i * h1, w1
        h[i, b], w[b] = h2, w2
    h, w = h * np.float32(size), w * np.float32(size)
    rms, t = norm_parts(h, w, 1e-5)
    want = q8_ref.codes_of(t)[0]
    # the reference itself against whole numbers
    for i, (h1, w1, h2, w2) in enumerate(PAIRS):
        twice, top = 254 * h2 * w2, h1 * w1
        code = (twice + top) // (2 * top)
        assert want[i, at[2 * i + 1]] == code and twice != (2 * code - 1) * top
    check_rows(q8.rms_norm(dev(gpu, h), dev(gpu, w), 1e-5).rows, t, rms, extra=(n + 8) * 2.0 ** -52)
    # the same values as a sum with the stream's
    half = np.where(h != 0, 1.0, 0).astype(np.float32) * np.float32(size)
    r = q8.rms_norm(dev(gpu, half), dev(gpu, w), 1e-5, residual=dev(gpu, h - half))
    assert gpu.equal(r.residual, dev(gpu, h))
    check_rows(r.rows, t, rms, extra=(n + 8) * 2.0 ** -52)


def test_ties_to_even(gpu):
    """Values exactly on a border, as products of 24 bits: the even code."""
    from cortexsdr_amd import q8

    r = np.random.default_rng(2)
    n, rows = 512, 50
    h, w = np.zeros((rows, n), np.float32), np.ones(n, np.float32)
    for i in range(rows):
        m, v, c = int(r.integers(2 ** 15, 66052)), int(r.integers(2 ** 22, 2 ** 24)), 2 * int(r.integers(0, 127)) + 1
        h[i, 2 * i], w[2 * i] = 254 * m, v           # top = 254 m v
        h[i, 2 * i + 1], w[2 * i + 1] = m * c, v     # t = c m v = (c / 254) top
    rms, t = norm_parts(h, w, 1e-5)
    x = q8.rms_norm(dev(gpu, h), dev(gpu, w), 1e-5).rows
    check_rows(x, t, rms, extra=(n + 8) * 2.0 ** -52)
    codes = x.codes.cpu().numpy()
    assert (codes[np.arange(rows), 2 * np.arange(rows) + 1] % 2 == 0).all()
