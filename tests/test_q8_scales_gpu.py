"""Products whose scales lie at the ends of fp32: what fits into fp32 comes out, whatever the scales' product with the
sum is on the way."""
import numpy as np
import pytest

import q8_ref
from test_q8_gpu import NP, U16, U32, dev

pytestmark = pytest.mark.gpu

MOST = {"f32": 2.0 ** 128 * (1 - 2.0 ** -25), "f16": 65520.0}  # from here on a value rounds to infinity


def check(y, sums, xs, ws, dtype):
    p, mag = q8_ref.linear(sums, xs, ws)
    y = y.cpu().numpy().astype(np.float64)
    # fp32: the sum's conversion and two products, exact or off by half a step of the subnormal numbers at most
    # below the normal ones; then one rounding to the type
    tol = 3 * U32 * 1.001 * mag + 2.0 ** -149
    if dtype == "f16":
        tol = tol + U16 * np.abs(p) * 1.01 + 2.0 ** -25
    over, under = np.abs(p) > MOST[dtype] * 1.001, np.abs(p) < MOST[dtype] * 0.999
    assert under.any()
    assert (np.abs(y - p)[under] <= tol[under]).all()
    np.testing.assert_array_equal(y[over], np.sign(p[over]) * np.inf)


# every tile, with rests of rows and tokens
@pytest.mark.parametrize("M,R", [(1, 17), (31, 257), (300, 1152), (420, 1003), (600, 1500), (900, 2102), (1500, 3001),
                                 (3900, 4090)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_scales_at_the_ends(gpu, M, R, dtype):
    from cortexsdr_amd import q8

    C = 300
    r = np.random.default_rng(M)
    xc, wc = (r.integers(-128, 128, (k, C), dtype=np.int8) for k in (M, R))
    ends = np.array([1e-45, 3e-42, 1e-38, 1e-30, 1e-5, 1.0, 1e5, 1e20, 8e31, 1e34, 2e36, 3.4e38], np.float32)
    xs, ws = ends[np.arange(M) % len(ends)], ends[r.integers(0, len(ends), R)]
    if M < len(ends):
        xs[0] = 8e31
    sums = q8_ref.sums(xc, wc)
    x, w = (q8.Q8Rows.pack(dev(gpu, c), dev(gpu, s)) for c, s in ((xc, xs), (wc, ws)))
    check(q8.linear(w, x, dtype=dtype), sums, xs, ws, dtype)
    # signs of scales, and sums of zero
    xs, ws = -xs, ws * r.choice([-1, 1], R).astype(np.float32)
    xc[M // 2], wc[R // 2] = 0, 0
    x, w = (q8.Q8Rows.pack(dev(gpu, c), dev(gpu, s)) for c, s in ((xc, xs), (wc, ws)))
    y = q8.linear(w, x, dtype=dtype)
    check(y, q8_ref.sums(xc, wc), xs, ws, dtype)
    assert not y[M // 2].any() and not y[:, R // 2].any()


def test_rows_of_large_values(gpu):
    """Quantised rows of up to 3e38 with weights that bring them back."""
    from cortexsdr_amd import q8

    r = np.random.default_rng(3)
    v = r.standard_normal((20, 4000)).astype(np.float32) * np.float32(5e37)
    m = r.standard_normal((50, 4000)).astype(np.float32) * np.float32(1e-6)
    x, w = q8.quantize(dev(gpu, v)), q8.quantize(dev(gpu, m))
    host = lambda q: (q.codes.cpu().numpy()[:, :4000], q.scales.cpu().numpy())  # noqa: E731
    (xc, xs), (wc, ws) = host(x), host(w)
    y = q8.linear(w, x)
    assert gpu.isfinite(y).all()
    check(y, q8_ref.sums(xc, wc), xs, ws, "f32")
    bias, add = (np.float32(1e33) * r.standard_normal(s).astype(np.float32) for s in (50, (20, 50)))
    y = q8.linear(w, x, bias=dev(gpu, bias), add=dev(gpu, add)).cpu().numpy()
    p, mag = q8_ref.linear(q8_ref.sums(xc, wc), xs, ws, bias, add)
    assert (np.abs(y - p) <= 5 * U32 * 1.001 * mag).all()
    assert NP["f32"] == y.dtype
