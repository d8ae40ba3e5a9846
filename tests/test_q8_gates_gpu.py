"""Gated rows whose gates fp32 holds with few bits, under values that lift the product back: codes as of any
other gate, against exact codes (tests/q8_ref.py)."""
import numpy as np
import pytest

import q8_ref
from test_q8_gpu import check_rows, dev

pytestmark = pytest.mark.gpu

STEP = np.float32(2.0 ** -149)  # the smallest subnormal number


def rows(n):
    r = np.random.default_rng(n)
    g, x = np.zeros((6, n), np.float32), np.zeros((6, n), np.float32)
    at = r.permutation(n)  # (not only in the first chunks)
    # gates of a few steps
    g[0, at[:6]], x[0, at[:6]] = STEP * np.array([3, 1, 1, 2, 5, -3], np.float32), 1e30
    # the row's largest beside one whose product with the sigmoid alone would round upwards past it
    g[1, at[0]], x[1, at[0]] = STEP * np.float32(3), 1e30
    g[1, at[1]], x[1, at[1]] = 1.0, 3.45e-15
    # any gate below the normal numbers, and around their end, under any large value
    g[2] = r.integers(-2 ** 23, 2 ** 23, n) * STEP
    x[2] = np.exp(r.uniform(np.log(1e20), np.log(3e38), n))
    g[3] = r.choice([-1, 1], n) * np.exp2(r.uniform(-130, -120, n))
    x[3] = r.standard_normal(n) * 1e36
    # and among gates and values of common size
    g[4], x[4] = r.standard_normal(n), r.standard_normal(n)
    g[4, at[:n // 3]] = r.integers(-2 ** 20, 2 ** 20, n // 3) * STEP
    x[4, at[:n // 3]] = 1e38
    # gates and values whose product alone passes fp32, the gated value far below
    g[5], x[5] = r.uniform(-80, -30, n), 1e37 * r.standard_normal(n)
    return g, x


@pytest.mark.parametrize("n", [7, 40, 5000, 33000])
def test_gates_of_few_bits(gpu, n):
    from cortexsdr_amd import q8

    g, x = rows(n)
    t = q8_ref.silu_mul(g, x)
    check_rows(q8.quantize(dev(gpu, x), gate=dev(gpu, g)), t)
    # many rows take another number of threads
    reps = 100
    r = q8.quantize(dev(gpu, np.tile(x, (reps, 1))), gate=dev(gpu, np.tile(g, (reps, 1))))
    check_rows(q8.Q8Rows(r.codes[-6:], r.scales[-6:], n), t)


@pytest.mark.parametrize("n", [40, 33000])
def test_lowest_gates(gpu, n):
    """Gates far below where the exponential is a number, under values whose product with them passes fp32:
    a gated value of nothing, not NaN; and infinite ones, NaN as the formula's."""
    from cortexsdr_amd import q8

    g, x = np.full((4, n), 0.5, np.float32), np.full((4, n), 0.25, np.float32)
    g[0, n // 2], x[0, n // 2] = -3e38, 3e38
    g[1, n // 2], x[1, n // 2] = -200.0, 3e38
    g[2, n // 2], x[2, n // 2] = -np.inf, 1.0
    g[3, n // 2], x[3, n // 2] = -np.inf, 0.0
    r = q8.quantize(dev(gpu, x), gate=dev(gpu, g))
    check_rows(q8.Q8Rows(r.codes[:2], r.scales[:2], n), q8_ref.silu_mul(g[:2], x[:2]))
    assert gpu.isnan(r.scales[2:]).all() and not r.codes[2:].any()
