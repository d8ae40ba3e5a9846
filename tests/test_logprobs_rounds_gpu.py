"""csdr_token_logprobs where a wave takes a row's segment in several rounds of 2048 values (many
rows), the running maximum moving between them, against fp64 numpy."""
import numpy as np
import pytest

import logprobs_ref as ref

pytestmark = pytest.mark.gpu

ROUND = 2048

# Z: a lane adds 32 values a round, up to 160 one after the other here, then 6 + 7 joins of lanes and
# segments: below 2^-16.5 of it at the very most. Exponents (x - m) / temperature are rounded four
# times (2^-22 of d, which moves Z by 2^-22 |d| exp(d) < 2^-23), and so is a value's own.
LP = 2.0 ** -16


def close(got, want, tol):
    got, want = got.cpu().numpy().astype(np.float64), np.asarray(want)
    with np.errstate(over="ignore"):
        want = np.where(np.isinf(want.astype(np.float32)), -np.inf, want)  # past fp32
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got == -np.inf, want == -np.inf)
    fine = np.isfinite(want)
    off = np.abs(got[fine] - want[fine]) - 2.0 ** -22 * np.abs(want[fine])
    assert off.size == 0 or float((off / np.broadcast_to(tol, want.shape)[fine]).max()) <= 1


def check(gpu, x, tokens, top_n, temperature=1.0, copies=1):
    """`copies` of the rows, so that a segment has as many rounds as that many rows leave it."""
    from cortexsdr_amd.logprobs import token_logprobs

    rows = len(x)
    d = gpu.from_numpy(x).cuda().repeat(copies, 1)
    t = gpu.tensor(np.asarray(tokens), dtype=gpu.int32, device="cuda").repeat(copies)
    r = token_logprobs(d, t, top_n=top_n, temperature=temperature)
    lp, h, ids, tl, far = ref.scores(x, tokens, top_n, temperature)
    close(r.logprobs[:rows], lp, LP)
    # entropy = log Z - sum e d / Z: both sums as above, the second of size mean |d|
    close(r.entropy[:rows], h, LP * (2 + far))
    if top_n:
        assert np.array_equal(r.top_ids[:rows].cpu().numpy(), ids)
        close(r.top_logprobs[:rows], tl, LP)
    for a in r:  # every copy as the first, bit for bit
        if a is not None:
            a = (a.view(gpu.int32)).unflatten(0, (copies, rows))
            assert gpu.equal(a, a[:1].expand_as(a))
    return r


# rows of five rounds and a value in one segment; of two rounds a segment, the last one short
SIZES = [(10241, 8192), (7001, 4096)]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("n,total", SIZES)
@pytest.mark.parametrize("top_n", [0, 5, 64])
def test_masked_rounds(gpu, dtype, n, total, top_n):
    """Whole rounds of the type's lowest value, of large negative values and of -infinity before,
    between and after the allowed tokens."""
    rng = np.random.default_rng(n)
    low = np.finfo(dtype).min
    x = (2.5 * rng.normal(size=(16, n))).astype(dtype)
    x[0, :ROUND] = low
    x[1, :ROUND] = low / 4
    x[2, :n - 3] = low                      # allowed: the last three
    x[3, :ROUND] = -np.inf
    x[3, ROUND:2 * ROUND] = low
    x[4, ROUND:] = low                      # allowed: the first round
    x[5] = low
    x[5, n // 2] = 1.0
    x[6, ::2] = low
    x[7, :ROUND] = low
    x[7, ROUND:2 * ROUND] = -1.2e37 if dtype == np.float32 else -30000
    x[8, :3 * ROUND] = low
    x[8, 100] = -50.0
    x[9] = low
    x[10] = -np.inf
    x[10, n - 1] = low
    x[11, :2 * ROUND + 17] = -1e30 if dtype == np.float32 else -6e4
    x[12, :-1] = -np.inf
    x[13, ROUND:2 * ROUND] = -np.inf
    x[14, :ROUND] = np.linspace(float(low), 0, ROUND)
    x[15, :ROUND] = low
    x[15, ROUND:2 * ROUND] -= dtype(100)
    check(gpu, x, [n - 1, 0, n - 2, n - 5, 3, n // 2, 1, ROUND, 100, 4, n - 1, 0, n - 1, 7, ROUND - 1,
                   n - 9], top_n, copies=total // 16)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("n,total", SIZES)
@pytest.mark.parametrize("top_n", [1, 20, 64])
def test_order_over_rounds(gpu, dtype, n, total, top_n):
    """Ties within and across rounds, sorted rows either way, constant rows, rounds that each beat
    the ones before."""
    rng = np.random.default_rng(n + 1)
    x = np.zeros((8, n), dtype)
    x[0] = rng.integers(-3, 3, n)
    x[1] = np.arange(n) * (20.0 / n)
    x[2] = x[1][::-1]
    x[4] = np.arange(n) // ROUND
    x[5] = x[4][::-1]
    x[6] = -5 * rng.random(n)
    x[6, ROUND - 30:ROUND + 30] = 2.0
    x[7] = np.arange(n) // 700 % 3
    check(gpu, x, [0, n - 1, 0, 5, n - 1, 0, ROUND, n // 2], top_n, copies=total // 8)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("n,total", SIZES)
def test_bad_values_over_rounds(gpu, dtype, n, total):
    """NaN and +infinity in the first, a middle and the last round, beside masked rounds."""
    rng = np.random.default_rng(n + 2)
    x = rng.normal(size=(8, n)).astype(dtype)
    for r, (i, v) in enumerate([(5, np.nan), (ROUND + 5, np.nan), (n - 1, np.nan), (5, np.inf),
                                (2 * ROUND + 7, np.inf), (n - 1, np.inf)]):
        x[r, i] = v
    x[6, :ROUND] = np.finfo(dtype).min
    x[6, ROUND + 1] = np.nan
    x[7] = -np.inf
    x[7, n - 2] = np.inf
    check(gpu, x, [0, 1, 2, 5, 3, n - 1, 0, 3], 9, copies=total // 8)
