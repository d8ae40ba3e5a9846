"""GPU parity of csdr_token_logprobs (log probabilities, entropy, top tokens) against fp64 numpy."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def expect(x, tokens, top_n, temperature=1.0):
    """x (rows, n) as the fp32 or fp16 values given."""
    inv = np.float32(1) / np.float32(temperature) if temperature > 0 else np.float32(1)
    y = (x.astype(np.float32) * inv).astype(np.float64)  # y is rounded to fp32 once
    rows, n = y.shape
    lp, h = np.full(rows, np.nan), np.full(rows, np.nan)
    ids = np.full((rows, top_n), -1, np.int32)
    tl = np.full((rows, top_n), -np.inf)
    for r in range(rows):
        bad = np.isnan(y[r]).any() or (y[r] == np.inf).any()
        live = np.isfinite(y[r])
        m = y[r][live].max() if live.any() else 0.0
        z = np.exp(y[r][live] - m).sum()
        # about the maximum: log Z is lost beside a maximum of the type's lowest value
        lz = np.nan if bad else np.log(z) if live.any() else 0.0
        p = np.exp(y[r][live] - m) / z if live.any() else np.zeros(0)
        h[r] = lz - (p * (y[r][live] - m)).sum()
        t = int(tokens[r])
        lp[r] = 0.0 if t < 0 else np.nan if t >= n or bad else \
            -np.inf if y[r][t] == -np.inf else y[r][t] - m - lz
        order = np.argsort(np.where(live, -y[r], np.inf), kind="stable")[:min(top_n, live.sum())]
        ids[r, :len(order)] = order
        tl[r, :len(order)] = y[r][order] - m - lz
    return lp, h, ids, tl


# y - m and log Z are rounded once each (values up to 2^5: half a step is 2^-20), Z is a sum of up to
# 2^18 rounded exponentials in a tree of fewer than 2^7 roundings per leaf: 2^-17 relative at the
# very most; the entropy's weighted sum likewise, times |y - m| up to 2^5 for terms whose weights
# add to one.
def close(got, want, tol):
    got, want = got.astype(np.float64), np.asarray(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got == -np.inf, want == -np.inf)
    fine = np.isfinite(want)
    if fine.any():
        # far below the maximum (|y - m| past 2^5) the two roundings are 2^-24 of the value each
        off = np.abs(got[fine] - want[fine]) - 2.0 ** -23 * np.abs(want[fine])
        assert float(off.max()) <= tol


def check(gpu, x, tokens, top_n, temperature=1.0, pad=0):
    from cortexsdr_amd.logprobs import token_logprobs

    rows, n = x.shape
    wide = np.full((rows, n + pad), 6e4, x.dtype) if pad else x
    wide[:, :n] = x
    d = gpu.from_numpy(np.ascontiguousarray(wide)).cuda()[:, :n]
    t = gpu.tensor(np.asarray(tokens), dtype=gpu.int32, device="cuda")
    r = token_logprobs(d, t, top_n=top_n, temperature=temperature)
    lp, h, ids, tl = expect(x, tokens, top_n, temperature)
    close(r.logprobs.cpu().numpy(), lp, 2.0 ** -16)
    close(r.entropy.cpu().numpy(), h, 2.0 ** -14)
    if top_n:
        assert np.array_equal(r.top_ids.cpu().numpy(), ids)
        close(r.top_logprobs.cpu().numpy(), tl, 2.0 ** -16)
    else:
        assert r.top_ids is None and r.top_logprobs is None
    return r


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("rows,n,top_n", [
    (1, 1, 1), (1, 1, 5), (3, 2, 2), (2, 63, 64), (5, 257, 20), (1, 151936, 20), (2, 151936, 64),
    (40, 5003, 5), (300, 1000, 1), (7, 32003, 0), (1, 262144, 50), (2, 16385, 64),
])
def test_shapes(gpu, dtype, rows, n, top_n):
    rng = np.random.default_rng(rows * 1000 + n)
    x = (2.5 * rng.normal(size=(rows, n))).astype(dtype)
    check(gpu, x, rng.integers(0, n, rows), top_n)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("pad", [1, 3, 8])
@pytest.mark.parametrize("temperature", [0.8, 0.0, 3.0])
def test_strides_and_temperature(gpu, dtype, pad, temperature):
    rng = np.random.default_rng(pad)
    x = rng.normal(size=(9, 4097)).astype(dtype)
    check(gpu, x, rng.integers(0, 4097, 9), 7, temperature, pad)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("n", [50, 5000, 100000])
def test_ties_go_to_the_lower_id(gpu, dtype, n):
    """Constant rows, few distinct values, a plateau at the end, zeros of both signs."""
    rng = np.random.default_rng(n)
    x = np.zeros((5, n), dtype)
    x[1] = rng.integers(-2, 2, n)
    x[2, n // 2:] = 3
    x[3, ::2] = -0.0
    x[4] = np.minimum(np.arange(n) // 7, 30000)
    check(gpu, x, [0, n - 1, n // 2, 1, n - 1], 64)
    check(gpu, x, [0, n - 1, n // 2, 1, n - 1], 1)


@pytest.mark.parametrize("n", [3000, 70000])
def test_sorted_rows(gpu, n):
    """Ascending and descending values: every value, or only the first ones, beat what came
    before."""
    up = (np.arange(n) * (20.0 / n)).astype(np.float32)
    check(gpu, np.stack([up, up[::-1]]), [n - 1, n - 1], 64)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("n", [40, 40000])
def test_masked_and_bad_logits(gpu, dtype, n):
    """-infinity among, before and after the rest and everywhere; the type's lowest value; NaN and
    +infinity; tokens that are masked, absent or out of range."""
    rng = np.random.default_rng(n)
    x = rng.normal(size=(9, n)).astype(dtype)
    x[0, ::2] = -np.inf
    x[1, :] = -np.inf
    x[2, :] = -np.inf
    x[2, n // 3] = 1.5
    x[3, 7] = np.nan
    x[4, 9] = np.inf
    x[5, 1:] = np.finfo(dtype).min
    x[6, :n // 2] = -np.inf
    x[8, :] = np.finfo(dtype).min
    check(gpu, x, [0, 3, n // 3, 1, 1, 0, n - 1, -1, n], 20)


def test_peaked_rows(gpu):
    """One token near probability 1: the entropy is small, the others' far below."""
    x = np.zeros((3, 30000), np.float32)
    x[0, 123] = 40
    x[1, 7] = 88
    x[2, 29999] = 15
    check(gpu, x, [123, 8, 0], 3)


def test_without_tokens(gpu):
    from cortexsdr_amd.logprobs import token_logprobs

    x = gpu.randn(4, 100, device="cuda")
    r = token_logprobs(x, top_n=2)
    assert r.logprobs is None
    want = gpu.log_softmax(x.double(), 1).topk(2)
    assert gpu.equal(r.top_ids.long(), want.indices)
    assert float((r.top_logprobs.double() - want.values).abs().max()) <= 2.0 ** -16


@pytest.mark.parametrize("rows,n", [(3, 151936), (500, 3001)])
def test_captured(gpu, rows, n):
    """Captured once, replayed on new logits with eager calls between: equal to the eager call."""
    from cortexsdr_amd.logprobs import token_logprobs

    x = gpu.randn(rows, n, device="cuda")
    t = gpu.zeros(rows, dtype=gpu.int32, device="cuda")
    token_logprobs(x, t, top_n=5)
    g = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(g):
        r = token_logprobs(x, t, top_n=5)
    for i in range(4):
        x.copy_(gpu.randn(rows, n, device="cuda"))
        t.fill_(i)
        g.replay()
        e = token_logprobs(x, t, top_n=5)
        gpu.cuda.synchronize()
        for a, b in zip(r, e):
            assert gpu.equal(a, b)


def test_two_streams(gpu):
    from cortexsdr_amd.logprobs import token_logprobs

    xs = [gpu.randn(2, 151936, device="cuda") for _ in range(2)]
    want = [token_logprobs(x, top_n=9) for x in xs]
    streams = [gpu.cuda.Stream() for _ in xs]
    gpu.cuda.synchronize()
    outs = [[token_logprobs(x, top_n=9, stream=st) for _ in range(10)]
            for x, st in zip(xs, streams)]
    gpu.cuda.synchronize()
    for w, os_ in zip(want, outs):
        for o in os_:
            assert gpu.equal(o.top_ids, w.top_ids) and gpu.equal(o.entropy, w.entropy)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("top_n", [56, 57, 64])
def test_most_segments_and_places(gpu, dtype, top_n):
    """The longest rows with the most places: the lists of a row's segments at their largest."""
    x = np.random.default_rng(top_n).normal(size=(2, 300000)).astype(dtype)
    check(gpu, x, [0, 299999], top_n)
