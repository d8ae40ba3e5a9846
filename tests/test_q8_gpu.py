"""8-bit rows (norm with residual, rows as they are or gated, back to values) and their products, on the
GPU against exact codes and fp64 (tests/q8_ref.py)."""
import numpy as np
import pytest

import q8_ref

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -11  # half a step, relative
NP = dict(f32=np.float32, f16=np.float16)


def dev(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def activations(rows, n, dtype, seed, spread=0.5):
    r = np.random.default_rng(seed)
    x = r.standard_normal((rows, n)) * np.exp(spread * r.standard_normal((rows, 1)))
    x[:, r.random(n) < 0.01] *= 6
    return x.astype(NP[dtype])


def check_rows(rows, t, factor=1.0, extra=0.0):
    """Codes exact, zeros behind them; scales within one rounding (and `extra`)."""
    n = t.shape[1]
    codes, scales = rows.codes.cpu().numpy(), rows.scales.cpu().numpy()
    want, top = q8_ref.codes_of(t)
    assert rows.n == n and codes.shape == (t.shape[0], -(-n // 128) * 128)
    np.testing.assert_array_equal(codes[:, :n], want)
    assert not codes[:, n:].any()
    s = (top * factor / 127).astype(np.float64)
    # one rounding to fp32 (an absolute half step below the normal numbers), fp64 in front of it
    assert (np.abs(scales - s) <= s * (U32 * (1 + 1e-6) + extra) + 2.0 ** -150).all()


SHAPES = [(1, 1), (3, 2), (1, 896), (5, 100), (2, 127), (2, 128), (2, 129), (7, 1001), (3, 2049), (2, 4096),
          (2, 5003), (64, 8192), (1, 11008), (2, 20001), (3, 33000), (2, 131071)]
MANY = [(515, 700), (513, 5003), (520, 9001), (512, 13001), (514, 17000)]  # up to 512 threads a row


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,n", SHAPES)
def test_quantize(gpu, rows, n, dtype):
    from cortexsdr_amd import q8

    x = activations(rows, n, dtype, seed=n)
    r = q8.quantize(dev(gpu, x))
    check_rows(r, x)
    codes, scales = r.codes.cpu().numpy()[:, :n], r.scales.cpu().numpy()
    v = scales[:, None] * codes.astype(np.float32)  # one rounding, the kernel's
    np.testing.assert_array_equal(r.values("f32").cpu().numpy(), v)
    np.testing.assert_array_equal(r.values("f16").cpu().numpy(), v.astype(np.float16))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,n", SHAPES)
def test_quantize_gated(gpu, rows, n, dtype):
    from cortexsdr_amd import q8

    # gate and x side by side, as one projection leaves them
    both = activations(rows, 2 * n, dtype, seed=n + 1)
    both[0, 0] = -95.0  # e^95 passes fp32
    d = dev(gpu, both)
    r = q8.quantize(d[:, n:], gate=d[:, :n])
    check_rows(r, q8_ref.silu_mul(both[:, :n], both[:, n:]))


def test_quantize_ties(gpu):
    """Values that lie exactly between two codes, of both signs, go to the even one."""
    from cortexsdr_amd import q8

    half = np.arange(-126.5, 127.0, 1.0)
    x = np.stack([np.append(half, 127.0), np.append(half, -127.0), np.append(half, 127.0) * 2.0 ** -20])
    for dtype in ("f32", "f16"):
        v = x[:2].astype(NP[dtype]) if dtype == "f16" else x.astype(np.float32)
        r = q8.quantize(dev(gpu, v))
        check_rows(r, v)
        assert (r.codes.cpu().numpy()[:, :254] % 2 == 0).all()
    # as gated values: silu(64) is 64 to every bit of fp64
    g = np.full((1, 255), 64.0, np.float32)
    r = q8.quantize(dev(gpu, x[:1].astype(np.float32)), gate=dev(gpu, g))
    check_rows(r, 64 * x[:1])


@pytest.mark.parametrize("scale", [1e-40, 1e-38, 1e-36, 1e-31, 1e-20, 1e30])
def test_quantize_ranges(gpu, scale):
    """Tiny and huge rows: denormal values too."""
    from cortexsdr_amd import q8

    x = (np.random.default_rng(5).standard_normal((4, 300)) * scale).astype(np.float32)
    check_rows(q8.quantize(dev(gpu, x)), x)
    g = np.random.default_rng(6).standard_normal((4, 300)).astype(np.float32)
    check_rows(q8.quantize(dev(gpu, x), gate=dev(gpu, g)), q8_ref.silu_mul(g, x))


@pytest.mark.parametrize("n", [40, 5000, 33000])
def test_quantize_gated_past_fp32(gpu, n):
    """Gated values past fp32 whose scale is not, and ones whose sigmoid leaves its normal numbers."""
    from cortexsdr_amd import q8

    g, x = activations(3, n, "f32", seed=n), activations(3, n, "f32", seed=n + 1)
    x[0] *= np.float32(1e36)
    x[0, 3], g[0, 3] = 3e38, 9.0
    x[1] = 1e-3
    x[1, ::7], g[1, ::7] = 1e37, -88.5
    g[2, 1], x[2, 1] = -120.0, 3e38
    r = q8.quantize(dev(gpu, x), gate=dev(gpu, g))
    check_rows(r, q8_ref.silu_mul(g, x))
    # and the scale past fp32 too
    x[0, 3], g[0, 3] = 3e38, 3e38
    r = q8.quantize(dev(gpu, x[:1]), gate=dev(gpu, g[:1]))
    assert gpu.isnan(r.scales).all() and not r.codes.any()


@pytest.mark.parametrize("n", [40, 700, 5000, 40000])
@pytest.mark.parametrize("gate", [False, True])
def test_quantize_not_finite(gpu, n, gate):
    """A row with a NaN or an infinity reads as NaN, a row of zeros as zeros, others as ever."""
    from cortexsdr_amd import q8

    x = activations(6, n, "f32", seed=n)
    g = activations(6, n, "f32", seed=n + 7)
    x[1, n - 1], x[2, 3], x[3, n // 2] = np.nan, np.inf, -np.inf
    x[4] = 0
    r = q8.quantize(dev(gpu, x), gate=dev(gpu, g) if gate else None)
    codes, scales = r.codes.cpu().numpy(), r.scales.cpu().numpy()
    assert np.isnan(scales[1:4]).all() and not codes[1:5].any() and scales[4] == 0.0
    t = q8_ref.silu_mul(g, x) if gate else x
    for i in (0, 5):
        want, top = q8_ref.codes_of(t[i:i + 1])
        np.testing.assert_array_equal(codes[i:i + 1, :n], want)
    v = r.values("f16").cpu().numpy()
    assert np.isnan(v[1:4]).all() and (v[4] == 0).all()


def test_rows_any_stride(gpu):
    """Rows at odd offsets and strides of larger buffers, the bytes around the outputs kept."""
    from cortexsdr_amd import _lib, q8

    torch = gpu
    for dtype in ("f32", "f16"):
        buf = dev(torch, activations(9, 777, dtype, seed=2))
        x = buf[:, 5:5 + 333]
        check_rows(q8.quantize(x), x.cpu().numpy())
        g = buf[:, 401:401 + 333]
        check_rows(q8.quantize(x, gate=g), q8_ref.silu_mul(g.cpu().numpy(), x.cpu().numpy()))
    # codes and scales into the middle of larger buffers
    x = dev(torch, activations(3, 200, "f32", seed=3))
    codes = torch.full((5, 256), 77, dtype=torch.int8, device="cuda")
    scales = torch.full((5,), 77.0, device="cuda")
    assert _lib.load().csdr_q8_quantize(x.data_ptr(), None, 0, 3, 200, 0, 0, codes[1].data_ptr(),
                                        scales[1:].data_ptr(),
                                        int(torch.cuda.current_stream().cuda_stream)) == 0
    check_rows(q8.Q8Rows(codes[1:4], scales[1:4], 200), x.cpu().numpy())
    assert (codes[0] == 77).all() and (codes[4] == 77).all() and scales[0] == 77 and scales[4] == 77


def norm_parts(h, w, eps):
    hd = h.astype(np.float64)  # (the call takes eps as fp32 holds it)
    return 1.0 / np.sqrt((hd * hd).mean(1) + float(np.float32(eps))), h.astype(q8_ref.LD) * w.astype(q8_ref.LD)


@pytest.mark.parametrize("x_type,res_type", [("f32", None), ("f16", None), ("f32", "f32"), ("f16", "f16"),
                                             ("f16", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("rows,n", SHAPES)
def test_norm(gpu, rows, n, x_type, res_type):
    from cortexsdr_amd import q8

    eps = 1e-5
    x = activations(rows, n, x_type, seed=n + 2)
    w = (1 + 0.3 * np.random.default_rng(n).standard_normal(n)).astype(np.float32)
    res, h = None, x
    if res_type:
        res = activations(rows, n, res_type, seed=n + 3)
        h = (x.astype(np.float32) + res.astype(np.float32)).astype(NP[res_type])
    r = q8.rms_norm(dev(gpu, x), dev(gpu, w), eps, residual=dev(gpu, res) if res_type else None, y=True)
    if res_type:
        np.testing.assert_array_equal(r.residual.cpu().numpy(), h)
    else:
        assert r.residual is None
    rms, t = norm_parts(h, w, eps)
    # fp64 statistics on both sides: sums of n terms, a root, a division
    check_rows(r.rows, t, rms, extra=(n + 8) * 2.0 ** -52)
    y = (t * rms[:, None]).astype(np.float64)
    # fp64, rounded to fp32 and then to the type
    tol = (U32 + (U16 if x_type == "f16" else 0)) * (1 + 1e-3)
    assert (np.abs(r.y.cpu().numpy() - y) <= np.abs(y) * tol + (2.0 ** -25 if x_type == "f16" else 2.0 ** -150)).all()
    # either output alone is the same
    a = q8.rms_norm(dev(gpu, x), dev(gpu, w), eps, residual=dev(gpu, res) if res_type else None)
    b = q8.rms_norm(dev(gpu, x), dev(gpu, w), eps, residual=dev(gpu, res) if res_type else None, q8=False,
                    y=True)
    assert a.y is None and b.rows is None
    assert gpu.equal(a.rows.codes, r.rows.codes) and gpu.equal(a.rows.scales, r.rows.scales)
    assert gpu.equal(b.y, r.y)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,n", MANY)
def test_many(gpu, rows, n, dtype):
    """Many rows of each kind, some of them against the formulas, the others against calls of few rows."""
    from cortexsdr_amd import q8

    torch = gpu
    both = activations(rows, 2 * n, dtype, seed=n)
    d, w = dev(torch, both), dev(torch, np.linspace(0.5, 2, n).astype(np.float32))
    x, g = d[:, n:], d[:, :n]
    pick = [0, 1, rows // 2, rows - 1]
    h = (both[pick, n:].astype(np.float32) + both[pick, :n].astype(np.float32)).astype(NP[dtype])
    rms, t = norm_parts(h, w.cpu().numpy(), 1e-5)
    kinds = [(lambda a, b: q8.quantize(a), both[pick, n:], 1.0, 0.0),
             (lambda a, b: q8.quantize(a, gate=b), q8_ref.silu_mul(both[pick, :n], both[pick, n:]), 1.0, 0.0),
             (lambda a, b: q8.rms_norm(a, w, residual=b).rows, t, rms, (n + 8) * 2.0 ** -52)]
    for f, v, factor, extra in kinds:
        r = f(x, g)
        check_rows(q8.Q8Rows(r.codes[pick], r.scales[pick], n), v, factor, extra)
        for first in range(0, rows, 100):
            few = f(x[first:first + 100], g[first:first + 100])
            assert torch.equal(few.codes, r.codes[first:first + 100])
            # (a norm's sum of squares in another order)
            assert ((few.scales - r.scales[first:first + 100]).abs() <= 2 * U32 * few.scales).all()


@pytest.mark.parametrize("n", [100, 4096, 40000])
@pytest.mark.parametrize("res_type", ["f32", "f16"])
def test_norm_in_place(gpu, n, res_type):
    """The stream updated in place, x at a stride."""
    from cortexsdr_amd import q8

    torch = gpu
    buf = dev(torch, activations(5, n + 9, "f16", seed=n))
    x, w = buf[:, 3:3 + n], torch.ones(n, device="cuda")
    res = dev(torch, activations(5, n, res_type, seed=n + 1))
    first = q8.rms_norm(x, w, residual=res)
    kept = res.clone()
    r = q8.rms_norm(x, w, residual=res, residual_out=res)
    assert r.residual is res and torch.equal(res, first.residual) and not torch.equal(res, kept)
    assert torch.equal(r.rows.codes, first.rows.codes) and torch.equal(r.rows.scales, first.rows.scales)
    # a strided stream out of place
    wide = torch.zeros((5, n + 4), dtype=res.dtype, device="cuda")
    wide[:, 1:1 + n] = kept
    again = q8.rms_norm(x, w, residual=wide[:, 1:1 + n])
    assert torch.equal(again.residual, res) and torch.equal(again.rows.codes, first.rows.codes)


def test_norm_ranges(gpu):
    """Rows of zeros, rows that hold what is not finite, squares past fp32, weights of zero."""
    from cortexsdr_amd import q8

    n = 600
    x = activations(8, n, "f32", seed=9)
    x[1] = 0
    x[2, 5], x[3, n - 1] = np.nan, -np.inf
    x[4] *= np.float32(1e25)
    x[5] *= np.float32(1e-30)
    w = np.linspace(-1, 1, n).astype(np.float32)
    w[5] = 0.0
    r = q8.rms_norm(dev(gpu, x), dev(gpu, w), 1e-5, y=True)
    codes, scales, y = r.rows.codes.cpu().numpy(), r.rows.scales.cpu().numpy(), r.y.cpu().numpy()
    assert scales[1] == 0 and not codes[1:4].any() and (y[1] == 0).all()
    assert np.isnan(scales[2]) and np.isnan(scales[3])
    rms, t = norm_parts(x, w, 1e-5)
    for i in (0, 4, 5, 6, 7):
        np.testing.assert_array_equal(codes[i:i + 1, :n], q8_ref.codes_of(t[i:i + 1])[0])
        want = (t[i] * rms[i]).astype(np.float64)
        assert (np.abs(y[i] - want) <= np.abs(want) * U32 * 1.001 + 2.0 ** -150).all()
    zero = q8.rms_norm(dev(gpu, x[:1]), gpu.zeros(n, device="cuda"))
    assert zero.rows.scales.item() == 0 and not zero.rows.codes.any()
    # without eps a row of zeros has no norm
    none = q8.rms_norm(gpu.zeros(2, 100, device="cuda"), gpu.ones(100, device="cuda"), 0.0, y=True)
    assert gpu.isnan(none.rows.scales).all() and not none.rows.codes.any() and gpu.isnan(none.y).all()
    nan = q8.rms_norm(dev(gpu, x[:1]), gpu.full((n,), float("nan"), device="cuda"))
    assert gpu.isnan(nan.rows.scales).all() and not nan.rows.codes.any()


# ---------------------------------------------------------------- products


def random_rows(torch, rows, n, seed, whole=False):
    """Codes over their whole range (with the one that no quantiser here makes, -128), scales."""
    from cortexsdr_amd import q8

    r = np.random.default_rng(seed)
    c = r.integers(-128, 128, (rows, n), dtype=np.int8)
    s = np.exp(r.standard_normal(rows)).astype(np.float32) / 64
    return c, s, q8.Q8Rows.pack(dev(torch, c), dev(torch, s))


def check_linear(y, xc, xs, wc, ws, bias=None, add=None):
    check_sums(y, q8_ref.sums(xc, wc), xs, ws, bias, add)


def check_sums(y, sums, xs, ws, bias=None, add=None):
    p, mag = q8_ref.linear(sums, xs, ws, bias, add)
    y = y.cpu().numpy()
    half = y.dtype == np.float16
    # fp32: the sum's conversion, two scales, two additions; then one rounding to the type
    tol = 5 * U32 * 1.001 * mag + (U16 if half else 0) * np.abs(p) * 1.01 + (2.0 ** -25 if half else 2.0 ** -149)
    over = np.abs(p) > 65000 if half else np.zeros(p.shape, bool)
    assert (np.abs(y - p)[~over] <= tol[~over]).all(), np.max((np.abs(y - p) - tol)[~over])


# By the tile that the rule takes for them (rows x tokens); each with rests of rows and tokens, with fewer steps of
# 128 columns than stages in flight and with more
PRODUCTS = [
    # 16 x 16, four waves sharing the columns
    (1, 1, 1), (1, 16, 64), (1, 17, 130), (2, 1152, 896), (3, 5, 4096), (5, 33, 1000), (16, 896, 4864),
    (17, 100, 777), (31, 257, 128), (33, 64, 300), (64, 1001, 999), (129, 257, 1024), (255, 511, 384),
    # 32 x 32, two waves sharing the columns
    (256, 512, 896), (300, 1152, 896), (515, 700, 129), (1000, 130, 2000), (64, 4096, 1100),
    # 32 x 64
    (333, 1001, 4999), (420, 1003, 3000),
    # 64 x 64
    (520, 4090, 100), (600, 1500, 1), (2, 33000, 257),
    # 128 x 64
    (1, 22001, 300), (1, 22016, 1), (260, 11001, 700), (900, 2100, 140), (1030, 1290, 257),
    # 128 x 128
    (1500, 3000, 130),
    # 256 x 256
    (3900, 4090, 1000), (3901, 3900, 385),
]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("M,R,C", PRODUCTS)
def test_linear(gpu, M, R, C, dtype):
    from cortexsdr_amd import q8

    xc, xs, x = random_rows(gpu, M, C, seed=M)
    wc, ws, w = random_rows(gpu, R, C, seed=R + 1)
    if dtype == "f16":  # keep within fp16
        ws = (ws / C).astype(np.float32)
        w = q8.Q8Rows.pack(dev(gpu, wc), dev(gpu, ws))
    sums = q8_ref.sums(xc, wc)
    check_sums(q8.linear(w, x, dtype=dtype), sums, xs, ws)
    r = np.random.default_rng(C)
    bias = r.standard_normal(R).astype(np.float32)
    add = r.standard_normal((M, R)).astype(NP[dtype])
    check_sums(q8.linear(w, x, bias=dev(gpu, bias), dtype=dtype), sums, xs, ws, bias)
    check_sums(q8.linear(w, x, add=dev(gpu, add), dtype=dtype), sums, xs, ws, None, add)
    # into rows of a larger buffer at an odd offset, onto what they hold
    wide = gpu.full((M, R + 7), 5.0, dtype=getattr(gpu, "float32" if dtype == "f32" else "float16"),
                    device="cuda")
    out = wide[:, 3:3 + R]
    out.copy_(dev(gpu, add))
    y = q8.linear(w, x, bias=dev(gpu, bias), add=out, dtype=dtype, out=out)
    check_sums(y, sums, xs, ws, bias, add)
    assert (wide[:, :3] == 5).all() and (wide[:, 3 + R:] == 5).all()


@pytest.mark.parametrize("M,R", [(1, 40), (4, 16), (20, 48), (70, 150), (300, 400)])
def test_linear_longest(gpu, M, R):
    """The widest rows with the largest codes: sums up to 2^31."""
    from cortexsdr_amd import q8

    C = 131071
    xc = np.full((M, C), -128, np.int8)
    wc = np.full((R, C), -128, np.int8)
    xc[M // 2, ::2] = 127
    wc[R // 2] = 127
    one = lambda n: np.ones(n, np.float32)  # noqa: E731
    y = q8.linear(q8.Q8Rows.pack(dev(gpu, wc), dev(gpu, one(R))), q8.Q8Rows.pack(dev(gpu, xc), dev(gpu, one(M))))
    check_linear(y, xc, one(M), wc, one(R))


def test_linear_nan_scales(gpu):
    """A token or a channel that reads as NaN is NaN, the others are not touched by it."""
    from cortexsdr_amd import q8

    for M in (5, 200):
        xc, xs, x = random_rows(gpu, M, 256, seed=1)
        wc, ws, w = random_rows(gpu, 300, 256, seed=2)
        x.scales[2] = float("nan")
        w.scales[7] = float("nan")
        y = q8.linear(w, x).cpu().numpy()
        assert np.isnan(y[2]).all() and np.isnan(y[:, 7]).all()
        rows, cols = np.arange(M) != 2, np.arange(300) != 7
        assert np.isfinite(y[rows][:, cols]).all()


def test_linear_one_order(gpu):
    """Every size gives a token the same values, whatever stands beside it."""
    from cortexsdr_amd import q8

    torch = gpu
    xc, xs, x = random_rows(torch, 600, 1024, seed=4)
    wc, ws, w = random_rows(torch, 700, 1024, seed=5)
    y = q8.linear(w, x)
    for M in (1, 4, 9, 16, 40, 64, 100, 129, 250, 257, 513):
        part = q8.Q8Rows(x.codes[:M], x.scales[:M], 1024)
        assert torch.equal(q8.linear(w, part), y[:M]), M


@pytest.mark.parametrize("rows", [2, 40000])
def test_linear_far(gpu, rows):
    """Offsets past 2^32 bytes: in the output (40000 tokens of 40000 channels), in the weights."""
    from cortexsdr_amd import q8

    torch = gpu
    if rows == 2:  # 40000 rows of 131072 bytes
        w = q8.Q8Rows(torch.zeros((40000, 131072), dtype=torch.int8, device="cuda"),
                      torch.ones(40000, device="cuda"), 131071)
        w.codes[39990:, 7] = torch.arange(1, 11, dtype=torch.int8, device="cuda")
        xc = np.zeros((rows, 131071), np.int8)
        xc[:, 7] = (3, 5)
        y = q8.linear(w, q8.Q8Rows.pack(dev(torch, xc), torch.ones(rows, device="cuda"))).cpu().numpy()
        want = np.arange(1, 11)
        np.testing.assert_array_equal(y[:, 39990:], np.stack([3 * want, 5 * want]))
        assert not y[:, :39990].any()
        return
    c = torch.zeros((rows, 128), dtype=torch.int8, device="cuda")
    c[:, 0] = (torch.arange(rows, device="cuda") % 101).to(torch.int8)
    r = q8.Q8Rows(c, torch.ones(rows, device="cuda"), 100)
    y = q8.linear(r, r)
    v = c[:, 0].float()
    for i in (0, 1, 26843, 26844, 39999):
        assert torch.equal(y[i], v[i] * v), i
    del y
    torch.cuda.empty_cache()


def test_norm_past_fp32(gpu):
    """Values whose products with the weights pass fp32, and some that leave its normal numbers."""
    from cortexsdr_amd import q8

    x = activations(4, 500, "f32", seed=21)
    x[0] *= np.float32(1e37)
    x[1] *= np.float32(1e-37)
    x[2, 7] = 3e38
    w = (1 + np.random.default_rng(3).random(500)).astype(np.float32) * np.float32(50)
    w[::3] = np.float32(1e-30)
    for n in (500, 499):
        r = q8.rms_norm(dev(gpu, x[:, :n]), dev(gpu, w[:n]), 1e-5)
        rms, t = norm_parts(x[:, :n], w[:n], 1e-5)
        check_rows(r.rows, t, rms, extra=(n + 8) * 2.0 ** -52)


def test_streams(gpu):
    """Products and norms on two streams at once, each with its own outputs."""
    from cortexsdr_amd import q8

    torch = gpu
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    sets = []
    for i in range(2):
        xc, xs, x = random_rows(torch, 200 + i, 700, seed=i)
        wc, ws, w = random_rows(torch, 900, 700, seed=i + 5)
        sets.append((x, w, torch.randn(300, 4000 + i, device="cuda"), torch.ones(4000 + i, device="cuda")))
    want = [(q8.linear(w, x), q8.rms_norm(v, n).rows.codes) for x, w, v, n in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate((a, b)):
            x, w, v, n = sets[i]
            got[i].append((q8.linear(w, x, stream=st), q8.rms_norm(v, n, stream=st).rows.codes))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i][0]) and torch.equal(c, want[i][1]) for y, c in got[i])


def test_rows_far(gpu):
    """Offsets past 2^32 bytes: in the values, the codes, the stream and the way back."""
    from cortexsdr_amd import q8

    torch = gpu
    n, rows = 131071, 33000
    x = torch.zeros((rows, n), dtype=torch.float16, device="cuda")
    last = activations(2, n, "f16", seed=1)
    x[rows - 2:] = dev(torch, last)
    r = q8.quantize(x)
    assert not r.scales[:rows - 2].any() and not r.codes[rows - 3].any()
    check_rows(q8.Q8Rows(r.codes[rows - 2:], r.scales[rows - 2:], n), last)
    v = r.values("f16")
    assert torch.equal(v[rows - 1], (r.scales[rows - 1] * r.codes[rows - 1, :n].float()).half())
    assert not v[rows - 3].any()
    del v
    w = torch.ones(n, device="cuda")
    normed = q8.rms_norm(x, w, residual=x, residual_out=None)
    assert torch.equal(normed.residual[rows - 2:], x[rows - 2:] + x[rows - 2:])
    h = (last.astype(np.float32) * 2).astype(np.float16)
    rms, t = norm_parts(h, np.ones(n, np.float32), 1e-5)
    check_rows(q8.Q8Rows(normed.rows.codes[rows - 2:], normed.rows.scales[rows - 2:], n), t, rms,
               extra=(n + 8) * 2.0 ** -52)
    del x, r, normed
    torch.cuda.empty_cache()


def test_python_refusals(gpu):
    from cortexsdr_amd import q8

    torch = gpu
    x = torch.randn(4, 100, device="cuda")
    w = torch.ones(100, device="cuda")
    r = q8.quantize(x)
    bad = [
        lambda: q8.quantize(x.double()), lambda: q8.quantize(x[0]), lambda: q8.quantize(x.t()),
        lambda: q8.quantize(x[:1].expand(4, 100)), lambda: q8.quantize(x, gate=x[:2]),
        lambda: q8.quantize(x, gate=x.half()), lambda: q8.quantize(x.cpu()),
        lambda: q8.quantize(torch.empty((2, 131072), device="cuda")),
        lambda: q8.quantize(torch.empty((2, 0), device="cuda")),
        lambda: q8.Q8Rows(r.codes[:, :100], r.scales, 100), lambda: q8.Q8Rows(r.codes, r.scales[:2], 100),
        lambda: q8.Q8Rows(r.codes, r.scales, 129), lambda: q8.Q8Rows(r.codes.float(), r.scales, 100),
        lambda: r.values("f64"), lambda: r.values("f32", out=torch.empty(4, 99, device="cuda")),
        lambda: q8.rms_norm(x, w[:99]), lambda: q8.rms_norm(x, w.half()), lambda: q8.rms_norm(x, w, q8=False),
        lambda: q8.rms_norm(x, w, residual=x[:3]), lambda: q8.rms_norm(x, w, residual_out=x),
        lambda: q8.rms_norm(x, w, residual=x, residual_out=x.half()),
        lambda: q8.linear(r, q8.quantize(x[:, :99])), lambda: q8.linear(r, r, dtype="bf16"),
        lambda: q8.linear(r, r, bias=torch.ones(3, device="cuda")),
        lambda: q8.linear(r, r, add=torch.ones((4, 4), device="cuda"), dtype="f16"),
        lambda: q8.linear(r, r, out=torch.ones((4, 5), device="cuda")),
        lambda: q8.linear(r, r, out=torch.ones((4, 4), device="cuda").t()[:, :]),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(RuntimeError):
        q8.rms_norm(x, w, eps=-1.0)


def test_no_rows(gpu):
    from cortexsdr_amd import q8

    x = gpu.empty((0, 300), device="cuda")
    r = q8.quantize(x)
    assert r.rows == 0 and r.codes.shape == (0, 384) and r.values().shape == (0, 300)
    n = q8.rms_norm(x, gpu.ones(300, device="cuda"), residual=x, y=True)
    assert n.y.shape == (0, 300) and n.residual.shape == (0, 300)
    w = q8.quantize(gpu.randn(5, 300, device="cuda"))
    assert q8.linear(w, r).shape == (0, 5) and q8.linear(r, w).shape == (5, 0)
