"""GPU parity of the paged K/V cache (append with rotation, read, attention over fp16 and 4-bit
pages) against the fp64 formulas of paged_ref, through the Python entry points."""
import numpy as np
import pytest

import paged_ref as ref
from conftest import rel_l2

pytestmark = pytest.mark.gpu

# fp32: unscaled scores reach about 64, where half a step is 2^-19; up to hd = 128 roundings of
# that size add up like a random walk (11 times one), times the scale 128^-1/2: 2^-19 absolute on
# the largest scores, which is the relative error of their weights. A factor of 4 beside it.
TOL32 = 2.0 ** -17
# fp16: half a step (2^-11) for the weights' rounding and one for the output's.
TOL16 = 2 * 2.0 ** -11 + TOL32


def tol(x):
    return TOL32 if x == "f32" else TOL16


class Setup:
    """Sequences of given lengths (new tokens included) whose cache is filled by appends, over
    shuffled pages; `ref` mirrors what each position holds."""

    def __init__(self, gpu, lens, heads, kv, x="f32", ps=16, seed=0, spare=3, theta=0.0):
        from cortexsdr_amd.paged import PagedCache

        self.gpu, self.rng = gpu, np.random.default_rng(seed)
        self.Hq, self.Hkv, self.hd = heads
        self.kv, self.x, self.theta = kv, x, theta
        self.np_x = np.float16 if x == "f16" else np.float32
        per = max(1, max((n + ps - 1) // ps for n in lens)) + 1
        n_pages = len(lens) * per + spare
        self.cache = PagedCache(n_pages, ps, self.Hkv, self.hd, kv)
        # what lies in pages that nobody wrote: NaN in fp16 pages, scales and minima
        self.cache.k.fill_(0xFF)
        self.cache.v.fill_(0xFF)
        table = self.rng.permutation(n_pages)[:len(lens) * per].reshape(len(lens), per)
        self.table = gpu.tensor(table, dtype=gpu.int32, device="cuda")
        self.lens = gpu.zeros(len(lens), dtype=gpu.int32, device="cuda")
        self.batch = self.cache.batch(self.table, self.lens)
        self.k = [np.zeros((0, self.Hkv, self.hd), np.float32) for _ in lens]
        self.v = [np.zeros((0, self.Hkv, self.hd), np.float32) for _ in lens]
        self.len = [0] * len(lens)

    def dev(self, a):
        return self.gpu.from_numpy(np.ascontiguousarray(a)).cuda()

    def draw(self, n, heads, sigma=1.0):
        return (sigma * self.rng.normal(size=(n, heads, self.hd))).astype(self.np_x)

    def starts(self, new):
        return self.gpu.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=self.gpu.int32,
                               device="cuda")

    def positions(self, new):
        return [np.arange(self.len[b] - n, self.len[b]) for b, n in enumerate(new)]

    def append(self, new, with_q=True, k=None, v=None):
        """new[b] more tokens of each sequence in one call; returns (device q, rotated q fp64)."""
        n = sum(new)
        self.len = [a + b for a, b in zip(self.len, new)]
        self.lens.copy_(self.gpu.tensor(self.len, dtype=self.gpu.int32))
        q = self.draw(n, self.Hq, 1.5) if with_q else None
        k = self.draw(n, self.Hkv) if k is None else k.astype(self.np_x)
        v = self.draw(n, self.Hkv) if v is None else v.astype(self.np_x)
        qd = self.batch.append(self.dev(q) if with_q else None, self.dev(k), self.dev(v),
                               theta=self.theta, q_start=self.starts(new), max_q=max(new))
        pos, qr, row = self.positions(new), [], 0
        for b, m in enumerate(new):
            kr = ref.rotate(k[row:row + m], pos[b], self.theta).astype(np.float32)
            self.k[b] = np.concatenate([self.k[b], ref.held(kr, self.kv)])
            self.v[b] = np.concatenate([self.v[b], ref.held(v[row:row + m], self.kv)])
            if with_q:
                qr.append(ref.rotate(q[row:row + m], pos[b], self.theta))
            row += m
        return qd, np.concatenate(qr) if with_q else None

    def expect(self, q, new, slopes=None, prefix=None, **opt):
        pos, out, row = self.positions(new), [], 0
        for b, m in enumerate(new):
            out.append(ref.attend(q[row:row + m], pos[b], self.k[b], self.v[b], slopes=slopes,
                                  prefix=prefix[b] if prefix is not None else 0, **opt))
            row += m
        return np.concatenate(out)


HEADS = {"qwen": (14, 2, 64), "llama": (4, 4, 128), "gqa": (8, 2, 128), "many": (20, 1, 64),
         "one": (2, 2, 64),
         "three": (6, 2, 64), "wide": (80, 1, 64), "wider": (130, 2, 128)}


# ---------------------------------------------------------------- append, read


@pytest.mark.parametrize("kv", ["f16", "q4"])
@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("heads", ["qwen", "gqa"])
def test_append_and_read_ragged(gpu, kv, x, heads):
    """Several appends of ragged lengths, blocks of 8 begun in one call and ended in another."""
    s = Setup(gpu, [60, 60, 60], HEADS[heads], kv, x, theta=1e6, seed=1)
    for new in ([3, 17, 0], [1, 1, 1], [8, 5, 16], [0, 13, 30]):
        qd, qr = s.append(new)
        # half a step: relative, and half of fp16's smallest step (2^-24) below 2^-14; twice
        # rounded (fp64 to fp32 to fp16), which adds 2^-24
        half, least = (2.0 ** -11, 2.0 ** -25) if x == "f16" else (2.0 ** -24, 2.0 ** -50)
        bound = half * np.abs(qr) * (1 + 2.0 ** -12) + least
        assert float((np.abs(qd.cpu().numpy().astype(np.float64) - qr) / bound).max()) <= 1
    k, v = s.batch.read(sum(s.len), q_start=s.starts(s.len), max_q=max(s.len))
    # the same values, bit for bit: the rotation is rounded once, and the codes are exact
    assert np.array_equal(v.cpu().numpy(), np.concatenate(s.v))
    assert np.array_equal(k.cpu().numpy(), np.concatenate(s.k))
    k16, _ = s.batch.read(sum(s.len), q_start=s.starts(s.len), max_q=max(s.len), dtype="f16")
    assert np.array_equal(k16.cpu().numpy(), np.concatenate(s.k).astype(np.float16))


@pytest.mark.parametrize("kv", ["f16", "q4"])
def test_append_step_far_positions(gpu, kv):
    """One token each, far out: angles of 65536 radians and more."""
    lens = [1, 65537, 100003, 16]
    s = Setup(gpu, [1, 1, 1, 1], (8, 2, 128), kv, theta=1e4, seed=2)
    ps = s.cache.page_size
    table = np.full((4, 100003 // ps + 1), -1, np.int32)
    for b, n in enumerate(lens):
        table[b, (n - 1) // ps] = b
    batch = s.cache.batch(s.dev(table), s.dev(np.array(lens, np.int32)))
    q, k, v = s.draw(4, 8), s.draw(4, 2), s.draw(4, 2)
    qd = batch.append(s.dev(q), s.dev(k), s.dev(v), theta=1e4)
    pos = np.array(lens) - 1
    qr = ref.rotate(q, pos, 1e4)
    assert np.abs(qd.cpu().numpy() - qr).max() <= 2.0 ** -24 * 8
    kd, vd = batch.read(4)
    assert np.array_equal(kd.cpu().numpy(),
                          ref.held(ref.rotate(k, pos, 1e4).astype(np.float32), kv))
    assert np.array_equal(vd.cpu().numpy(), ref.held(v, kv))


@pytest.mark.parametrize("x", ["f32", "f16"])
def test_append_strided_projection(gpu, x):
    """q, k and v as slices of one projection's rows, at an odd row stride."""
    s = Setup(gpu, [9, 9], (6, 2, 64), "q4", x, theta=1e4, seed=3)
    rows = s.rng.normal(size=(10, 10 * 64 + 3)).astype(s.np_x)
    d = s.dev(rows)
    part = lambda a, b: d[:, 1 + 64 * a:1 + 64 * b]  # noqa: E731
    s.lens.fill_(5)
    qd = s.batch.append(part(0, 6), part(6, 8), part(8, 10), theta=1e4)
    pos = np.tile(np.arange(5), 2)
    host = lambda a, b: rows[:, 1 + 64 * a:1 + 64 * b].reshape(10, b - a, 64)  # noqa: E731
    qr = ref.rotate(host(0, 6), pos, 1e4)
    assert rel_l2(qd.cpu().numpy(), qr) <= (2.0 ** -11 if x == "f16" else 2.0 ** -24)
    k, v = s.batch.read(10)
    assert np.array_equal(k.cpu().numpy(), ref.quantised(
        ref.rotate(host(6, 8), pos, 1e4).astype(np.float32)))
    assert np.array_equal(v.cpu().numpy(), ref.quantised(host(8, 10)))


def test_append_quantised_borders(gpu):
    """Groups of one value, ties between codes, ranges below a scale's smallest step, values past
    fp16, infinities and NaN: each group as the formulas say, the others untouched."""
    s = Setup(gpu, [8], (2, 2, 64), "q4", seed=4)
    v = s.rng.normal(size=(8, 2, 64)).astype(np.float32)
    v[0] = 3.25                                   # one value
    v[1, :, :32] = np.arange(32) / 2.0 - 4.0      # min -4, max 11.5: ties where exact
    v[2, :, 32:] = 1.0 + np.arange(32) * 2.0 ** -23
    v[3, 0, 5] = 1e6
    v[4, 1, 40] = np.inf
    v[5, 0, 0] = np.nan
    v[6] *= 1e-9
    v[7, :, :32] = np.float16(65504) * (np.arange(32) % 2 * 2 - 1)
    s.append([8], with_q=False, k=v[::-1], v=v)
    k, vv = s.batch.read(8)
    assert np.array_equal(vv.cpu().numpy(), ref.quantised(v), equal_nan=True)
    assert np.array_equal(k.cpu().numpy(), ref.quantised(v[::-1]), equal_nan=True)
    assert np.isnan(vv[5, 0, :32].cpu().numpy()).all()
    assert np.isfinite(vv[5, 0, 32:].cpu().numpy()).all()


@pytest.mark.parametrize("kv", ["f16", "q4"])
def test_append_leaves_the_rest(gpu, kv):
    """Rows behind the last sequence, pages of others and positions without a page stay as they
    were; lengths shorter than the tokens drop the first ones."""
    s = Setup(gpu, [40, 40], (4, 2, 64), kv, seed=5, theta=1e4)
    k0, v0 = s.cache.k.clone(), s.cache.v.clone()
    table = np.array([[1, 2, -1], [3, 10 ** 6, 4]], np.int32)
    lens = np.array([37, 3], np.int32)  # sequence 1: five tokens, three positions
    batch = s.cache.batch(s.dev(table), s.dev(lens))
    k, v, q = s.draw(15, 2), s.draw(15, 2), s.draw(15, 4)
    q_out = s.gpu.full((15, 4, 64), 7.0, device="cuda")
    start = s.gpu.tensor([0, 7, 12], dtype=s.gpu.int32, device="cuda")
    batch.append(s.dev(q), s.dev(k), s.dev(v), theta=1e4, q_start=start, max_q=7, q_out=q_out)
    assert (q_out[12:] == 7.0).all() and (q_out[7:9] == 7.0).all()
    pos = np.r_[30:37, 0:3]
    rows = np.r_[0:7, 9:12]
    assert rel_l2(q_out[s.dev(rows)].cpu().numpy(), ref.rotate(q[rows], pos, 1e4)) < 2.0 ** -23
    kd, vd = batch.read(15, q_start=start, max_q=7)
    want = ref.held(v, kv)
    got = vd.cpu().numpy()
    assert np.array_equal(got[:2], want[:2]) and np.array_equal(got[9:12], want[9:12])
    assert not got[2:7].any() and not got[7:9].any()  # page -1, negative positions
    for page in range(s.cache.n_pages):
        if page not in (2, 3):
            assert s.gpu.equal(s.cache.k[page], k0[page]) and s.gpu.equal(s.cache.v[page], v0[page])


# ---------------------------------------------------------------- attention, one token each


@pytest.mark.parametrize("kv", ["f16", "q4"])
@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("heads,lens,ps", [
    ("qwen", [1, 2, 31, 33, 577], 16),
    ("llama", [129, 64, 1, 300], 32),
    ("gqa", [1000, 15, 16, 17], 64),
    ("many", [70, 5], 16),
    ("three", [257], 128),
])
def test_attend_step(gpu, kv, x, heads, lens, ps):
    s = Setup(gpu, lens, HEADS[heads], kv, x, ps=ps, seed=6, theta=1e6)
    if max(lens) > 1:
        s.append([n - 1 for n in lens], with_q=False)
    one = [1] * len(lens)
    qd, _ = s.append(one)
    want = s.expect(qd.cpu().numpy(), one)
    for max_len in (0, max(lens)):
        got = s.batch.attend(qd, max_len=max_len)
        assert rel_l2(got.cpu().numpy(), want) <= tol(x)
    # a bound that is too small costs parallelism, not positions
    got = s.batch.attend(qd, max_len=1)
    assert rel_l2(got.cpu().numpy(), want) <= tol(x)


OPTIONS = [
    dict(cap=5.0),
    dict(window=1),
    dict(window=40),
    dict(slopes=True),
    dict(cap=20.0, window=100, slopes=True, prefix=True),
    dict(window=7, prefix=True),
]


def options(s, o):
    """(keyword arguments of attend, of expect)."""
    gpu, a, e = s.gpu, {}, {}
    if o.get("cap"):
        a["softcap"] = e["cap"] = o["cap"]
    if o.get("window"):
        a["window"] = e["window"] = o["window"]
    if o.get("slopes"):
        e["slopes"] = (2.0 ** -np.linspace(0.5, 6, s.Hq)).astype(np.float32)
        a["slopes"] = s.dev(e["slopes"])
    if o.get("prefix"):
        e["prefix"] = [(5, 0, 33, 10 ** 9)[b % 4] for b in range(len(s.len))]
        a["prefix"] = gpu.tensor(e["prefix"], dtype=gpu.int32, device="cuda")
    return a, e


@pytest.mark.parametrize("kv", ["f16", "q4"])
@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("o", OPTIONS)
def test_attend_step_options(gpu, kv, x, o):
    lens = [300, 41, 129, 90]
    s = Setup(gpu, lens, HEADS["gqa"], kv, x, ps=32, seed=7)
    s.append([n - 1 for n in lens], with_q=False)
    qd, _ = s.append([1] * 4)
    a, e = options(s, o)
    got = s.batch.attend(qd, max_len=300, **a).cpu().numpy()
    assert rel_l2(got, s.expect(qd.cpu().numpy(), [1] * 4, **e)) <= tol(x)


# ---------------------------------------------------------------- attention, many tokens


@pytest.mark.parametrize("kv", ["f16", "q4"])
@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("heads,old,new,ps", [
    ("qwen", [0, 100, 7], [65, 3, 1], 16),
    ("llama", [0, 50], [33, 64], 32),
    ("gqa", [200, 0, 0], [17, 129, 0], 64),
    ("many", [31], [2], 16),
    ("three", [5, 0, 64], [1, 40, 0], 16),
    ("gqa", [30, 1, 0], [2, 1, 2], 16),
    ("llama", [0, 333], [150, 70], 16),
    ("llama", [2000], [66], 64),           # few columns, many positions: split
    ("three", [1500, 0], [30, 25], 128),
    ("many", [700], [9], 32),
    ("one", [90, 0], [70, 200], 32),
])
def test_attend_tokens(gpu, kv, x, heads, old, new, ps):
    s = Setup(gpu, [a + b for a, b in zip(old, new)], HEADS[heads], kv, x, ps=ps, seed=8,
              theta=1e6)
    if max(old):
        s.append(old, with_q=False)
    qd, _ = s.append(new)
    got = s.batch.attend(qd, q_start=s.starts(new), max_q=max(new)).cpu().numpy()
    assert rel_l2(got, s.expect(qd.cpu().numpy(), new)) <= tol(x)


@pytest.mark.parametrize("kv", ["f16", "q4"])
@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("o", OPTIONS)
def test_attend_tokens_options(gpu, kv, x, o):
    old, new = [100, 0, 60, 3], [40, 50, 1, 70]
    s = Setup(gpu, [a + b for a, b in zip(old, new)], HEADS["three"], kv, x, ps=16, seed=9)
    s.append(old, with_q=False)
    qd, _ = s.append(new)
    a, e = options(s, o)
    got = s.batch.attend(qd, q_start=s.starts(new), max_q=70, **a).cpu().numpy()
    assert rel_l2(got, s.expect(qd.cpu().numpy(), new, **e)) <= tol(x)


@pytest.mark.parametrize("kv", ["f16", "q4"])
@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("o", OPTIONS)
def test_attend_tokens_options_long(gpu, kv, x, o):
    """The same where positions are split and most lie left of the window."""
    s = Setup(gpu, [1700], HEADS["gqa"], kv, x, ps=32, seed=21)
    s.append([1660], with_q=False)
    qd, _ = s.append([40])
    a, e = options(s, o)
    got = s.batch.attend(qd, max_len=1700, **a).cpu().numpy()
    assert rel_l2(got, s.expect(qd.cpu().numpy(), [40], **e)) <= tol(x)


@pytest.mark.parametrize("kv", ["f16", "q4"])
@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("tokens", [1, 11, 40])
def test_attend_uniform_tokens_and_stride(gpu, kv, x, tokens):
    """As many tokens of each sequence, without q_start; queries as slices of wider rows, at odd
    offsets, and the output at one too."""
    s = Setup(gpu, [80, 80], HEADS["three"], kv, x, seed=10)
    s.append([20, 9], with_q=False)
    qd, _ = s.append([tokens, tokens])
    n = 2 * tokens
    wide = s.gpu.zeros((n, 6 * 64 + 5), device="cuda", dtype=qd.dtype)
    wide[:, 5:] = qd.reshape(n, -1)
    room = s.gpu.full((n * 6 * 64 + 2,), 7.0, device="cuda", dtype=qd.dtype)
    out = room[1:-1].view(n, 6, 64)
    s.batch.attend(wide[:, 5:], out=out)
    assert room[0] == 7.0 and room[-1] == 7.0
    assert rel_l2(out.cpu().numpy(), s.expect(qd.cpu().numpy(), [tokens] * 2)) <= tol(x)


def test_python_refusals(gpu):
    """What the Python entry points refuse before a launch."""
    from cortexsdr_amd import _lib
    from cortexsdr_amd.logprobs import token_logprobs
    from cortexsdr_amd.paged import PagedCache

    s = Setup(gpu, [16], HEADS["three"], "f16", seed=22)
    s.append([4], with_q=False)
    b, q = s.batch, gpu.zeros(1, 6, 64, device="cuda")
    k = gpu.zeros(1, 2, 64, device="cuda")
    two = gpu.zeros(2, dtype=gpu.int32, device="cuda")
    for call in (
        lambda: b.attend(q.double()), lambda: b.attend(q.cpu()), lambda: b.attend(q[:, :, ::2]),
        lambda: b.attend(gpu.zeros(1, 6 * 64 + 1, device="cuda")),
        lambda: b.attend(q.expand(3, 6, 64), q_start=two, max_q=3),  # rows that overlap
        lambda: b.attend(q, q_start=two), lambda: b.attend(q, q_start=two.long(), max_q=1),
        lambda: b.attend(q, slopes=gpu.zeros(5, device="cuda")),
        lambda: b.attend(q, prefix=two), lambda: b.attend(q, out=q.half()),
        lambda: b.append(q, k, k.half()), lambda: b.append(q, k[:, :1], k),
        lambda: b.append(None, k, k, q_out=q), lambda: b.append(q, k, k, q_out=q[:, :3]),
        lambda: b.read(1, dtype="bf16"),
        lambda: PagedCache(4, 24, 2, 64), lambda: PagedCache(0, 16, 2, 64),
        lambda: PagedCache(4, 16, 2, 64, "f32"), lambda: PagedCache(4, 16, 2, 64, k=q, v=q),
        lambda: s.cache.batch(two, two), lambda: s.cache.batch(two.view(1, 2).long(), two[:1]),
        lambda: s.cache.batch(two.view(2, 1), two[:1]),
        lambda: token_logprobs(q), lambda: token_logprobs(gpu.zeros(4, 8, device="cuda")[:, ::2]),
        lambda: token_logprobs(gpu.zeros(1, 8, device="cuda").expand(4, 8)),
        lambda: token_logprobs(gpu.zeros(4, 8, device="cuda"), two),
        lambda: b.attend(q, workspace=two[:1].expand(1 << 20)),
        lambda: token_logprobs(gpu.zeros(4, 8, device="cuda"), workspace=two[:1].expand(1 << 20)),
    ):
        with pytest.raises(ValueError):
            call()
    for call in (
        lambda: b.attend(gpu.zeros(1, 5, 64, device="cuda")),  # 5 heads over 2
        lambda: b.attend(q, window=-1), lambda: b.attend(q, softcap=float("nan")),
        lambda: b.attend(q, workspace=gpu.zeros(4, device="cuda")), lambda: b.attend(q, out=q),
        lambda: token_logprobs(gpu.zeros(4, 8, device="cuda"), top_n=65),
        lambda: token_logprobs(gpu.zeros(4, 8, device="cuda"), workspace=q[0, 0, :4]),
    ):
        with pytest.raises(_lib.CsdrError):
            call()


def test_cache_of_another_device(gpu):
    """The current device is another than the cache's, and the call's tensors are on it."""
    from cortexsdr_amd.paged import PagedBatch

    s = Setup(gpu, [16], HEADS["three"], "f16", seed=24)
    s.append([4], with_q=False)
    s.batch._device += 1  # as if
    q, k = gpu.zeros(1, 6, 64, device="cuda"), gpu.zeros(1, 2, 64, device="cuda")
    for call in (lambda: s.batch.append(q, k, k), lambda: s.batch.attend(q),
                 lambda: s.batch.read(1)):
        with pytest.raises(ValueError, match="current device"):
            call()
    s.batch._device -= 1

    class Elsewhere(gpu.cuda.Stream):
        device_index = 1

    for call in (lambda: s.batch.append(q, k, k, q_out=q, stream=Elsewhere()),
                 lambda: s.batch.attend(q, out=q.clone(), max_len=1, stream=Elsewhere())):
        with pytest.raises(ValueError, match="stream"):
            call()
    pools, s.cache.k = s.cache.k, s.cache.k.cpu()
    with pytest.raises(ValueError, match="current device"):
        PagedBatch(s.cache, s.table, s.lens)
    s.cache.k = pools


def test_bounds_past_an_int(gpu):
    """A window, a length bound and a most of tokens past 2^31 bound nothing."""
    s = Setup(gpu, [300], HEADS["three"], "f16", seed=23)
    qd, _ = s.append([300])
    want = s.batch.attend(qd)
    for far in (2 ** 31, 2 ** 32 + 3):
        assert gpu.equal(s.batch.attend(qd, window=far), want)
        assert gpu.equal(s.batch.attend(qd, max_len=far), want)
        assert gpu.equal(s.batch.attend(qd, q_start=s.starts([300]), max_q=far), want)


# ---------------------------------------------------------------- what is not seen


@pytest.mark.parametrize("kv", ["f16", "q4"])
@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_unseen_values_have_no_influence(gpu, kv, x, what):
    """NaN and infinities in keys and values behind a token's own position, left of its window and
    in unwritten pages; a token that sees one is not finite."""
    s = Setup(gpu, [80, 80], HEADS["three"], kv, x, seed=11)
    k, v = s.draw(100, 2), s.draw(100, 2)
    for i in (10, 70):                   # sequence 0 position 10; sequence 1 position 20
        v[i, 0, 3] = what
    k[75, 1, 9] = what                   # sequence 1 position 25
    s.append([50, 50], with_q=False, k=k, v=v)
    qd, _ = s.append([30, 30])
    want = s.expect(qd.cpu().numpy(), [30, 30], window=45)
    got = s.batch.attend(qd, q_start=s.starts([30, 30]), max_q=30, window=45).cpu().numpy()
    fine = np.isfinite(want)
    assert fine.any() and not fine.all()
    assert np.isfinite(got[fine]).all() and not np.isfinite(got[~fine]).any()
    assert rel_l2(got[fine], want[fine]) <= tol(x)


@pytest.mark.parametrize("kv", ["f16", "q4"])
@pytest.mark.parametrize("what", [np.nan, np.inf])
def test_causal_rows_before_a_bad_value(gpu, kv, what):
    """A value that is not finite among the prompt's own tokens: rows before it are untouched."""
    s = Setup(gpu, [70], HEADS["gqa"], kv, seed=12)
    k, v = s.draw(70, 2), s.draw(70, 2)
    v[37, 1, 100] = what
    qd, _ = s.append([70], k=k, v=v)
    want = s.expect(qd.cpu().numpy(), [70])
    got = s.batch.attend(qd).cpu().numpy()
    fine = np.isfinite(want)
    assert np.isfinite(got[:37]).all() and not fine[37:].all()
    assert np.isfinite(got[fine]).all() and not np.isfinite(got[~fine]).any()
    assert rel_l2(got[fine], want[fine]) <= TOL32


@pytest.mark.parametrize("kv", ["f16", "q4"])
@pytest.mark.parametrize("tokens", [1, 5])
def test_rows_that_see_nothing(gpu, kv, tokens):
    """Empty sequences, tokens without a position, sequences whose pages are missing: zeros. Rows
    behind the last sequence: as they were."""
    s = Setup(gpu, [40, 40, 40, 40], HEADS["three"], kv, seed=13)
    s.append([20, 9, 30, 1], with_q=False)
    lens = s.gpu.tensor([20, 0, 30, 1], dtype=s.gpu.int32, device="cuda")
    table = s.table.clone()
    table[2, 0], table[2, 1] = -1, s.cache.n_pages
    batch = s.cache.batch(table, lens)
    n = 4 * tokens
    q = s.dev(s.draw(n + 2, 6))
    out = s.gpu.full((n + 2, 6, 64), 7.0, device="cuda")
    start = s.gpu.arange(0, n + 1, tokens, dtype=s.gpu.int32, device="cuda")
    batch.attend(q, q_start=start, max_q=tokens, out=out)
    o = out.cpu().numpy()
    assert (o[n:] == 7.0).all()
    assert not o[tokens:3 * tokens].any()
    assert not o[3 * tokens:n - 1].any() and o[n - 1].any()
    want = ref.attend(q[:tokens].cpu().numpy(), np.arange(20 - tokens, 20), s.k[0], s.v[0])
    assert rel_l2(o[:tokens], want) <= TOL32


def test_bad_starts_stay_in_bounds(gpu):
    """Row numbers that run backwards or past the tokens are clamped to them."""
    s = Setup(gpu, [40, 40, 40], HEADS["three"], "f16", seed=14)
    s.append([20, 20, 20], with_q=False)
    q = s.dev(s.draw(6, 6))
    for starts in ([0, 100, 100, 100], [-5, 3, 2, 6], [4, -1, 9, 1]):
        start = s.gpu.tensor(starts, dtype=s.gpu.int32, device="cuda")
        out = s.gpu.full((6, 6, 64), 7.0, device="cuda")
        s.batch.attend(q, q_start=start, max_q=100, out=out)
        s.batch.append(None, q[:, :2], q[:, 2:4], q_start=start, max_q=100)
        s.batch.read(6, q_start=start, max_q=100)
        assert np.isfinite(out.cpu().numpy()).all()


# ---------------------------------------------------------------- as they are used together


@pytest.mark.parametrize("kv", ["f16", "q4"])
def test_serving_loop(gpu, kv):
    """A prompt in two chunks, then single tokens, then a token of one sequence beside a new
    prompt of another: each call's attention against the whole history; then the scores of the
    last rows."""
    from cortexsdr_amd.logprobs import token_logprobs

    s = Setup(gpu, [200, 200], HEADS["qwen"], kv, ps=32, seed=15, theta=1e6)
    for new in ([40, 25], [30, 2], [1, 1], [1, 1], [1, 60], [2, 3]):
        qd, _ = s.append(new)
        got = s.batch.attend(qd, q_start=s.starts(new), max_q=max(new), max_len=200)
        want = s.expect(qd.cpu().numpy(), new)
        assert rel_l2(got.cpu().numpy(), want) <= TOL32
    w = s.rng.normal(size=(14 * 64, 999)).astype(np.float32) / 30
    logits = got.reshape(5, -1) @ s.dev(w)
    r = token_logprobs(logits, s.gpu.arange(5, dtype=s.gpu.int32, device="cuda"), top_n=3)
    y = logits.double().cpu().numpy()
    lp = y - np.log(np.exp(y - y.max(1, keepdims=True)).sum(1, keepdims=True)) - \
        y.max(1, keepdims=True)
    assert np.abs(r.logprobs.cpu().numpy() - lp[np.arange(5), np.arange(5)]).max() < 1e-5
    assert np.array_equal(r.top_ids.cpu().numpy(), np.argsort(-y, 1, kind="stable")[:, :3])


@pytest.mark.parametrize("kv", ["f16", "q4"])
def test_captured_step(gpu, kv):
    """A step captured once and replayed while lengths advance, on a stream of its own, two graphs
    in turn, with eager calls between; each replay against the formulas."""
    s = Setup(gpu, [90, 90], HEADS["gqa"], kv, seed=16, theta=1e6)
    s.append([33, 20], with_q=False)
    q, k, v = (gpu.zeros((2, h, 128), device="cuda") for h in (8, 2, 2))

    def step():
        return s.batch.attend(s.batch.append(q, k, v, theta=1e6), max_len=90)

    side = gpu.cuda.Stream()
    side.wait_stream(gpu.cuda.current_stream())
    with gpu.cuda.stream(side):
        s.lens.copy_(gpu.tensor([34, 21], dtype=gpu.int32))
        step()
    gpu.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = gpu.cuda.CUDAGraph()
        with gpu.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for i in range(6):
        s.len = [n + 1 for n in s.len]
        s.lens.copy_(gpu.tensor(s.len, dtype=gpu.int32))
        qn, kn, vn = s.draw(2, 8, 1.5), s.draw(2, 2), s.draw(2, 2)
        for d, h in ((q, qn), (k, kn), (v, vn)):
            d.copy_(s.dev(h))
        g, out = graphs[i % 2]
        g.replay()
        pos = np.array(s.len) - 1
        kr = ref.held(ref.rotate(kn, pos, 1e6).astype(np.float32), kv)
        for b in range(2):
            s.k[b] = np.concatenate([s.k[b], kr[b:b + 1]])
            s.v[b] = np.concatenate([s.v[b], ref.held(vn[b:b + 1], kv)])
        want = s.expect(ref.rotate(qn, pos, 1e6), [1, 1])
        assert rel_l2(out.cpu().numpy(), want) <= TOL32
        eager = s.batch.attend(s.dev(ref.rotate(qn, pos, 1e6).astype(np.float32)))
        assert rel_l2(eager.cpu().numpy(), want) <= TOL32


def test_calls_at_once_on_two_streams(gpu):
    """Two batches over one cache, each on its own stream with its own workspace."""
    a = Setup(gpu, [700, 300], HEADS["gqa"], "f16", seed=17)
    b = Setup(gpu, [500], HEADS["qwen"], "q4", seed=18)
    jobs = []
    for s, n in ((a, [699, 299]), (b, [499])):
        s.append(n, with_q=False)
        qd, _ = s.append([1] * len(n))
        jobs.append((s, qd, s.expect(qd.cpu().numpy(), [1] * len(n)), gpu.cuda.Stream()))
    gpu.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, (s, qd, _, st) in enumerate(jobs):
            outs[i].append(s.batch.attend(qd, stream=st))
    gpu.cuda.synchronize()
    for i, (_, _, want, _) in enumerate(jobs):
        for o in outs[i]:
            assert rel_l2(o.cpu().numpy(), want) <= TOL32


def test_shared_prefix_pages(gpu):
    """Two sequences whose first pages are the same."""
    s = Setup(gpu, [64], HEADS["three"], "q4", seed=19)
    s.append([48], with_q=False)
    table = gpu.cat([s.table, s.table])
    table[1, 3] = next(p for p in range(s.cache.n_pages) if p not in s.table.cpu().tolist()[0])
    lens = gpu.tensor([50, 49], dtype=gpu.int32, device="cuda")
    batch = s.cache.batch(table, lens)
    k, v, q = s.draw(3, 2), s.draw(3, 2), s.draw(3, 6)
    start = gpu.tensor([0, 2, 3], dtype=gpu.int32, device="cuda")
    batch.append(None, s.dev(k), s.dev(v), q_start=start, max_q=2)
    out = batch.attend(s.dev(q), q_start=start, max_q=2).cpu().numpy()
    kh, vh = ref.held(k, "q4"), ref.held(v, "q4")
    for rows, pos in ((slice(0, 2), [48, 49]), (slice(2, 3), [48])):
        want = ref.attend(q[rows], pos, np.concatenate([s.k[0], kh[rows]]),
                          np.concatenate([s.v[0], vh[rows]]))
        assert rel_l2(out[rows], want) <= TOL32


def test_large_queries_and_keys(gpu):
    """Magnitudes at the ends of fp16 and beyond it in q: the pairs of fp16 follow the row's
    size."""
    for sigma in (1e-12, 1e-3, 3e4, 1e9):
        s = Setup(gpu, [60], HEADS["three"], "f16", seed=20)
        s.append([59], with_q=False)
        s.append([1], with_q=False)
        q = (s.rng.normal(size=(1, 6, 64)) * sigma).astype(np.float32)
        got = s.batch.attend(s.dev(q), scale=float(1 / sigma / 8)).cpu().numpy()
        want = ref.attend(q, [59], s.k[0], s.v[0], scale=float(np.float32(1 / sigma / 8)))
        assert rel_l2(got, want) <= TOL32, sigma


@pytest.mark.parametrize("kv", ["f16", "q4"])
@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("heads", ["wide", "wider"])
def test_step_of_many_heads(gpu, kv, x, heads):
    """More than 64 query heads to a KV head: single tokens, in the form for prompts."""
    s = Setup(gpu, [700, 1, 40], HEADS[heads], kv, x, ps=32, seed=41)
    s.append([699, 0, 39], with_q=False)
    qd, _ = s.append([1, 1, 1])
    want = s.expect(qd.cpu().numpy(), [1, 1, 1])
    assert rel_l2(s.batch.attend(qd).cpu().numpy(), want) <= tol(x)
    assert rel_l2(s.batch.attend(qd, max_len=700).cpu().numpy(), want) <= tol(x)


@pytest.mark.parametrize("kv", ["f16", "q4"])
@pytest.mark.parametrize("x", ["f32", "f16"])
def test_largest_pages(gpu, kv, x):
    s = Setup(gpu, [4200, 17], HEADS["three"], kv, x, ps=4096, seed=42, theta=1e4)
    s.append([4100, 10], with_q=False)
    for new in ([1, 1], [99, 6]):
        qd, _ = s.append(new)
        got = s.batch.attend(qd, q_start=s.starts(new), max_q=max(new))
        assert rel_l2(got.cpu().numpy(), s.expect(qd.cpu().numpy(), new)) <= tol(x)


@pytest.mark.parametrize("kv", ["f16", "q4"])
@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("scale", [-0.125, 1e-3])
def test_given_scale(gpu, kv, x, tokens, scale):
    s = Setup(gpu, [200], HEADS["three"], kv, x, seed=43)
    s.append([150], with_q=False)
    qd, _ = s.append([tokens])
    for o in ({}, dict(cap=3.0)):
        want = s.expect(qd.cpu().numpy(), [tokens], scale=scale, **o)
        got = s.batch.attend(qd, scale=scale, softcap=o.get("cap", 0.0))
        assert rel_l2(got.cpu().numpy(), want) <= tol(x)


@pytest.mark.parametrize("kv", ["f16", "q4"])
def test_a_page_twice(gpu, kv):
    """One page at two places of a row, and in two rows: read at each."""
    s = Setup(gpu, [64, 64], HEADS["three"], kv, ps=16, seed=44)
    s.append([64, 64], with_q=False)
    s.table[:, 2] = s.table[0, 0]
    for b in range(2):
        s.k[b][32:48], s.v[b][32:48] = s.k[0][:16], s.v[0][:16]
    for tokens in (1, 30):
        q = s.draw(2 * tokens, 6, 1.5)
        got = s.batch.attend(s.dev(q))
        assert rel_l2(got.cpu().numpy(), s.expect(q, [tokens] * 2)) <= TOL32


@pytest.mark.parametrize("kv", ["f16", "q4"])
def test_given_pools_queries_in_place_other_stream(gpu, kv):
    """Pools of the caller's, rotation over the queries themselves, every call on a given stream."""
    from cortexsdr_amd.paged import PagedCache

    s = Setup(gpu, [90, 50], HEADS["gqa"], kv, seed=45, theta=1e5)
    s.cache = PagedCache(s.cache.n_pages, 16, 2, 128, kv, k=s.cache.k.view(-1), v=s.cache.v)
    s.batch = s.cache.batch(s.table, s.lens)
    s.append([50, 10], with_q=False)
    s.len = [90, 50]
    s.lens.copy_(gpu.tensor(s.len, dtype=gpu.int32))
    q, k, v = s.draw(80, 8), s.draw(80, 2), s.draw(80, 2)
    qd, kd, vd = s.dev(q), s.dev(k), s.dev(v)
    side = gpu.cuda.Stream()
    side.wait_stream(gpu.cuda.current_stream())
    assert s.batch.append(qd, kd, vd, theta=1e5, q_out=qd, stream=side) is qd
    got = s.batch.attend(qd, stream=side)
    rk, rv = s.batch.read(80, stream=side)
    gpu.cuda.current_stream().wait_stream(side)
    pos = s.positions([40, 40])
    qr = np.concatenate([ref.rotate(q[:40], pos[0], 1e5), ref.rotate(q[40:], pos[1], 1e5)])
    # half a step of fp32, and the rounding of the fp64 pair before it
    assert float(np.abs(qd.cpu().numpy() - qr).max()) <= 2.0 ** -24 * 1.01 * np.abs(qr).max()
    for b in range(2):
        kr = ref.rotate(k[40 * b:40 * b + 40], pos[b], 1e5).astype(np.float32)
        s.k[b] = np.concatenate([s.k[b], ref.held(kr, kv)])
        s.v[b] = np.concatenate([s.v[b], ref.held(v[40 * b:40 * b + 40], kv)])
    last = [np.concatenate([a[0][-40:], a[1][-40:]]) for a in (s.k, s.v)]
    assert rel_l2(rk.cpu().numpy(), last[0]) <= TOL32
    assert rel_l2(rv.cpu().numpy(), last[1]) <= TOL32
    assert rel_l2(got.cpu().numpy(), s.expect(qr, [40, 40])) <= TOL32
