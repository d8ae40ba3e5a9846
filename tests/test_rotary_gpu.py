"""csdr_rotary against the formulas in fp64, and against the cache's own rotation."""
import math

import numpy as np
import pytest

import q8_ref

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -11
# what sine and cosine may be off: the turn rounded to fp32 (at most a half: 2^-26 turns, 2 pi radians each),
# two steps of a value up to 1 for sincospif, the product with the magnitude
TRIG = 2 * math.pi * 2.0 ** -26 + 2 * 2.0 ** -24 + U32


def check(y, x, positions, freqs, layout, magnitude=1.0):
    want = q8_ref.rotary(x, positions, freqs, layout, magnitude)
    d = 2 * len(freqs)
    y = y.cpu().numpy()
    np.testing.assert_array_equal(y[..., d:], x[..., d:])
    xd = np.abs(x[..., :d].astype(np.float64))
    if layout == "adjacent":
        pair = np.repeat(xd[..., 0::2] + xd[..., 1::2], 2, -1)
    else:
        pair = np.tile(xd[..., :d // 2] + xd[..., d // 2:], 2)
    half = y.dtype == np.float16
    # two products and their sum in fp32, one rounding to the type
    tol = abs(magnitude) * pair * (TRIG + 2 * U32) * 1.01
    tol = tol + (U16 if half else 0) * np.abs(want[..., :d]) * 1.01 + (2.0 ** -25 if half else 2.0 ** -149)
    err = np.abs(y[..., :d] - want[..., :d])
    assert (err <= tol).all(), np.max(err / tol)


CASES = [
    # tokens, query heads, key heads, head_dim, dims
    (1, 14, 2, 64, 64), (1, 1, 0, 2, 2), (3, 4, 2, 64, 32), (5, 32, 8, 128, 128), (2, 3, 1, 96, 96),
    (7, 5, 3, 80, 20), (4, 2, 2, 33, 6), (3, 2, 1, 47, 46), (600, 32, 32, 128, 32), (1100, 14, 2, 64, 64),
    (2, 3, 2, 1024, 1024), (3, 1, 1, 256, 16), (5, 2, 2, 72, 48), (5, 2, 2, 64, 60),
    # several tokens to a workgroup, the last one's fewer
    (1025, 3, 1, 64, 64), (3001, 1, 0, 64, 32), (2050, 2, 1, 33, 6), (1031, 1, 1, 16, 16), (5000, 1, 0, 2, 2),
]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("layout", ["adjacent", "halves"])
@pytest.mark.parametrize("n,hq,hk,hd,dims", CASES)
def test_rotary(gpu, n, hq, hk, hd, dims, layout, dtype):
    from cortexsdr_amd.rotary import Rotary, frequencies

    torch = gpu
    r = np.random.default_rng(n + hd)
    x = r.standard_normal((n, hq + 2 * hk, hd)).astype(np.float32 if dtype == "f32" else np.float16)
    pos = r.integers(0, 1 << 20, n).astype(np.int32)
    pos[0] = 0 if n > 1 else pos[0]
    rot = Rotary(hd, theta=5e5, dims=dims, layout=layout, magnitude=1.2)
    f = frequencies(dims, 5e5)
    d, p = torch.from_numpy(x).cuda(), torch.from_numpy(pos).cuda()
    q, k = d[:, :hq], d[:, hq:hq + hk]
    if hk == 0:
        check(rot.apply(q, p), x[:, :hq], pos, f, layout, 1.2)
        return
    qo, ko = rot.apply(q, p, k=k)
    check(qo, x[:, :hq], pos, f, layout, 1.2)
    check(ko, x[:, hq:hq + hk], pos, f, layout, 1.2)
    assert torch.equal(rot.apply(q, p), qo) and torch.equal(rot.apply(k, p), ko)
    # in place in the projection's output: values are not touched
    rot.apply(q, p, k=k, q_out=q, k_out=k)
    assert torch.equal(q, qo) and torch.equal(k, ko)
    assert torch.equal(d[:, hq + hk:].cpu(), torch.from_numpy(x[:, hq + hk:]))


@pytest.mark.parametrize("layout", ["adjacent", "halves"])
def test_padding_among_many(gpu, layout):
    """Rows without a token between others of one workgroup."""
    from cortexsdr_amd.rotary import Rotary, frequencies

    torch = gpu
    r = np.random.default_rng(8)
    x = r.standard_normal((1500, 2, 64)).astype(np.float32)
    pos = r.integers(-3, 5000, 1500).astype(np.int32)
    pos[r.random(1500) < 0.3] = -1
    out = torch.full((1500, 2, 64), 9.0, device="cuda")
    Rotary(64, layout=layout).apply(torch.from_numpy(x).cuda(), torch.from_numpy(pos).cuda(), q_out=out)
    none = torch.from_numpy(pos < 0).cuda()
    assert (out[none] == 9).all()
    check(out[~none], x[pos >= 0], pos[pos >= 0], frequencies(64, 1e6), layout)


@pytest.mark.parametrize("hd,dims", [(64, 64), (70, 50)])
def test_no_tokens_and_padding(gpu, hd, dims):
    """Rows with a negative position are left as they were."""
    from cortexsdr_amd.rotary import Rotary, frequencies

    torch = gpu
    x = np.random.default_rng(1).standard_normal((6, 3, hd)).astype(np.float32)
    pos = np.array([5, -1, 7, -2 ** 31, 0, 2 ** 31 - 1], np.int32)
    rot = Rotary(hd, dims=dims, layout="halves")
    out = torch.full((6, 3, hd), 9.0, device="cuda")
    rot.apply(torch.from_numpy(x).cuda(), torch.from_numpy(pos).cuda(), q_out=out)
    assert (out[1] == 9).all() and (out[3] == 9).all()
    keep = [0, 2, 4]
    check(out[keep], x[keep], pos[keep], frequencies(dims, 1e6), "halves")
    # the farthest position: 2^31 turns of fp64 leave 2^-23 of a turn
    far = q8_ref.rotary(x[5:], pos[5:], frequencies(dims, 1e6), "halves")
    assert np.abs(out[5].cpu().numpy() - far[0]).max() < 2 * np.abs(x).max() * (2 * math.pi * 2.0 ** -21 + TRIG)
    e = torch.empty((0, 3, hd), device="cuda")
    assert rot.apply(e, torch.empty(0, dtype=torch.int32, device="cuda")).shape == (0, 3, hd)


def test_far(gpu):
    """Tokens more than 2^32 bytes apart."""
    from cortexsdr_amd.rotary import Rotary, frequencies

    torch = gpu
    buf = torch.empty((1 << 32) + 64, dtype=torch.float16, device="cuda")
    x = buf.as_strided((3, 1, 64), (1 << 31, 64, 1))
    h = np.random.default_rng(4).standard_normal((3, 1, 64)).astype(np.float16)
    x.copy_(torch.from_numpy(h).cuda())
    pos = np.array([3, 70000, 131071], np.int32)
    p, rot = torch.from_numpy(pos).cuda(), Rotary(64, layout="halves")
    check(rot.apply(x, p), h, pos, frequencies(64, 1e6), "halves")
    rot.apply(x, p, q_out=x)
    check(x, h, pos, frequencies(64, 1e6), "halves")
    del buf, x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("kv", ["f16", "q4"])
def test_like_the_caches_own(gpu, kv, dtype):
    """Keys turned here and appended as they are attend as keys that the append turns."""
    from cortexsdr_amd.paged import PagedCache
    from cortexsdr_amd.rotary import Rotary

    torch = gpu
    g = torch.Generator(device="cuda").manual_seed(3)
    B, T, hq, hk, hd = 3, 7, 8, 2, 64
    x = torch.randn(B * T, hq + 2 * hk, hd, generator=g, device="cuda")
    x = x.half() if dtype == "f16" else x
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    table = torch.arange(B * 2, dtype=torch.int32, device="cuda").reshape(B, 2)
    lens = torch.full((B,), 20, dtype=torch.int32, device="cuda")
    pos = torch.arange(13, 20, dtype=torch.int32, device="cuda").repeat(B)
    outs = []
    for own in (True, False):
        b = PagedCache(B * 2, 16, hk, hd, kv).batch(table, lens)
        if own:
            turned = b.append(q, k, v, theta=1e6)
        else:
            turned, keys = Rotary(hd, theta=1e6).apply(q, pos, k=k)
            b.append(None, keys, v)
        outs.append((turned.float(), b.read(B * T)[0]))
    # fp16: both round once, so they differ by a step at most; 4 bits: by a code at most, a fifteenth of a
    # group's range, which 32 unit normal values keep below 8
    step = 2 * U16 if dtype == "f16" else 4 * TRIG
    (q0, k0), (q1, k1) = outs
    big = 2.0 ** 3  # larger than any pair's length here
    assert q0.abs().max() < big and (q0 - q1).abs().max() <= step * big
    assert (k0 - k1).abs().max() <= (step + 2 * U16) * big + (8 / 15 if kv == "q4" else 0)


def test_python_refusals(gpu):
    from cortexsdr_amd.rotary import Rotary

    torch = gpu
    rot = Rotary(64)
    q, p = torch.randn(4, 2, 64, device="cuda"), torch.arange(4, dtype=torch.int32, device="cuda")
    bad = [
        lambda: Rotary(64, dims=63), lambda: Rotary(64, dims=66), lambda: Rotary(2048), lambda: Rotary(0),
        lambda: Rotary(64, layout="other"), lambda: Rotary(64, freqs=[1.0] * 31),
        lambda: Rotary(64, freqs=[math.nan] * 32), lambda: rot.apply(q[:, :, :32], p),
        lambda: rot.apply(q, p.long()), lambda: rot.apply(q, p[:3]), lambda: rot.apply(q.double(), p),
        lambda: rot.apply(q, p, k=q.half()), lambda: rot.apply(q, p, k=q[:3]), lambda: rot.apply(q, p, k_out=q),
        lambda: rot.apply(q, p, q_out=torch.empty(4, 3, 64, device="cuda")),
        lambda: rot.apply(q[:1].expand(4, 2, 64), p), lambda: rot.apply(q.transpose(1, 2), p),
        lambda: rot.apply(q.cpu(), p), lambda: rot.apply(q.flatten(1), p),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(RuntimeError):
        Rotary(64, magnitude=math.inf).apply(q, p)
