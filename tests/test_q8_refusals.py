"""What the 8-bit rows' calls and csdr_rotary refuse, without a GPU: every refusal comes before a launch,
with a status and a message. And the scaled frequencies."""
import math

import pytest

from cortexsdr_amd import _lib
from cortexsdr_amd.rotary import frequencies

INVALID, UNSUPPORTED = -1, -6
P = 4096  # aligned addresses that no refused call reads
OUT, OTHER, K, KO = 2 * P, 3 * P, 4 * P, 5 * P


def refused(rc, status):
    assert rc == status
    assert _lib.load().csdr_last_error()


def test_pitch():
    f = _lib.load().csdr_q8_pitch
    assert [f(n) for n in (1, 127, 128, 129, 4096, 131071)] == [128, 128, 128, 256, 4096, 131072]
    assert [f(n) for n in (0, -1, 131072, 2 ** 31 - 1)] == [0] * 4


QUANTIZE = dict(x=P, gate=None, dtype=0, rows=2, n=100, xs=0, gs=0, codes=OUT, scales=P)


@pytest.mark.parametrize("over,status", [
    (dict(x=None), INVALID), (dict(codes=None), INVALID), (dict(scales=None), INVALID),
    (dict(dtype=2), INVALID), (dict(dtype=-1), INVALID), (dict(rows=0), INVALID),
    (dict(rows=-1), INVALID), (dict(rows=1 << 22), INVALID), (dict(n=0), INVALID),
    (dict(n=-5), INVALID), (dict(n=131072), UNSUPPORTED), (dict(xs=99), INVALID),
    (dict(xs=-100), INVALID), (dict(gate=P, gs=99), INVALID), (dict(codes=OUT + 8), INVALID),
    (dict(codes=P), INVALID), (dict(gate=OUT), INVALID),
])
def test_quantize(over, status):
    a = {**QUANTIZE, **over}
    refused(_lib.load().csdr_q8_quantize(a["x"], a["gate"], a["dtype"], a["rows"], a["n"], a["xs"],
                                         a["gs"], a["codes"], a["scales"], None), status)


@pytest.mark.parametrize("over,status", [
    (dict(codes=None), INVALID), (dict(scales=None), INVALID), (dict(out=None), INVALID),
    (dict(dtype=2), INVALID), (dict(rows=0), INVALID), (dict(rows=1 << 22), INVALID),
    (dict(n=0), INVALID), (dict(n=131072), UNSUPPORTED), (dict(codes=P + 4), INVALID),
    (dict(out=P), INVALID), (dict(rows=(1 << 22) - 1, n=131071), INVALID),  # more workgroups than a launch may have
])
def test_dequantize(over, status):
    a = {**dict(codes=P, scales=P, rows=2, n=100, out=OUT, dtype=0), **over}
    refused(_lib.load().csdr_q8_dequantize(a["codes"], a["scales"], a["rows"], a["n"], a["out"],
                                           a["dtype"], None), status)


NORM = dict(x=P, dtype=0, xs=0, res=K, rdt=0, rs=0, rout=OUT, w=P, eps=1e-5, rows=2, n=100, y=None,
            codes=OTHER, scales=KO)


@pytest.mark.parametrize("over,status", [
    (dict(x=None), INVALID), (dict(w=None), INVALID), (dict(codes=None), INVALID),
    (dict(scales=None), INVALID), (dict(codes=None, scales=None), INVALID), (dict(res=None), INVALID),
    (dict(rout=None), INVALID), (dict(dtype=2), INVALID), (dict(rdt=2), INVALID),
    (dict(rows=0), INVALID), (dict(rows=1 << 22), INVALID), (dict(n=0), INVALID),
    (dict(n=131072), UNSUPPORTED), (dict(eps=-1.0), INVALID), (dict(eps=math.nan), INVALID),
    (dict(eps=math.inf), INVALID), (dict(xs=99), INVALID), (dict(rs=99), INVALID),
    (dict(codes=OUT + 8), INVALID), (dict(rout=K, rs=128), INVALID), (dict(rout=P), INVALID),
    (dict(y=P), INVALID), (dict(y=K), INVALID), (dict(y=OUT), INVALID),
])
def test_norm(over, status):
    a = {**NORM, **over}
    refused(_lib.load().csdr_add_rms_norm(
        a["x"], a["dtype"], a["xs"], a["res"], a["rdt"], a["rs"], a["rout"], a["w"], a["eps"],
        a["rows"], a["n"], a["y"], a["codes"], a["scales"], None), status)


LINEAR = dict(w=P, ws=P, R=8, x=P, xs=P, M=4, C=100, bias=None, add=None, ads=0, y=OUT, dt=0, ys=0)


@pytest.mark.parametrize("over,status", [
    (dict(w=None), INVALID), (dict(ws=None), INVALID), (dict(x=None), INVALID),
    (dict(xs=None), INVALID), (dict(y=None), INVALID), (dict(R=0), INVALID), (dict(M=0), INVALID),
    (dict(C=0), INVALID), (dict(R=-1), INVALID), (dict(M=-1), INVALID), (dict(C=131072), UNSUPPORTED),
    (dict(dt=2), INVALID), (dict(ys=7), INVALID), (dict(add=P, ads=7), INVALID), (dict(w=P + 8), INVALID),
    (dict(x=P + 4), INVALID), (dict(M=1 << 22), INVALID), (dict(R=2 ** 31 - 1), INVALID),
    (dict(add=OUT, ads=16), INVALID),  # y in place with another stride
    (dict(y=P), INVALID),
])
def test_linear(over, status):
    a = {**LINEAR, **over}
    refused(_lib.load().csdr_q8_linear(a["w"], a["ws"], a["R"], a["x"], a["xs"], a["M"], a["C"],
                                       a["bias"], a["add"], a["ads"], a["y"], a["dt"], a["ys"], None),
            status)


ROTARY = dict(q=P, qo=OUT, Hq=4, qs=0, qos=0, k=K, ko=KO, Hk=2, ks=0, kos=0, dt=0, n=3, hd=64, dims=64,
              layout=0, pos=P, turns=P, mag=1.0)


@pytest.mark.parametrize("over,status", [
    (dict(q=None), INVALID), (dict(qo=None), INVALID), (dict(pos=None), INVALID),
    (dict(turns=None), INVALID), (dict(k=None), INVALID), (dict(ko=None), INVALID),
    (dict(dt=2), INVALID), (dict(layout=2), INVALID), (dict(layout=-1), INVALID), (dict(n=0), INVALID),
    (dict(n=-1), INVALID), (dict(Hq=0), INVALID), (dict(Hk=0), INVALID), (dict(Hq=65536), INVALID),
    (dict(Hk=65536), INVALID), (dict(hd=0), UNSUPPORTED), (dict(hd=1025), UNSUPPORTED),
    (dict(dims=0), UNSUPPORTED), (dict(dims=63), UNSUPPORTED), (dict(dims=66), UNSUPPORTED),
    (dict(mag=math.nan), INVALID), (dict(mag=math.inf), INVALID), (dict(qs=255), INVALID),
    (dict(qos=255), INVALID), (dict(ks=127), INVALID), (dict(kos=-128), INVALID),
    (dict(qo=P, qs=512), INVALID), (dict(ko=K, kos=512), INVALID), (dict(n=1 << 24), INVALID),
    (dict(qo=K), INVALID), (dict(ko=P), INVALID), (dict(ko=OUT), INVALID),
])
def test_rotary(over, status):
    a = {**ROTARY, **over}
    refused(_lib.load().csdr_rotary(
        a["q"], a["qo"], a["Hq"], a["qs"], a["qos"], a["k"], a["ko"], a["Hk"], a["ks"], a["kos"],
        a["dt"], a["n"], a["hd"], a["dims"], a["layout"], a["pos"], a["turns"], a["mag"], None), status)


def test_frequencies():
    d, theta = 64, 5e5
    plain = frequencies(d, theta)
    assert len(plain) == 32 and plain[0] == 1.0
    assert plain[31] == pytest.approx(theta ** (-62 / 64), rel=1e-14)
    assert frequencies(d, theta, "linear", 4.0) == [f / 4.0 for f in plain]
    # the fastest pair is kept, the slowest divided by the factor
    base = frequencies(d, theta, "base", 8.0)
    assert base[0] == 1.0 and base[31] == pytest.approx(plain[31] / 8.0, rel=1e-12)
    # by turns over the original positions: kept, between, divided
    parts = frequencies(d, theta, "parts", 8.0, original=8192, low=1.0, high=4.0)
    kinds = set()
    for f, g in zip(plain, parts):
        turns = 8192 * f / (2 * math.pi)
        if turns >= 4:
            kinds.add("kept")
            assert g == f
        elif turns <= 1:
            kinds.add("divided")
            assert g == f / 8.0
        else:
            kinds.add("between")
            assert f / 8.0 < g < f
            assert g == pytest.approx(f * (1 / 8 + (turns - 1) / 3 * (7 / 8)), rel=1e-12)
    assert kinds == {"kept", "between", "divided"}


@pytest.mark.parametrize("args", [
    dict(dims=0), dict(dims=7), dict(dims=-2), dict(dims=8, theta=0.0), dict(dims=8, theta=math.inf),
    dict(dims=8, theta=math.nan), dict(dims=8, scaling="linear", factor=0.0),
    dict(dims=8, scaling="other"), dict(dims=2, scaling="base", factor=2.0),
    dict(dims=8, scaling="parts", factor=8.0), dict(dims=8, scaling="parts", original=4096, low=4.0, high=4.0),
    dict(dims=8, scaling="parts", original=4096, low=-1.0, high=4.0),
])
def test_frequencies_refused(args):
    with pytest.raises(ValueError):
        frequencies(**args)
