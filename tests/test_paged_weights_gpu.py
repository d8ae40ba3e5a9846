"""Paged attention in fp16 calls: softmax weights and the sum that divides them belong together, and
where weights are held in pairs only the output's rounding is left."""
import numpy as np
import pytest

import paged_ref as ref
from test_paged_gpu import HEADS, TOL32, Setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["f16", "q4"])
@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("tokens", [1, 70])
@pytest.mark.parametrize("below", [0.1, 0.3, 0.45, 0.7, 0.9, 1.3])
def test_constant_values_come_back(gpu, kv, x, tokens, below):
    """V = 1 everywhere, one position in 32 scored `below` above the others, so that nearly all
    weights are the same number, rounded the same way: every output is 1."""
    hq, hkv, hd = HEADS["three"]
    n = 640
    s = Setup(gpu, [n + tokens], HEADS["three"], kv, x, ps=32, seed=51)
    k = np.zeros((n, hkv, hd), np.float32)
    k[np.arange(n) % 32 != 0] = -1.0
    s.append([n], with_q=False, k=k, v=np.ones((n, hkv, hd)))
    s.append([tokens], with_q=False, k=np.full((tokens, hkv, hd), -1.0),
             v=np.ones((tokens, hkv, hd)))
    q = np.full((tokens, hq, hd), below / hd, s.np_x)
    out = s.batch.attend(s.dev(q), scale=1.0).cpu().numpy().astype(np.float64)
    # numerator and denominator are the same sum, or the same to 2^-20 (pairs); one division
    assert np.abs(out - 1).max() <= (0 if x == "f16" else 2.0 ** -20)


@pytest.mark.parametrize("heads,lens,o", [
    ("gqa", [900, 64, 33], {}), ("qwen", [3000], {}), ("three", [500, 1], dict(cap=20.0)),
    ("llama", [257], dict(window=100)),
])
def test_single_tokens_on_fp16_pages(gpu, heads, lens, o):
    """fp16 calls there: fp32 quality, then the output's one rounding."""
    s = Setup(gpu, lens, HEADS[heads], "f16", "f16", ps=16, seed=52, theta=1e4)
    s.append([n - 1 for n in lens], with_q=False)
    qd, _ = s.append([1] * len(lens))
    want = s.expect(qd.cpu().numpy(), [1] * len(lens), **o)
    got = s.batch.attend(qd, softcap=o.get("cap", 0.0), window=o.get("window", 0))
    off = np.abs(got.cpu().numpy().astype(np.float64) - want)
    # half a step of fp16; beside it fp32's error, on any element up to 8 times its mean
    bound = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + 8 * TOL32 * np.sqrt((want ** 2).mean())
    assert float((off / bound).max()) <= 1
