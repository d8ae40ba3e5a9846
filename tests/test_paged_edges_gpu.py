"""Paged attention at the ends of what a call may be: scores of -infinity alone, lengths past the
table, prompts captured before their first launch."""
import numpy as np
import pytest

import paged_ref as ref
from conftest import rel_l2
from test_paged_gpu import HEADS, TOL32, Setup, tol

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["f16"])
@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("tokens", [1, 70])
def test_nothing_but_minus_infinity(gpu, kv, x, tokens):
    """A token whose every score is -infinity has no softmax: NaN, as the formula says, and not the
    zeros of a token that sees nothing."""
    s = Setup(gpu, [100 + tokens, 40 + tokens], HEADS["three"], kv, x, seed=61)
    k = s.draw(140, 2)
    k[:100, 1, 3] = -np.inf              # sequence 0, KV head 1
    s.append([100, 40], with_q=False, k=k)
    k = s.draw(2 * tokens, 2)
    k[:tokens, 1, 3] = -np.inf
    s.append([tokens, tokens], with_q=False, k=k)
    q = s.draw(2 * tokens, 6)
    q[:, :, 3] = np.abs(q[:, :, 3]) + s.np_x(0.5)
    want = s.expect(q, [tokens, tokens])
    got = s.batch.attend(s.dev(q)).cpu().numpy()
    assert np.isnan(want[:tokens, 3:]).all()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = np.isfinite(want)
    assert rel_l2(got[fine], want[fine]) <= tol(x)


@pytest.mark.parametrize("kv", ["f16", "q4"])
@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("window", [0, 9, 30])
def test_lengths_past_the_table(gpu, kv, x, tokens, window):
    """Positions past a row's end are neither written nor seen; a window that lies there sees
    nothing, and the prefix still does."""
    s = Setup(gpu, [64], HEADS["three"], kv, x, ps=16, seed=62)
    s.append([64], with_q=False)
    batch = s.cache.batch(s.table[:, :4].contiguous(), s.lens)
    s.lens.fill_(100)
    k0, v0 = s.cache.k.clone(), s.cache.v.clone()
    new = s.draw(tokens, 2)
    batch.append(None, s.dev(new), s.dev(new))
    pos = np.arange(100 - tokens, 100)
    kept = pos < 64
    if not kept.any():
        assert gpu.equal(s.cache.k, k0) and gpu.equal(s.cache.v, v0)
    k, v = s.k[0].copy(), s.v[0].copy()
    k[pos[kept]] = v[pos[kept]] = ref.held(new[kept].astype(np.float32), kv)
    q = s.draw(tokens, 6, 1.5)
    for prefix in (0, 5, 1000):
        want = ref.attend(q, pos, k, v, window=window, prefix=prefix)
        p = gpu.tensor([prefix], dtype=gpu.int32, device="cuda")
        got = batch.attend(s.dev(q), window=window, prefix=p).cpu().numpy()
        assert rel_l2(got, want) <= tol(x)
        assert not got[~want.any((1, 2))].any()


@pytest.mark.parametrize("kv", ["f16", "q4"])
@pytest.mark.parametrize("x", ["f32", "f16"])
def test_captured_prompts(gpu, kv, x):
    """Chunks of prompts captured (append and attention), replayed as lengths and starts change, with
    eager calls between; two graphs in turn."""
    heads = (64, 16, 128)  # columns for the larger workgroups too
    old, new = [30, 0, 17, 5], [260, 150, 40, 301]
    s = Setup(gpu, [2 * (a + b) for a, b in zip(old, new)], heads, kv, x, ps=32, seed=63, theta=1e4)
    s.append(old, with_q=False)
    n, mq = sum(new), max(new)
    q, k, v = (gpu.zeros((n, h, 128), device="cuda", dtype=gpu.float16 if x == "f16" else
                         gpu.float32) for h in (64, 16, 16))
    start = s.starts(new)
    graphs = []
    for _ in range(2):
        g = gpu.cuda.CUDAGraph()
        with gpu.cuda.graph(g):
            out = s.batch.attend(s.batch.append(q, k, v, theta=1e4, q_start=start, max_q=mq),
                                 q_start=start, max_q=mq)
        graphs.append((g, out))
    for i, part in enumerate((new, [100, 150, 1, 0], [1, 1, 1, 1])):
        m = sum(part)
        s.len = [a + b for a, b in zip(s.len, part)]
        s.lens.copy_(gpu.tensor(s.len, dtype=gpu.int32))
        start.copy_(s.starts(part))
        hq, hk, hv = s.draw(m, 64, 1.5), s.draw(m, 16), s.draw(m, 16)
        for d, h in ((q, hq), (k, hk), (v, hv)):
            d[:m].copy_(s.dev(h))
        g, out = graphs[i % 2]
        g.replay()
        # (the same sizes: these choose the kernel)
        qd = s.batch.append(q, k, v, theta=1e4, q_start=start, max_q=mq)
        eager = s.batch.attend(qd, q_start=start, max_q=mq)
        gpu.cuda.synchronize()
        assert gpu.equal(out[:m], eager[:m])
        pos = s.positions(part)
        row = 0
        for b, c in enumerate(part):
            kr = ref.rotate(hk[row:row + c], pos[b], 1e4).astype(np.float32)
            s.k[b] = np.concatenate([s.k[b], ref.held(kr, kv)])
            s.v[b] = np.concatenate([s.v[b], ref.held(hv[row:row + c], kv)])
            row += c
    want = s.expect(qd[:m].cpu().numpy(), part)
    assert rel_l2(out[:m].cpu().numpy(), want) <= tol(x)


@pytest.mark.parametrize("kv", ["f16", "q4"])
@pytest.mark.parametrize("x", ["f32", "f16"])
@pytest.mark.parametrize("heads,tokens", [
    ("three", 6), ("three", 21), ("three", 30), ("three", 42), ("gqa", 5), ("gqa", 16), ("gqa", 17),
    ("gqa", 32), ("llama", 18), ("llama", 64), ("llama", 128), ("qwen", 18), ("many", 3),
])
def test_both_forms_for_few_tokens(gpu, kv, x, heads, tokens):
    """17 to 128 pairs of token and query head: the bound of the lengths, here a table's capacity,
    decides between the kernels; either is right."""
    s = Setup(gpu, [150 + tokens, 40 + tokens], HEADS[heads], kv, x, ps=16, seed=64)
    s.append([150, 40], with_q=False)
    qd, _ = s.append([tokens, tokens])
    wide = gpu.full((2, 65536), -1, dtype=gpu.int32, device="cuda")
    wide[:, :s.table.shape[1]] = s.table
    far = s.cache.batch(wide, s.lens)
    prefix = gpu.tensor([3, 170], dtype=gpu.int32, device="cuda")
    for a, e in (({}, {}), (dict(window=50, prefix=prefix), dict(window=50, prefix=[3, 170]))):
        want = s.expect(qd.cpu().numpy(), [tokens, tokens], **e)
        for batch, n in ((s.batch, 0), (far, 0), (far, 200), (far, 5000)):
            assert rel_l2(batch.attend(qd, max_len=n, **a).cpu().numpy(), want) <= tol(x)
