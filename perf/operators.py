"""Serving from a paged K/V cache, and the log probabilities of what a model says: the operators as
cases that can be timed and compared, in their plain form or by the framework's kernels.

Kinds, each through its public entry point:
  append    new tokens' keys (rotated) and values into the pages of their sequences, their queries
            rotated, and the new rows read back as the values the cache holds (paged.PagedBatch
            .append, .read): single tokens of many sequences, prompts of different lengths
  attend    softmax attention of new tokens over the pages of their sequences (PagedBatch.attend):
            one token per sequence, or the tokens of prompts; scores capped by a tanh, lowered by
            distance, limited to a window and a prefix
  logprobs  log probability of a given token per row of logits, the row's entropy and its most
            likely tokens (logprobs.token_logprobs)

Pages (page_size positions of every KV head; K pages and V pages apart), per KV head:
  f16  K [position][dim]; V [position / 8][dim][position % 8]
  q4   codes, then per group of 32 dims and position a scale and a minimum (fp16, [group][position]
       each), value = minimum + scale * code. Eight codes share a 32-bit word, code e of the word
       in bits 4 (e / 2) + 16 (e % 2): K, for each position, words [dim % 32 / 8][dim / 32] of
       dims; V, for each 8 positions, words [dim % 16][dim / 16] of positions

Inputs are made from the seed alone.
"""
import math
import random

import torch

own = False

HEADS = dict(qwen=(14, 2, 64), llama=(32, 32, 128), gqa=(32, 8, 128))
VOCAB = 151936
THETA = 1e6
GROUP = 32
DT = dict(f32=torch.float32, f16=torch.float16)


def listed():
    return [
        # one token of one chat: the smallest append, as each layer of a 0.5B model makes it
        dict(name="append_step_b1", kind="append", heads="qwen", B=1, T=1, L=577, kv="f16",
             x="f32", ps=16),
        # one token of each of 64 conversations, far positions, 4-bit pages
        dict(name="append_step_b64_q4", kind="append", heads="gqa", B=64, T=1, L=8192, kv="q4",
             x="f16", ps=32),
        # four prompts of different lengths into 4-bit pages
        dict(name="append_prompts_q4", kind="append", heads="gqa", B=4, T=2048, L=2048, kv="q4",
             x="f32", ps=64),
        # the attention of that one chat's token: latency
        dict(name="attend_step_b1", kind="attend", heads="qwen", B=1, T=1, L=577, kv="f16",
             x="f32", ps=16, cap=0.0, window=0, slopes=False, prefix=0),
        # a batch of 32 conversations generating together
        dict(name="attend_step_b32", kind="attend", heads="gqa", B=32, T=1, L=4096, kv="f16",
             x="f16", ps=16, cap=0.0, window=0, slopes=False, prefix=0),
        # 64 long conversations of different lengths on a 4-bit cache
        dict(name="attend_step_b64_q4", kind="attend", heads="gqa", B=64, T=1, L=8192, kv="q4",
             x="f32", ps=32, cap=0.0, window=0, slopes=False, prefix=0),
        # one very long document on a 4-bit cache, capped scores
        dict(name="attend_long_q4", kind="attend", heads="gqa", B=1, T=1, L=131071, kv="q4",
             x="f16", ps=64, cap=30.0, window=0, slopes=False, prefix=0),
        # a whole prompt
        dict(name="attend_prompt", kind="attend", heads="gqa", B=1, T=4096, L=4096, kv="f16",
             x="f16", ps=64, cap=0.0, window=0, slopes=False, prefix=0),
        # the next chunks of four prompts of different lengths, 4-bit cache, fp32 activations
        dict(name="attend_prompts_q4", kind="attend", heads="gqa", B=4, T=1024, L=4096, kv="q4",
             x="f32", ps=32, cap=0.0, window=0, slopes=False, prefix=0),
        # a model with capped scores, distance bias and a sliding window behind a fixed prefix
        dict(name="attend_prompt_capped", kind="attend", heads="qwen", B=2, T=1000, L=2000,
             kv="f16", x="f32", ps=16, cap=30.0, window=500, slopes=True, prefix=16),
        # the alternatives beside the tokens of one decode step
        dict(name="logprobs_step", kind="logprobs", rows=8, n=VOCAB, x="f32", top=20),
        # a text scored under the model: perplexity, with the five likeliest tokens
        dict(name="logprobs_prompt", kind="logprobs", rows=2048, n=VOCAB, x="f32", top=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["append", "attend", "attend", "attend", "logprobs"])
    if kind == "logprobs":
        while True:
            rows, n = _log(rng, 1, 4096), _log(rng, 1000, 262144)
            if rows * n <= 2048 * VOCAB:
                return dict(kind=kind, rows=rows, n=n, x=rng.choice(["f32", "f16"]),
                            top=rng.choice([0, 1, 5, 20, 50]))
    heads = rng.choice(list(HEADS))
    Hq, Hkv, hd = HEADS[heads]
    kv, x, ps = rng.choice(["f16", "q4"]), rng.choice(["f32", "f16"]), rng.choice([16, 32, 64, 128])
    if kind == "append":
        while True:
            B, T, L = _log(rng, 1, 128), rng.choice([1, _log(rng, 2, 4096)]), _log(rng, 1, 16384)
            if T <= L and B * T * (Hq + 2 * Hkv) <= 8192 * 48 and B * L * Hkv <= 64 * 8192 * 8:
                return dict(kind=kind, heads=heads, B=B, T=T, L=L, kv=kv, x=x, ps=ps)
    while True:
        B, L = _log(rng, 1, 64), _log(rng, 1, 32768)
        T = rng.choice([1, 1, _log(rng, 2, 4096)])
        if (T <= L and B * L * Hkv <= 64 * 8192 * 8 and
                (T == 1 or B * T * L * Hq * hd <= 4096 * 4096 * 32 * 128)):
            break
    return dict(kind=kind, heads=heads, B=B, T=T, L=L, kv=kv, x=x, ps=ps,
                cap=rng.choice([0.0, 0.0, 30.0, 50.0]), slopes=rng.random() < 0.2,
                window=rng.choice([0, 0, _log(rng, 1, L)]),
                prefix=rng.choice([0, 0, rng.randint(1, min(L, 256))]))


# ---------------------------------------------------------------- inputs


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _lengths(case):
    """Positions and new tokens of each sequence: L and T of the first, at most those (down to
    half) of the others, the same for every seed."""
    B, T, L = case["B"], case["T"], case["L"]
    r = random.Random(B * 1000003 + T * 1009 + L)
    lens = [L] + [r.randint((L + 1) // 2, L) for _ in range(B - 1)]
    new = [T] + [min(n, r.randint((T + 1) // 2, T)) for n in lens[1:]]
    return lens, new


def _page_bytes(case):
    _, Hkv, hd = HEADS[case["heads"]]
    return case["ps"] * Hkv * (hd * 2 if case["kv"] == "f16" else hd // 2 + hd // GROUP * 4)


def _filled_pages(case, n_pages, g):
    """Pages of a cache in use: unit normal values (their layout does not matter: every value has
    the same distribution), quantised ones as codes of a normal over its group's range."""
    _, Hkv, hd = HEADS[case["heads"]]
    ps, dev = case["ps"], "cuda"
    if case["kv"] == "f16":
        p = torch.randn(n_pages, _page_bytes(case) // 2, generator=g, device=dev,
                        dtype=torch.float16)
        return p.view(torch.uint8)
    pages = torch.empty(n_pages, Hkv, ps * (hd // 2 + hd // GROUP * 4), dtype=torch.uint8,
                        device=dev)
    nc, npar = ps * hd // 2, ps * (hd // GROUP)
    z = torch.randn(2, n_pages, Hkv, nc, generator=g, device=dev, dtype=torch.float16)
    code = (z * 3.6 + 7.5).round().clamp(0, 15).to(torch.uint8)
    pages[:, :, :nc] = code[0] + 16 * code[1]
    u = torch.rand(2, n_pages, Hkv, npar, generator=g, device=dev)
    scale = 0.22 + 0.12 * u[0]
    low = -7.5 * scale + 0.3 * (u[1] - 0.5)
    pages[:, :, nc:nc + 2 * npar] = scale.half().contiguous().view(torch.uint8)
    pages[:, :, nc + 2 * npar:] = low.half().contiguous().view(torch.uint8)
    return pages.reshape(n_pages, -1)


def prepare(case, seed):
    g, dev = _generator(seed), "cuda"
    if case["kind"] == "logprobs":
        rows, n = case["rows"], case["n"]
        x = torch.randn(rows, n, generator=g, device=dev, dtype=DT[case["x"]])
        x.mul_(2.5)
        tokens = torch.randint(0, n, (rows,), generator=g, device=dev, dtype=torch.int32)
        x.scatter_add_(1, tokens.long()[:, None],
                       5 * torch.rand(rows, 1, generator=g, device=dev).to(x.dtype))
        return dict(case=case, logits=x, tokens=tokens)
    Hq, Hkv, hd = HEADS[case["heads"]]
    lens, new = _lengths(case)
    ps, B = case["ps"], case["B"]
    per_seq = (case["L"] + ps - 1) // ps
    n_pages = B * per_seq
    total = sum(new)
    st = dict(case=case, max_q=max(new), max_len=max(lens),
              lens=torch.tensor(lens, dtype=torch.int32, device=dev),
              table=torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
              .reshape(B, per_seq),
              k=_filled_pages(case, n_pages, g), v=_filled_pages(case, n_pages, g))
    # a step of one token each, or prompts one behind the other
    st["q_start"] = None if st["max_q"] == 1 else torch.tensor(
        [sum(new[:i]) for i in range(B + 1)], dtype=torch.int32, device=dev)
    if case["kind"] == "append":
        # one projection's output: queries, keys and values of a token side by side
        x = torch.randn(total, Hq + 2 * Hkv, hd, generator=g, device=dev).to(DT[case["x"]])
        st["q"], st["kn"], st["vn"] = x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]
        return st
    st["q"] = (1.5 * torch.randn(total, Hq, hd, generator=g, device=dev)).to(DT[case["x"]])
    st["slopes"] = (2.0 ** (-8.0 * torch.arange(1, Hq + 1, device=dev) / Hq)
                    if case["slopes"] else None)
    st["prefix"] = (torch.full((B,), case["prefix"], dtype=torch.int32, device=dev)
                    if case["prefix"] else None)
    return st


# ---------------------------------------------------------------- the plain forms


def _rows(st):
    """Sequence and position of every new token."""
    lens = st["lens"].long()
    if st["q_start"] is None:
        seq = torch.arange(len(lens), device="cuda")
        return seq, lens - 1, lens - 1
    start = st["q_start"].long()
    r = torch.arange(st["q"].shape[0], device="cuda")
    seq = torch.searchsorted(start, r, right=True) - 1
    first = lens - (start[1:] - start[:-1])
    return seq, first[seq] + r - start[seq], first[seq]


def _shifts():
    e = torch.arange(8, device="cuda", dtype=torch.int32)
    return 4 * (e // 2) + 16 * (e % 2)


def _parts(pages, case):
    """Views of q4 pages: codes as words, scales and minima."""
    _, Hkv, hd = HEADS[case["heads"]]
    ps, G = case["ps"], hd // GROUP
    nc, npar = ps * hd // 2, 2 * ps * G
    p = pages.unflatten(-1, (Hkv, nc + 2 * npar))
    return (p[..., :nc].view(torch.int32),
            p[..., nc:nc + npar].view(torch.float16).unflatten(-1, (G, ps)),
            p[..., nc + npar:].view(torch.float16).unflatten(-1, (G, ps)))


def _values(pages, case, is_v):
    """(..., page bytes) to (..., position in page, kv head, dim) in fp32."""
    _, Hkv, hd = HEADS[case["heads"]]
    ps, G = case["ps"], hd // GROUP
    if case["kv"] == "f16":
        p = pages.view(torch.float16)
        if is_v:
            p = p.unflatten(-1, (Hkv, ps // 8, hd, 8)).movedim(-1, -2).flatten(-3, -2)
        else:
            p = p.unflatten(-1, (Hkv, ps, hd))
        return p.movedim(-3, -2).float()
    words, scale, low = _parts(pages, case)
    if is_v:
        c = (words.unflatten(-1, (ps // 8, 16, hd // 16))[..., None] >> _shifts()) & 15
        c = c.movedim(-1, -3).transpose(-1, -2).flatten(-2).flatten(-3, -2)  # (Hkv, ps, hd)
    else:
        c = (words.unflatten(-1, (ps, 4, G))[..., None] >> _shifts()) & 15
        c = c.transpose(-3, -2).flatten(-3)
    c = c.unflatten(-1, (G, GROUP)).float()
    x = low.transpose(-1, -2)[..., None].float() + scale.transpose(-1, -2)[..., None].float() * c
    return x.flatten(-2).movedim(-3, -2)


def _quantise(x):
    """(n, kv heads, dims) fp32 to codes and the groups' fp16 scales and minima."""
    x = x.unflatten(-1, (-1, GROUP))
    low = x.amin(-1).half()
    scale = ((x.amax(-1) - low.float()) / x.new_full((), 15)).clamp(min=0).half()
    s = scale.double()[..., None]
    t = torch.where(s > 0, (x.double() - low.double()[..., None]) / s, 0.0)
    return t.round().clamp(0, 15).to(torch.int32).flatten(-2), scale, low


def _plain_append(st):
    case = st["case"]
    Hq, Hkv, hd = HEADS[case["heads"]]
    ps, G = case["ps"], hd // GROUP
    seq, pos, first = _rows(st)
    freq = THETA ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    ang = pos.double()[:, None, None] * freq
    c, s = ang.cos(), ang.sin()

    def turned(x):
        x = x.double()
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2).float()

    q = turned(st["q"]).to(st["q"].dtype)
    k, v = turned(st["kn"]), st["vn"].float()
    page = st["table"][seq, pos // ps].long()
    slot = pos % ps
    heads = torch.arange(Hkv, device="cuda")
    at = (page[:, None], heads, slot[:, None])
    if case["kv"] == "f16":
        st["k"].view(torch.float16).unflatten(-1, (Hkv, ps, hd))[at] = k.half()
        vp = st["v"].view(torch.float16).unflatten(-1, (Hkv, ps // 8, hd, 8))
        vp[page[:, None], heads, (slot // 8)[:, None], :, (slot % 8)[:, None]] = v.half()
    else:
        sh = _shifts()
        words, scale, low = _parts(st["k"], case)
        code, sc, lo = _quantise(k)
        w = (code.unflatten(-1, (G, 4, 8)).transpose(-3, -2) << sh).sum(-1)
        words.unflatten(-1, (ps, 4, G))[at] = w.to(torch.int32)
        scale[page[:, None], heads, :, slot[:, None]] = sc
        low[page[:, None], heads, :, slot[:, None]] = lo
        words, scale, low = _parts(st["v"], case)
        code, sc, lo = _quantise(v)
        # the words of a token's 8 positions: codes of this call's tokens, old ones elsewhere
        words = words.unflatten(-1, (ps // 8, 16, hd // 16))
        blk = (page[:, None], heads, (slot // 8)[:, None])
        e = torch.arange(8, device="cuda")
        p8 = pos[:, None] // 8 * 8 + e
        mine = (p8 >= first[:, None]) & (p8 < st["lens"].long()[seq][:, None])
        r = torch.arange(len(pos), device="cuda")[:, None] + p8 - pos[:, None]
        new = code.unflatten(-1, (hd // 16, 16)).transpose(-1, -2)[r.clamp(0, len(pos) - 1)]
        new = new.movedim(1, -1)  # (n, kv heads, 16, hd / 16, 8)
        old = (words[blk][..., None] >> sh) & 15
        w = (torch.where(mine[:, None, None, None], new, old) << sh).sum(-1)
        words[blk] = w.to(torch.int32)
        scale[page[:, None], heads, :, slot[:, None]] = sc
        low[page[:, None], heads, :, slot[:, None]] = lo
    return dict(q=q, k=_row_values(st["k"], case, page, slot, False).half(),
                v=_row_values(st["v"], case, page, slot, True).half())


def _row_values(pages, case, page, slot, is_v):
    """Single rows (page i, slot i) in fp32, (n, kv heads, dims)."""
    _, Hkv, hd = HEADS[case["heads"]]
    ps, G, sh = case["ps"], hd // GROUP, _shifts()
    if case["kv"] == "f16":
        p = pages.view(torch.float16)
        if is_v:
            return p.unflatten(-1, (Hkv, ps // 8, hd, 8))[page, :, slot // 8, :, slot % 8].float()
        return p.unflatten(-1, (Hkv, ps, hd))[page, :, slot].float()
    words, scale, low = _parts(pages, case)
    if is_v:
        w = words.unflatten(-1, (ps // 8, 16, hd // 16))[page, :, slot // 8]
        c = ((w >> sh[slot % 8][:, None, None, None]) & 15).transpose(-1, -2).flatten(-2)
    else:
        w = words.unflatten(-1, (ps, 4, G))[page, :, slot]
        c = ((w[..., None] >> sh) & 15).transpose(-3, -2).flatten(-3)
    scale, low = scale[page, :, :, slot], low[page, :, :, slot]
    c = c.unflatten(-1, (G, GROUP)).float()
    return (low[..., None].float() + scale[..., None].float() * c).flatten(-2)


def _plain_attend(st):
    case = st["case"]
    Hq, Hkv, hd = HEADS[case["heads"]]
    G, B, T, L = Hq // Hkv, case["B"], st["max_q"], st["max_len"]
    seq, pos, first = _rows(st)
    table = st["table"].long()
    k = _values(st["k"][table], case, False).flatten(1, 2)[:, :L]  # (B, L, kv heads, hd)
    v = _values(st["v"][table], case, True).flatten(1, 2)[:, :L]
    t = pos - first
    q = torch.zeros(B, T, Hq, hd, device="cuda")
    q[seq, t] = st["q"].float()
    # (B, kv heads, T G, hd) against (B, kv heads, hd, L)
    qh = q.unflatten(2, (Hkv, G)).permute(0, 2, 1, 3, 4).flatten(2, 3).contiguous()
    s = torch.matmul(qh, k.permute(0, 2, 3, 1).contiguous()) * (1.0 / math.sqrt(hd))
    s = s.unflatten(2, (T, G))
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    n = torch.bincount(seq, minlength=B)
    qpos = (st["lens"].long() - n)[:, None] + torch.arange(T, device="cuda")  # (B, T)
    p = torch.arange(L, device="cuda")
    away = qpos[:, :, None] - p
    if st["slopes"] is not None:
        bias = st["slopes"].reshape(Hkv, 1, G, 1) * away.abs()[:, None, :, None].float()
        s = s - bias
    see = away >= 0
    if case["window"]:
        see = see & (away < case["window"])
    if st["prefix"] is not None:
        see = see | (p < st["prefix"][:, None, None])
    see = see & (p < st["lens"][:, None, None])
    s = s.masked_fill(~see[:, None, :, None], -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    w = e / e.sum(-1, keepdim=True)
    o = torch.matmul(w.flatten(2, 3), v.permute(0, 2, 1, 3).contiguous())
    o = o.unflatten(2, (T, G)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # (B, T, Hq, hd)
    return o[seq, t].to(st["q"].dtype)


def _plain_logprobs(st):
    case, x = st["case"], st["logits"].float()
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    lse = m + torch.log(z)
    lp = (x.gather(1, st["tokens"].long()[:, None]) - lse)[:, 0]
    h = (lse - m - (e * (x - m)).sum(1, keepdim=True) / z)[:, 0]
    if not case["top"]:
        return dict(logprob=lp, entropy=h)
    # order by value, lower index first among equals: one whole-number key for both
    bits = x.view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20)
    key = key + ((1 << 20) - 1 - torch.arange(x.shape[1], device="cuda"))
    top = (1 << 20) - 1 - (key.topk(case["top"], 1).values & ((1 << 20) - 1))
    return dict(logprob=lp, entropy=h, top=top.to(torch.int32),
                top_logprob=x.gather(1, top) - lse)


# ---------------------------------------------------------------- one pass


def _batch(st):
    """The framework's handle of the sequences, kept as a serving loop keeps it."""
    if "batch" not in st:
        from cortexsdr_amd.paged import PagedCache

        case = st["case"]
        _, Hkv, hd = HEADS[case["heads"]]
        cache = PagedCache(st["k"].shape[0], case["ps"], Hkv, hd, case["kv"], k=st["k"], v=st["v"])
        st["batch"] = cache.batch(st["table"], st["lens"])
    return st["batch"]


def run(st):
    case = st["case"]
    if case["kind"] == "append":
        if not own:
            return _plain_append(st)
        b = _batch(st)
        q = b.append(st["q"], st["kn"], st["vn"], theta=THETA, q_start=st["q_start"],
                     max_q=st["max_q"])
        k, v = b.read(q.shape[0], q_start=st["q_start"], max_q=st["max_q"], dtype="f16")
        return dict(q=q, k=k, v=v)
    if case["kind"] == "attend":
        if not own:
            return _plain_attend(st)
        return _batch(st).attend(st["q"], q_start=st["q_start"], max_q=st["max_q"],
                                 max_len=st["max_len"], softcap=case["cap"],
                                 window=case["window"], slopes=st["slopes"], prefix=st["prefix"])
    if not own:
        return _plain_logprobs(st)
    from cortexsdr_amd.logprobs import token_logprobs

    r = token_logprobs(st["logits"], st["tokens"], top_n=case["top"])
    out = dict(logprob=r.logprobs, entropy=r.entropy)
    if case["top"]:
        out.update(top=r.top_ids, top_logprob=r.top_logprobs)
    return out


def _visible(case, lens, new):
    """Pairs of new token and visible position, and positions that some new token sees."""
    pairs = seen = 0
    for n, m in zip(lens, new):
        w, f = case["window"] or n, min(case["prefix"], n)
        for p in range(n - m, n):
            lo = max(0, p + 1 - w)
            pairs += p + 1 - max(lo, f) + f if p + 1 > f else f
        seen += n - max(0, min(n, max(0, n - m + 1 - w) - f))
    return pairs, seen


def work(case):
    if case["kind"] == "logprobs":
        size = 4 if case["x"] == "f32" else 2
        rows, n = case["rows"], case["n"]
        return {"bytes": rows * n * size + rows * (12 + 8 * case["top"]), "flops": 4.0 * rows * n}
    Hq, Hkv, hd = HEADS[case["heads"]]
    lens, new = _lengths(case)
    total, size = sum(new), 4 if case["x"] == "f32" else 2
    row = Hkv * (hd * 2 if case["kv"] == "f16" else hd // 2 + hd // GROUP * 4)  # K or V, one position
    if case["kind"] == "append":
        # inputs, turned queries, cache rows written and read, the rows' values
        by = total * ((2 * Hq + 2 * Hkv) * hd * size + 4 * row + 4 * Hkv * hd)
        return {"bytes": by, "flops": 3.0 * total * (Hq + Hkv) * hd}
    pairs, seen = _visible(case, lens, new)
    return {"bytes": 2 * seen * row + 2 * total * Hq * hd * size, "flops": 4.0 * pairs * Hq * hd}


# ---------------------------------------------------------------- in 64 bits


def _exact_row_values(pages, case, page, slot, is_v):
    """Rows (page i, slot i) in fp64, (n, kv heads, dims), read byte by byte."""
    _, Hkv, hd = HEADS[case["heads"]]
    ps, d = case["ps"], torch.arange(hd, device="cuda")
    raw = pages.reshape(len(pages), Hkv, -1)
    at = (page[:, None, None], torch.arange(Hkv, device="cuda")[:, None])

    def byte_at(off):  # bytes at offsets (n, m) of each head, (n, kv heads, m)
        return raw[(*at, off[:, None])].to(torch.int32)

    def half_at(off):
        b = byte_at(off) + 256 * byte_at(off + 1)
        return b.to(torch.int16).view(torch.float16).double()

    s = slot[:, None]
    if case["kv"] == "f16":
        return half_at(2 * ((s // 8 * hd + d) * 8 + s % 8) if is_v else 2 * (s * hd + d))
    e = s % 8 + 0 * d if is_v else (d % 8) + 0 * s
    nib = e // 2 + 4 * (e % 2)
    word = s // 8 * hd + d % 16 * (hd // 16) + d // 16 if is_v else \
        s * (hd // 8) + d % 32 // 8 * (hd // 32) + d // 32
    byte = byte_at(4 * word + nib // 2)
    code = torch.where((nib % 2 == 1)[:, None], byte // 16, byte % 16).double()
    par = ps * hd // 2 + 2 * (d // 32 * ps + s)
    return half_at(par + 2 * ps * (hd // 32)) + half_at(par) * code


def _exact_append(case, st):
    """The turned queries and, for fp16 pages, the rows they hold; 4-bit rows hang on borders
    between codes and have none."""
    Hq, Hkv, hd = HEADS[case["heads"]]
    lens, new = _lengths(case)
    pos = torch.cat([torch.arange(n - m, n, device="cuda") for n, m in zip(lens, new)]).double()
    i = torch.arange(hd // 2, device="cuda").double()
    turn = torch.polar(torch.ones_like(pos[:, None] + i),
                       pos[:, None] * torch.exp(i * (-2.0 * math.log(THETA) / hd)))[:, None]

    def turned(x):
        z = torch.view_as_complex(x.double().reshape(*x.shape[:-1], hd // 2, 2).contiguous())
        return torch.view_as_real(z * turn).reshape(x.shape)

    if case["kv"] == "q4":
        return dict(q=turned(st["q"]), k=None, v=None)
    return dict(q=turned(st["q"]), k=turned(st["kn"]), v=st["vn"].double())


def _exact_attend(case, st):
    Hq, Hkv, hd = HEADS[case["heads"]]
    lens, new = _lengths(case)
    out, row = [], 0
    slopes = st["slopes"].double().tolist() if case["slopes"] else None
    for b, (n, m) in enumerate(zip(lens, new)):
        p = torch.arange(n, device="cuda")
        page = st["table"][b].long()[p // case["ps"]]
        k = torch.empty(n, Hkv, hd, dtype=torch.float64, device="cuda")
        v = torch.empty_like(k)
        for i in range(0, n, 16384):
            at, sl = page[i:i + 16384], p[i:i + 16384] % case["ps"]
            k[i:i + 16384] = _exact_row_values(st["k"], case, at, sl, False)
            v[i:i + 16384] = _exact_row_values(st["v"], case, at, sl, True)
        qp = torch.arange(n - m, n, device="cuda")[:, None]
        hide = p > qp
        if case["window"]:
            hide = hide | (p <= qp - case["window"])
        if case["prefix"]:
            hide = hide & (p >= case["prefix"])
        o = torch.empty(m, Hq, hd, dtype=torch.float64, device="cuda")
        for h in range(Hq):
            kh = h * Hkv // Hq
            y = st["q"][row:row + m, h].double() @ k[:, kh].t().contiguous() / hd ** 0.5
            if case["cap"]:
                y = torch.tanh(y / case["cap"]) * case["cap"]
            if slopes:
                y = y - slopes[h] * (qp - p).abs()
            y = torch.softmax(y.masked_fill(hide, -math.inf), -1)
            o[:, h] = y @ v[:, kh].contiguous()
        out.append(o)
        row += m
    return torch.cat(out)


def _exact_logprobs(case, st):
    got = dict(logprob=[], entropy=[], top_logprob=[])
    for x, t in zip(st["logits"].split(256), st["tokens"].split(256)):
        lp = torch.log_softmax(x.double(), 1)
        got["logprob"].append(lp.gather(1, t.long()[:, None])[:, 0])
        got["entropy"].append(-(lp.exp() * lp).sum(1))
        got["top_logprob"].append(lp.topk(max(case["top"], 1), 1).values)
    out = {k: torch.cat(v) for k, v in got.items()}
    if not case["top"]:
        del out["top_logprob"]
        return out
    return dict(out, top=None)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, st)
    if case["kind"] == "attend":
        return _exact_attend(case, st)
    return _exact_logprobs(case, st)
