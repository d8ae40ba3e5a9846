"""A transformer layer in 8 bits: the operators around and in its products, as cases that can be timed
and compared, in their plain form or by the framework's kernels.

Kinds, each through its public entry point:
  norm      root-mean-square norm of a residual stream to which a sublayer's output is added first:
            the new stream, the norm as 8-bit rows, and on request as values too (q8.rms_norm)
  quantise  rows of activations, or of silu(gate) * x, or of a weight matrix, as 8-bit rows
            (q8.quantize)
  linear    product of 8-bit tokens with 8-bit weights, with a scale per token and per output channel,
            a bias, and the addition of a residual (q8.linear)
  rotary    queries and keys turned at their positions: adjacent pairs or halves, a whole head or its
            first dims, frequencies scaled for long contexts (rotary.Rotary.apply)

8-bit rows: codes of a row are round(127 v / max|v|), ties to even, its scale max|v| / 127; their values
(scale * code, q8.Q8Rows.values) are what norm and quantise return here. A row of codes takes a whole
number of 128 bytes, zeros behind its last value.

Inputs are made from the seed alone.
"""
import math
import random

import torch

own = False

# (query heads, key-value heads, head dim)
HEADS = dict(qwen=(14, 2, 64), llama=(32, 32, 128), gqa=(32, 8, 128))
DT = dict(f32=torch.float32, f16=torch.float16)
EPS = 1e-5
PITCH = 128
# widths of a layer: hidden sizes, projections of queries, keys and values, feed-forward sizes
WIDTHS = (896, 1152, 4096, 4864, 6144, 11008, 14336)
MOST = 4096 * 4096 * 11008  # multiply-adds of the largest product


def listed():
    return [
        # one token of one chat through a 0.5B model: the smallest norm, fp32 stream
        dict(name="norm_step", kind="norm", rows=1, n=896, x="f32", res="f32", y=False),
        # 777 tokens of prompts whose norm is also wanted as values, an odd width
        dict(name="norm_odd", kind="norm", rows=777, n=5003, x="f32", res="f32", y=True),
        # a prompt of 4096 tokens of a 7B model, fp16 stream
        dict(name="norm_prompt", kind="norm", rows=4096, n=4096, x="f16", res="f16", y=False),
        # the attention's outputs of 64 conversations generating together, for the output projection
        dict(name="quantise_step", kind="quantise", rows=64, n=4096, x="f16", gate=False),
        # the feed-forward's gate and up projections of a prompt, for the down projection
        dict(name="quantise_gated_prompt", kind="quantise", rows=4096, n=11008, x="f16", gate=True),
        # queries, keys and values of one token of a 0.5B model: latency
        dict(name="linear_step_small", kind="linear", M=1, R=1152, C=896, y="f32", bias=True,
             add=False),
        # gate and up of one token of a 7B model: the stream of the weights
        dict(name="linear_step", kind="linear", M=1, R=22016, C=4096, y="f16", bias=False, add=False),
        # down, onto the residual stream, for 64 conversations generating together
        dict(name="linear_batch", kind="linear", M=64, R=4096, C=11008, y="f16", bias=False, add=True),
        # odd sizes
        dict(name="linear_odd", kind="linear", M=333, R=1001, C=4999, y="f32", bias=True, add=False),
        # down of a prompt of 4096 tokens
        dict(name="linear_prompt", kind="linear", M=4096, R=4096, C=11008, y="f16", bias=False,
             add=True),
        # queries and keys of one token of each of 64 conversations at far positions
        dict(name="rotary_step", kind="rotary", heads="gqa", tokens=64, x="f16", layout="halves",
             part=1, scaling="parts", far=True),
        # a prompt of a model that turns a quarter of a head's dims
        dict(name="rotary_prompt", kind="rotary", heads="llama", tokens=8192, x="f16",
             layout="adjacent", part=4, scaling="none", far=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng):
    return rng.choice(WIDTHS) if rng.random() < 0.6 else _log(rng, 100, 16000)


def draw(rng: random.Random):
    kind = rng.choice(["norm", "quantise", "linear", "linear", "rotary"])
    x = rng.choice(["f32", "f16"])
    if kind == "rotary":
        while True:
            heads, tokens = rng.choice(list(HEADS)), _log(rng, 1, 16384)
            Hq, Hkv, hd = HEADS[heads]
            if tokens * (Hq + Hkv) * hd * (2 if x == "f16" else 4) <= 8192 * 64 * 128 * 2:
                return dict(kind=kind, heads=heads, tokens=tokens, x=x,
                            layout=rng.choice(["adjacent", "halves"]), part=rng.choice([1, 1, 2, 4]),
                            scaling=rng.choice(["none", "linear", "base", "parts"]),
                            far=rng.random() < 0.5)
    if kind == "linear":
        while True:
            M = rng.choice([_log(rng, 1, 32), _log(rng, 1, 8192)])
            R, C = _width(rng), _width(rng)
            if M * R * C <= MOST:
                return dict(kind=kind, M=M, R=R, C=C, y=rng.choice(["f32", "f16"]),
                            bias=rng.random() < 0.3, add=rng.random() < 0.3)
    while True:
        rows, n = _log(rng, 1, 16384), _width(rng)
        if rows * n <= (4096 * 4096 if kind == "norm" else 4096 * 11008):
            break
    if kind == "norm":
        return dict(kind=kind, rows=rows, n=n, x=x, res=rng.choice(["", x, "f32"]),
                    y=rng.random() < 0.3)
    return dict(kind=kind, rows=rows, n=n, x=x, gate=rng.random() < 0.6)


# ---------------------------------------------------------------- inputs


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _activations(g, rows, n):
    """Unit normal, tokens of different size, a few channels far larger than the others."""
    x = torch.randn(rows, n, generator=g, device="cuda")
    x.mul_(torch.exp(0.5 * torch.randn(rows, 1, generator=g, device="cuda")))
    return x.mul_(torch.where(torch.rand(n, generator=g, device="cuda") < 0.004, 6.0, 1.0))


def _codes(v):
    """8-bit rows of v: codes with zeros up to the pitch, scales."""
    top = v.abs().amax(1, keepdim=True)
    codes = torch.zeros(v.shape[0], -(-v.shape[1] // PITCH) * PITCH, dtype=torch.int8, device="cuda")
    codes[:, :v.shape[1]] = (v * (127.0 / top)).round().to(torch.int8)
    return codes, (top / 127)[:, 0].contiguous()


def _frequencies(case, dims):
    """The scaled frequencies' parameters, as a model's configuration holds them."""
    s = case["scaling"]
    return dict(theta=1e6 if case["heads"] == "qwen" else 5e5, dims=dims, layout=case["layout"],
                scaling=s, factor=1.0 if s == "none" else 8.0,
                original=8192 if s == "parts" else 0, low=1.0, high=4.0,
                magnitude=1.0 + 0.1 * math.log(8.0) if s == "parts" else 1.0)


def prepare(case, seed):
    g, dev = _generator(seed), "cuda"
    if case["kind"] == "norm":
        st = dict(case=case, x=_activations(g, case["rows"], case["n"]).to(DT[case["x"]]),
                  w=1 + 0.3 * torch.randn(case["n"], generator=g, device=dev), residual=None)
        if case["res"]:
            st["residual"] = (3 * _activations(g, case["rows"], case["n"])).to(DT[case["res"]])
        return st
    if case["kind"] == "quantise":
        rows, n = case["rows"], case["n"]
        # gate and up lie side by side in one projection's output
        both = _activations(g, rows, 2 * n if case["gate"] else n).to(DT[case["x"]])
        return dict(case=case, x=both[:, n:] if case["gate"] else both,
                    gate=both[:, :n] if case["gate"] else None)
    if case["kind"] == "linear":
        M, R, C = case["M"], case["R"], case["C"]
        xc, xs = _codes(_activations(g, M, C))
        wc, ws = _codes(torch.randn(R, C, generator=g, device=dev) * (1 / math.sqrt(C)))
        return dict(case=case, x=xc, x_scales=xs, w=wc, w_scales=ws,
                    bias=torch.randn(R, generator=g, device=dev) if case["bias"] else None,
                    add=torch.randn(M, R, generator=g, device=dev).to(DT[case["y"]])
                    if case["add"] else None)
    Hq, Hkv, hd = HEADS[case["heads"]]
    n = case["tokens"]
    x = torch.randn(n, Hq + 2 * Hkv, hd, generator=g, device=dev, dtype=DT[case["x"]])
    if case["far"]:
        pos = torch.randint(0, 131072, (n,), generator=g, device=dev, dtype=torch.int32)
    else:
        first = torch.randint(0, 4096, (1,), generator=g, device=dev, dtype=torch.int32)
        pos = first + torch.arange(n, device=dev, dtype=torch.int32)
    return dict(case=case, q=x[:, :Hq], k=x[:, Hq:Hq + Hkv], positions=pos)


# ---------------------------------------------------------------- the plain forms


def _eight_bits(t):
    """Codes and largest magnitudes of rows t (fp64: a code is the nearest, also next to a border)."""
    top = t.abs().amax(1, keepdim=True)
    return (127 * t / top).round(), top


def _plain_norm(st):
    x, w = st["x"].float(), st["w"]
    out = {}
    if st["residual"] is not None:
        h = (x + st["residual"].float()).to(st["residual"].dtype)
        out["residual"] = h
        x = h.float()
    r = 1 / torch.sqrt(x.square().mean(1, keepdim=True) + EPS)
    code, top = _eight_bits(x.double() * w.double())
    scale = (top * r.double() / 127).float()
    out.update(values=(scale * code.float()).half(), scales=scale[:, 0])
    if st["case"]["y"]:
        out["y"] = (x * r * w).to(st["x"].dtype)
    return out


def _plain_quantise(st):
    t = st["x"].double()
    if st["gate"] is not None:
        g = st["gate"].double()
        t = g / (1 + torch.exp(-g)) * t
    code, top = _eight_bits(t)
    scale = (top / 127).float()
    return dict(values=(scale * code.float()).half(), scales=scale[:, 0])


def _plain_linear(st):
    C = st["case"]["C"]
    y = st["x"][:, :C].float() @ st["w"][:, :C].float().t()
    y = y * st["x_scales"][:, None] * st["w_scales"]
    if st["bias"] is not None:
        y = y + st["bias"]
    if st["add"] is not None:
        y = y + st["add"].float()
    return y.to(DT[st["case"]["y"]])


def _plain_rotary(st):
    case = st["case"]
    hd = HEADS[case["heads"]][2]
    f = _frequencies(case, hd // case["part"])
    dims, theta = f["dims"], f["theta"]
    if f["scaling"] == "base":
        theta = theta * f["factor"] ** (dims / (dims - 2))
    freq = theta ** (-torch.arange(0, dims, 2, device="cuda", dtype=torch.float64) / dims)
    if f["scaling"] == "linear":
        freq = freq / f["factor"]
    elif f["scaling"] == "parts":
        turns = f["original"] * freq / (2 * math.pi)
        keep = ((turns - f["low"]) / (f["high"] - f["low"])).clamp(0, 1)
        freq = freq * (keep + (1 - keep) / f["factor"])
    ang = st["positions"].double()[:, None, None] * freq
    c, s = (ang.cos() * f["magnitude"]).float(), (ang.sin() * f["magnitude"]).float()

    def turned(x):
        y = x.float()
        z = y[..., :dims]
        if case["layout"] == "adjacent":
            a, b = z[..., 0::2], z[..., 1::2]
            z = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
        else:
            a, b = z[..., :dims // 2], z[..., dims // 2:]
            z = torch.cat((a * c - b * s, a * s + b * c), -1)
        return torch.cat((z, y[..., dims:]), -1).to(x.dtype)

    return dict(q=turned(st["q"]), k=turned(st["k"]))


# ---------------------------------------------------------------- one pass


def _handles(st):
    """What a program keeps between calls: the two 8-bit matrices, or the rotation."""
    case = st["case"]
    if "handles" not in st:
        if case["kind"] == "linear":
            from cortexsdr_amd.q8 import Q8Rows

            st["handles"] = (Q8Rows(st["w"], st["w_scales"], case["C"]),
                             Q8Rows(st["x"], st["x_scales"], case["C"]))
        else:
            from cortexsdr_amd.rotary import Rotary

            hd = HEADS[case["heads"]][2]
            st["handles"] = Rotary(hd, **_frequencies(case, hd // case["part"]))
    return st["handles"]


def run(st):
    case = st["case"]
    kind = case["kind"]
    if not own:
        return dict(norm=_plain_norm, quantise=_plain_quantise, linear=_plain_linear,
                    rotary=_plain_rotary)[kind](st)
    if kind == "rotary":
        q, k = _handles(st).apply(st["q"], st["positions"], k=st["k"])
        return dict(q=q, k=k)
    from cortexsdr_amd import q8

    if kind == "linear":
        w, x = _handles(st)
        return q8.linear(w, x, bias=st["bias"], add=st["add"], dtype=case["y"])
    if kind == "quantise":
        rows = q8.quantize(st["x"], gate=st["gate"])
        return dict(values=rows.values("f16"), scales=rows.scales)
    r = q8.rms_norm(st["x"], st["w"], EPS, residual=st["residual"], y=case["y"])
    out = dict(values=r.rows.values("f16"), scales=r.rows.scales)
    if case["res"]:
        out["residual"] = r.residual
    if case["y"]:
        out["y"] = r.y
    return out


def work(case):
    size = dict(f32=4, f16=2)
    if case["kind"] == "rotary":
        Hq, Hkv, hd = HEADS[case["heads"]]
        n = case["tokens"]
        turned = n * (Hq + Hkv) * hd
        return {"bytes": 2 * turned * size[case["x"]] + 4 * n, "flops": 3.0 * turned / case["part"]}
    if case["kind"] == "linear":
        M, R, C = case["M"], case["R"], case["C"]
        by = (M + R) * (C + 4) + M * R * size[case["y"]] * (2 if case["add"] else 1)
        return {"bytes": by + (4 * R if case["bias"] else 0), "flops": 2.0 * M * R * C}
    rows, n, s = case["rows"], case["n"], size[case["x"]]
    # the codes are written; what they stand for is written too
    by = rows * n * (s + 1 + 2) + 4 * rows
    if case["kind"] == "quantise":
        return {"bytes": by + (rows * n * s if case["gate"] else 0),
                "flops": (9.0 if case["gate"] else 4.0) * rows * n}
    by += 4 * n + (2 * rows * n * size[case["res"]] if case["res"] else 0)
    return {"bytes": by + (rows * n * s if case["y"] else 0), "flops": 8.0 * rows * n}


# ---------------------------------------------------------------- in 64 bits


def _exact_rows(t):
    """Values and scales of 8-bit rows of t; codes by the distance to both neighbours."""
    scale = torch.linalg.vector_norm(t, ord=math.inf, dim=1, keepdim=True) / 127
    low = torch.floor(t / scale)
    up = t - low * scale - ((low + 1) * scale - t)  # above zero: nearer to low + 1
    code = torch.where((up > 0) | ((up == 0) & (low.remainder(2) == 1)), low + 1, low)
    return code, scale


def _exact_norm(case, st):
    h, out = st["x"].double(), {}
    if case["res"]:
        # the stream holds the sum in its own type, and the norm is of what the stream holds
        out["residual"] = h + st["residual"].double()
        h = out["residual"].to(DT[case["res"]]).double()
    t = h * st["w"].double()
    r = (torch.linalg.vector_norm(h, dim=1, keepdim=True).square() / case["n"] + EPS).rsqrt()
    code, scale = _exact_rows(t)
    out.update(values=code * scale * r, scales=(scale * r)[:, 0])
    if case["y"]:
        out["y"] = t * r
    return out


def _exact_linear(case, st):
    xs, ws = st["x_scales"].double(), st["w_scales"].double()
    C = case["C"]
    y = torch.mm(xs[:, None] * st["x"][:, :C].double(),
                 (ws[:, None] * st["w"][:, :C].double()).t().contiguous())
    if case["bias"]:
        y = y + st["bias"].double()
    return y + st["add"].double() if case["add"] else y


def _exact_rotary(case, st):
    hd = HEADS[case["heads"]][2]
    f = _frequencies(case, hd // case["part"])
    dims, half = f["dims"], f["dims"] // 2
    base = math.log(f["theta"])
    if f["scaling"] == "base":
        base += math.log(f["factor"]) * dims / (dims - 2)
    freq = []
    for j in range(half):
        w = math.exp(-2.0 * j / dims * base)
        if f["scaling"] == "linear":
            w /= f["factor"]
        elif f["scaling"] == "parts":
            turns = f["original"] / (2 * math.pi / w)
            if turns <= f["low"]:
                w /= f["factor"]
            elif turns < f["high"]:
                part = (turns - f["low"]) / (f["high"] - f["low"])
                w = (1 - part) * w / f["factor"] + part * w
        freq.append(w)
    pos = st["positions"].double()
    turn = torch.polar(torch.full((len(pos), half), f["magnitude"], dtype=torch.float64, device="cuda"),
                       pos[:, None] * torch.tensor(freq, dtype=torch.float64, device="cuda"))[:, None]

    def turned(x):
        y = x.double().contiguous()
        if case["layout"] == "adjacent":
            z = torch.complex(y[..., 0:dims:2].contiguous(), y[..., 1:dims:2].contiguous()) * turn
            y[..., 0:dims:2], y[..., 1:dims:2] = z.real, z.imag
        else:
            z = torch.complex(y[..., :half].contiguous(), y[..., half:dims].contiguous()) * turn
            y[..., :half], y[..., half:dims] = z.real, z.imag
        return y

    return dict(q=turned(st["q"]), k=turned(st["k"]))


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(case, st)
    if case["kind"] == "linear":
        return _exact_linear(case, st)
    if case["kind"] == "rotary":
        return _exact_rotary(case, st)
    t = st["x"].double()
    if case["gate"]:
        t = t * st["gate"].double() * torch.sigmoid(st["gate"].double())
    code, scale = _exact_rows(t)
    return dict(values=code * scale, scales=scale[:, 0])
