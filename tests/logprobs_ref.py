"""Token log probabilities in fp64 on the CPU: numpy, from the formulas, row by row.

A row with a NaN or +infinity has no probabilities; its top is of the values below +infinity."""
import numpy as np


def scores(x, tokens, top_n, temperature=1.0):
    """(log probabilities, entropy, top ids, their log probabilities, mean |y - max y|) of the rows
    x, fp32 or fp16 values as given."""
    x = x.astype(np.float64)
    t = float(np.float32(temperature)) if temperature > 0 else 1.0
    rows, n = x.shape
    lp, h, far = np.full(rows, np.nan), np.full(rows, np.nan), np.zeros(rows)
    ids, tl = np.full((rows, top_n), -1, np.int32), np.full((rows, top_n), -np.inf)
    for r in range(rows):
        live = np.isfinite(x[r])
        bad = np.isnan(x[r]).any() or (x[r] == np.inf).any()
        m = x[r][live].max() if live.any() else 0.0
        d = (x[r] - m) / t
        e = np.exp(d[live])
        z = e.sum()
        lz = np.nan if bad else np.log(z) if live.any() else 0.0
        if live.any():
            far[r] = (e * -d[live]).sum() / z
        h[r] = lz + far[r]
        i = int(tokens[r])
        lp[r] = 0.0 if i < 0 else np.nan if i >= n or bad else d[i] - lz
        order = np.argsort(np.where(live, -x[r], np.inf), kind="stable")[:min(top_n, live.sum())]
        ids[r, :len(order)] = order
        tl[r, :len(order)] = d[order] - lz
    return lp, h, ids, tl, far
