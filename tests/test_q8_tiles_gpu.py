"""Every tile of the 8-bit products with fewer stages of columns than it has in flight, as many and more, at rests of
rows, tokens and columns (tests/q8_tiles.py), against exact sums in fp64 (tests/q8_ref.py)."""
import numpy as np
import pytest

import q8_ref
from q8_tiles import CASES
from test_q8_gpu import NP, check_sums, dev, random_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,R,C,stages,tile", [(*c, t) for t, cases in CASES.items() for c in cases],
                         ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else str(v))
def test_tile(gpu, M, R, C, stages, tile):
    from cortexsdr_amd import q8

    xc, xs, x = random_rows(gpu, M, C, seed=M + C)
    wc, ws, _ = random_rows(gpu, R, C, seed=R)
    ws = (ws / C).astype(np.float32)  # within fp16
    w = q8.Q8Rows.pack(dev(gpu, wc), dev(gpu, ws))
    sums = q8_ref.sums(xc, wc)
    check_sums(q8.linear(w, x), sums, xs, ws)
    r = np.random.default_rng(C)
    bias = r.standard_normal(R).astype(np.float32)
    for dtype in ("f32", "f16"):
        # onto rows of a larger buffer, whose other values stay
        wide = r.standard_normal((M, R + 3)).astype(NP[dtype])
        buf = dev(gpu, wide)
        out = buf[:, 1:1 + R]
        check_sums(q8.linear(w, x, bias=dev(gpu, bias), add=out, dtype=dtype, out=out), sums, xs, ws, bias,
                   wide[:, 1:1 + R])
        rest = buf.cpu().numpy()
        assert (rest[:, 0] == wide[:, 0]).all() and (rest[:, 1 + R:] == wide[:, 1 + R:]).all()
