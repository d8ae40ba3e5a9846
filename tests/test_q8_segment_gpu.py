"""From the framework's coded weights to 8-bit ones: a segment decoded, quantised and multiplied, against the
product of its codes."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R,C,M", [(300, 1024, 3), (700, 896, 70)])
def test_segment_in_8_bits(gpu, R, C, M):
    from cortexsdr_amd import q8, synth
    from cortexsdr_amd.hsdr import HsdbSegment

    seg = HsdbSegment(synth.hsdb_layer(R, C, 512, 8, seed_dict=1, seed_codes=2))
    dense = seg.decompress()
    w = q8.quantize(dense)
    x = gpu.from_numpy(np.random.default_rng(3).standard_normal((M, C)).astype(np.float32)).cuda()
    rows = q8.quantize(x)
    y = q8.linear(w, rows).cpu().numpy().astype(np.float64)
    coded = seg.matmul(x.t().contiguous()).cpu().numpy().T
    seg.free()
    # each value is off by half a scale at most (and the scale's own rounding)
    ws, xs = w.scales.cpu().numpy()[None] * 0.5001, rows.scales.cpu().numpy()[:, None] * 0.5001
    aw, ax = np.abs(dense.cpu().numpy()).astype(np.float64), np.abs(x.cpu().numpy()).astype(np.float64)
    bound = ax.sum(1)[:, None] * ws + aw.sum(1)[None] * xs + C * xs * ws
    # the product of the codes itself: fp16 dictionary and weights at most, 2^-10 of the terms' magnitudes
    bound = bound + 2.0 ** -10 * (ax @ aw.T)
    assert (np.abs(y - coded) <= bound).all()
    # and nearer than that in the mean: errors of random sign
    assert np.abs(y - coded).mean() <= 0.1 * bound.mean()
