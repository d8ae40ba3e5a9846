"""A transformer layer in 8 bits as a serving loop runs it: norm with the residual, products, rotary
positions, a paged cache, the gated feed-forward; each operator's output against fp64 of what it was
given, the layer on another stream and as a captured graph."""
import numpy as np
import pytest

import q8_ref
from test_q8_gpu import check_linear, check_rows, norm_parts
from test_rotary_gpu import check as check_rotary

pytestmark = pytest.mark.gpu

H, HQ, HK, HD, F = 640, 8, 2, 64, 1100
EPS = 1e-5


class Layer:
    def __init__(self, torch, seed=0):
        from cortexsdr_amd import q8
        from cortexsdr_amd.rotary import Rotary

        g = torch.Generator(device="cuda").manual_seed(seed)
        mk = lambda r, c: torch.randn(r, c, generator=g, device="cuda") / c ** 0.5  # noqa: E731
        self.w = {k: q8.quantize(mk(r, c)) for k, r, c in
                  (("qkv", (HQ + 2 * HK) * HD, H), ("o", H, HQ * HD), ("gu", 2 * F, H), ("down", H, F))}
        self.norms = [1 + 0.2 * torch.randn(H, generator=g, device="cuda") for _ in range(2)]
        self.bias = 0.1 * torch.randn((HQ + 2 * HK) * HD, generator=g, device="cuda")
        self.rot = Rotary(HD, theta=5e5, dims=32, layout="halves", scaling="parts", factor=4.0, original=4096)

    def __call__(self, x, stream_in, batch, positions, dtype, keep=None, **on):
        from cortexsdr_amd import q8

        n1 = q8.rms_norm(x, self.norms[0], EPS, residual=stream_in, **on)
        qkv = q8.linear(self.w["qkv"], n1.rows, bias=self.bias, dtype=dtype, **on).unflatten(1, (-1, HD))
        q, k = self.rot.apply(qkv[:, :HQ], positions, k=qkv[:, HQ:HQ + HK], **on)
        batch.append(None, k, qkv[:, HQ + HK:], **on)
        att = batch.attend(q, **on)
        a = q8.quantize(att.flatten(1), **on)
        o = q8.linear(self.w["o"], a, dtype=dtype, **on)
        n2 = q8.rms_norm(o, self.norms[1], EPS, residual=n1.residual, residual_out=n1.residual, **on)
        gu = q8.linear(self.w["gu"], n2.rows, dtype=dtype, **on)
        d = q8.quantize(gu[:, F:], gate=gu[:, :F], **on)
        y = q8.linear(self.w["down"], d, dtype=dtype, **on)
        if keep is not None:
            keep.update(n1=n1, qkv=qkv, q=q, k=k, att=att, a=a, o=o, n2=n2, gu=gu, d=d, y=y)
        return y, n2.residual


def inputs(torch, B, T, dtype, res, seed=1):
    from cortexsdr_amd.paged import PagedCache

    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B * T, H, generator=g, device="cuda").to(dtype)
    s = (2 * torch.randn(B * T, H, generator=g, device="cuda")).to(res)
    table = torch.arange(B * 6, dtype=torch.int32, device="cuda").reshape(B, 6)
    lens = torch.full((B,), 70 + T, dtype=torch.int32, device="cuda")
    pos = torch.arange(70, 70 + T, dtype=torch.int32, device="cuda").repeat(B)
    batch = PagedCache(B * 6, 32, HK, HD, "f16").batch(table, lens)
    batch.append(None, torch.randn(B * (70 + T), HK, HD, generator=g, device="cuda"),
                 torch.randn(B * (70 + T), HK, HD, generator=g, device="cuda"))
    return x, s, batch, pos


@pytest.mark.parametrize("B,T,dtype,res", [(1, 1, "f32", "f32"), (5, 1, "f16", "f32"), (2, 50, "f16", "f16"),
                                           (3, 33, "f32", "f32")])
def test_layer(gpu, B, T, dtype, res):
    torch = gpu
    types = dict(f32=torch.float32, f16=torch.float16)
    layer = Layer(torch)
    x, s, batch, pos = inputs(torch, B, T, types[dtype], types[res])
    k = {}
    stream_before = s.clone()
    layer(x, s, batch, pos, dtype, k)
    assert torch.equal(s, stream_before)  # the second norm updated its own stream
    host = lambda t: t.cpu().numpy()  # noqa: E731
    codes = lambda r: (host(r.codes)[:, :r.n], host(r.scales))  # noqa: E731
    h1 = (host(x).astype(np.float32) + host(s).astype(np.float32)).astype(host(s).dtype)
    rms, t = norm_parts(h1, host(layer.norms[0]), EPS)
    check_rows(k["n1"].rows, t, rms, extra=H * 2.0 ** -52)
    check_linear(k["qkv"].flatten(1), *codes(k["n1"].rows), *codes(layer.w["qkv"]), host(layer.bias))
    from cortexsdr_amd.rotary import frequencies
    f = frequencies(32, 5e5, "parts", 4.0, 4096)
    check_rotary(k["q"], host(k["qkv"][:, :HQ]), host(pos), f, "halves")
    check_rotary(k["k"], host(k["qkv"][:, HQ:HQ + HK]), host(pos), f, "halves")
    check_rows(k["a"], host(k["att"].flatten(1)))
    check_linear(k["o"], *codes(k["a"]), *codes(layer.w["o"]))
    h2 = (host(k["o"]).astype(np.float32) + h1.astype(np.float32)).astype(h1.dtype)
    np.testing.assert_array_equal(host(k["n2"].residual), h2)
    rms, t = norm_parts(h2, host(layer.norms[1]), EPS)
    check_rows(k["n2"].rows, t, rms, extra=H * 2.0 ** -52)
    check_linear(k["gu"], *codes(k["n2"].rows), *codes(layer.w["gu"]))
    check_rows(k["d"], q8_ref.silu_mul(host(k["gu"][:, :F]), host(k["gu"][:, F:])))
    check_linear(k["y"], *codes(k["d"]), *codes(layer.w["down"]))


@pytest.mark.parametrize("B,T", [(4, 1), (2, 90)])
def test_layer_captured(gpu, B, T):
    """Two graphs of the layer on two inputs, replayed in turn with eager work between: as eager, bit
    for bit; and a stream of its own."""
    torch = gpu
    layer = Layer(torch)
    sets = [inputs(torch, B, T, torch.float16, torch.float32, seed=i) for i in (1, 2)]
    want = [[t.clone() for t in layer(*s, "f16")] for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = layer(*sets[0], "f16", stream=side)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = layer(*s, "f16")
        graphs.append((g, out))
    for i in (0, 1, 1, 0, 0, 1):
        graphs[i][0].replay()
        layer(*sets[1 - i], "f16")
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(graphs[i][1], want[i])), i
