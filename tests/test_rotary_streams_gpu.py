"""A Rotary dropped while its call is queued on another stream: its table stays until the call has run."""
import pytest

pytestmark = pytest.mark.gpu

HD = 64


@pytest.mark.parametrize("how", ["given", "current", "made elsewhere", "captured and eager"])
def test_dropped_while_queued(gpu, how):
    from cortexsdr_amd.rotary import Rotary

    torch = gpu
    q = torch.randn(50, 4, HD, device="cuda")
    p = torch.arange(1000, 1050, dtype=torch.int32, device="cuda")
    want = Rotary(HD, theta=5e5).apply(q, p)
    out = torch.zeros_like(q)
    busy = torch.randn(4096, 4096, device="cuda")
    other = torch.zeros_like(busy)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    if how == "made elsewhere":
        with torch.cuda.stream(side):
            rot = Rotary(HD, theta=5e5)
        runs, makes = torch.cuda.current_stream(), side
    else:
        rot = Rotary(HD, theta=5e5)
        runs, makes = side, torch.cuda.current_stream()
    if how == "captured and eager":
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            rot.apply(q, p, q_out=out)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        out.zero_()
        torch.cuda.synchronize()
    at = rot._turns.data_ptr()
    with torch.cuda.stream(runs):
        for _ in range(30):  # some 10 ms
            torch.mm(busy, busy, out=other)
        if how == "current":
            rot.apply(q, p, q_out=out)
    if how != "current":
        rot.apply(q, p, q_out=out, stream=runs)
    done = runs.record_event()
    del rot
    with torch.cuda.stream(makes):  # where the table's memory came from
        new = [torch.full((HD // 2,), 7.0, dtype=torch.float64, device="cuda") for _ in range(200)]
    if not done.query():
        assert all(t.data_ptr() != at for t in new)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_streams_in_turn(gpu):
    """One Rotary on several streams, as on its own."""
    from cortexsdr_amd.rotary import Rotary

    torch = gpu
    q = torch.randn(300, 4, HD, device="cuda")
    p = torch.arange(300, dtype=torch.int32, device="cuda")
    rot = Rotary(HD, layout="halves")
    want = rot.apply(q, p)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = [rot.apply(q, p, stream=streams[i % 3]) for i in range(12)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
