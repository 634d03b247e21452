"""Narrow-type calls in CUDA graphs, without other kernels between them."""
import pytest
import torch

import clblas_b200 as cb
from tests.cases_narrow import quantize_reference
from tests.test_narrow_handover import Chain

pytestmark = pytest.mark.gpu

BF16 = cb.clblasB200Bfloat16


@pytest.mark.parametrize("side", ["left", "right"])
@pytest.mark.parametrize("T,O,K", [(48, 96, 512), (300, 1000, 264), (5000, 1504, 1024)])
def test_a_captured_chain_equals_waited_calls(T, O, K, side):
    """All calls of several steps in one graph, replayed back to back: the weight goes on changing from replay to replay."""
    side = cb.clblasLeft if side == "left" else cb.clblasRight
    captured, waited = Chain(T, O, K, 4, side), Chain(T, O, K, 4, side)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        captured.queue()
    for _ in range(3):
        graph.replay()
        waited.run(wait=True)
    torch.cuda.synchronize()
    for i in range(4):
        assert torch.equal(captured.sy[i], waited.sy[i]) and torch.equal(captured.qy[i], waited.qy[i]), i
        assert torch.equal(captured.sy2[i], waited.sy2[i]) and torch.equal(captured.qy2[i], waited.qy2[i]), i
    assert torch.equal(captured.w, waited.w) and cb.lib.clblasB200DeviceFault() == 0


def test_two_graphs_with_workspaces_at_once():
    """Column scales in two passes, packed products and orthogonalisations by the chain all take workspaces."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    sets = []
    for k in range(2):
        x = torch.randn(4608, 4096 + 64 * k, generator=gen, device="cuda").bfloat16()
        g = torch.randn(300, 420 + 10 * k, generator=gen, device="cuda")
        M, N = x.shape
        q, s = torch.zeros(M, N, dtype=torch.int8, device="cuda"), torch.zeros(N, device="cuda")
        c = torch.zeros(40, N, device="cuda")
        a = torch.randint(-127, 128, (40, M), generator=gen, device="cuda", dtype=torch.int32).to(torch.int8)
        o = torch.zeros(g.shape, dtype=torch.bfloat16, device="cuda")
        sets.append((x, g, q, s, a, c, o))

    def calls(x, g, q, s, a, c, o):
        M, N = x.shape
        cb.check(cb.clblasB200QuantizeI8(0, cb.clblasRight, M, N, BF16, x, 0, N, q, 0, N, s, 0))
        cb.check(cb.clblasB200I8gemm(0, 0, 0, 40, N, M, 1.0, a, 0, M, None, 0, q, 0, N, s, 0, 0.0, 0, c, 0, N))
        cb.check(cb.clblasB200Orthogonalize(0, *g.shape, 1, 5, None, 1.0, 0, g, 0, g.shape[1], 0, 0.0, o, 0, g.shape[1], 0))

    want = []
    for z in sets:
        calls(*z)
        torch.cuda.synchronize()
        want.append([t.clone() for t in (z[2], z[3], z[5], z[6])])
        for t in (z[2], z[3], z[5], z[6]):
            t.zero_()
    ref_q, ref_s = quantize_reference(sets[0][0], 0)
    assert torch.equal(want[0][0].cpu(), ref_q) and torch.equal(want[0][1].cpu(), ref_s)
    streams, graphs = [torch.cuda.Stream() for _ in sets], []
    torch.cuda.synchronize()
    for z, stream in zip(sets, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            calls(*z)
        graphs.append(graph)
    for _ in range(4):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for z, w in zip(sets, want):
        assert all(torch.equal(t, v) for t, v in zip((z[2], z[3], z[5], z[6]), w))
