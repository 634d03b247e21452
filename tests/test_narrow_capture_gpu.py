"""Narrow-type calls in CUDA graphs, without other kernels between them, and beside a capture of another thread."""
import os
import subprocess
import sys

import pytest
import torch

import clblas_b200 as cb
from tests.cases_narrow import quantize_reference
from tests.test_narrow_handover import Chain

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
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


OTHER_THREAD = """
import sys, threading, torch, clblas_b200 as cb
def make(seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    x = torch.randn(4608, 4096, generator=gen, device='cuda').bfloat16()
    a = torch.randint(-127, 128, (40, 4608), generator=gen, device='cuda', dtype=torch.int32).to(torch.int8)
    g, m = torch.randn(300, 420, generator=gen, device='cuda'), torch.randn(200, 300, generator=gen, device='cuda')
    t = torch.eye(200, device='cuda') * 16 + torch.randn(200, 200, generator=gen, device='cuda').tril()
    return (x, a, g, t, m), (torch.zeros_like(x, dtype=torch.int8), torch.zeros(4096, device='cuda'), torch.zeros(40, 4096, device='cuda'),
                          torch.zeros(300, 420, dtype=torch.bfloat16, device='cuda'))
def calls(z, stream):
    (x, a, g, t, m), (q, s, c, o) = z
    k = dict(queues=[stream])
    return [cb.clblasB200QuantizeI8(0, 1, 4608, 4096, 2, x, 0, 4096, q, 0, 4096, s, 0, **k),
            cb.clblasB200I8gemm(0, 0, 0, 40, 4096, 4608, 1.0, a, 0, 4608, None, 0, q, 0, 4096, s, 0, 0.0, 0, c, 0, 4096, **k),
            cb.clblasB200Orthogonalize(0, 300, 420, 1, 5, None, 1.0, 0, g, 0, 420, 0, 0.0, o, 0, 420, 0, **k),
            cb.clblasStrsm(0, 0, 1, 0, 1, 200, 300, 1.0, t, 0, 200, m, 0, 300, **k)]
assert cb.clblasSetup() == 0
a, b, want = make(1), make(2), make(2)
streams = [torch.cuda.Stream() for _ in range(2)]
torch.cuda.synchronize()
if sys.argv[1] == 'warm':
    assert calls(make(3), streams[0]) == [0] * 4
    torch.cuda.synchronize()
got, graph = [], torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=streams[0]):               # the global mode: nothing unsafe in any thread
    t = threading.Thread(target=lambda: got.append(calls(b, streams[1])))
    t.start(); t.join()
    got.append(calls(a, streams[0]))
graph.replay()
assert calls(want, streams[1]) == [0] * 4
torch.cuda.synchronize()
assert got == [[0] * 4] * 2, got
assert all(torch.equal(u, v) for u, v in zip(b[1], want[1])) and torch.equal(b[0][4], want[0][4])
assert int(a[1][0].abs().max()) == 127 and 15 < float(a[1][3].float().norm()) < 21
print('captured beside another thread')
"""


@pytest.mark.parametrize("state", ["cold", "warm"])
def test_calls_beside_another_threads_capture(state):
    """One thread captures while another makes calls with workspaces on a stream of its own: neither disturbs the other."""
    r = subprocess.run([sys.executable, "-c", OTHER_THREAD, state], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured beside another thread" in r.stdout, r.stderr[-2000:]
