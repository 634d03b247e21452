"""The narrow-type operators together, as a program uses them, and where calls meet: queued without waiting, captured first thing in
a process, from several threads, on buffers beyond 32-bit offsets."""
import os
import subprocess
import sys
import threading

import pytest
import torch

import clblas_b200 as cb
from tests.cases_narrow import HALF_STEP, QUINTIC, i8gemm_bound, orth_bound, orth_exact, quantize_reference

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, F32 = cb.clblasB200Bfloat16, cb.clblasB200Float32


class Layer:
    """A linear layer that is quantised, served in 8 bits and updated with an orthogonalised gradient."""

    def __init__(self, T, O, K, seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
        self.T, self.O, self.K = T, O, K
        self.w = (r(O, K) / K ** 0.5).bfloat16()
        self.x = [r(T, K).bfloat16() for _ in range(4)]
        self.g = [r(O, K).bfloat16() for _ in range(4)]
        self.qw, self.qx = (torch.zeros(n, K, dtype=torch.int8, device="cuda") for n in (O, T))
        self.sw, self.sx = torch.zeros(O, device="cuda"), torch.zeros(T, device="cuda")
        self.xin, self.gin = torch.empty_like(self.x[0]), torch.empty_like(self.g[0])
        self.y = torch.zeros(T, O, dtype=torch.bfloat16, device="cuda")

    def step(self, i, queues=None):
        """Everything queued: new inputs, both quantisations, the product, the update of the weight, inputs overwritten."""
        O, T, K = self.O, self.T, self.K
        self.xin.copy_(self.x[i % 4])
        self.gin.copy_(self.g[i % 4])
        cb.check(cb.clblasB200QuantizeI8(0, cb.clblasLeft, O, K, BF16, self.w, 0, K, self.qw, 0, K, self.sw, 0, queues=queues))
        cb.check(cb.clblasB200QuantizeI8(0, cb.clblasLeft, T, K, BF16, self.xin, 0, K, self.qx, 0, K, self.sx, 0, queues=queues))
        cb.check(cb.clblasB200I8gemm(0, 0, 1, T, O, K, 1.0, self.qx, 0, K, self.sx, 0, self.qw, 0, K, self.sw, 0, 0.0, BF16, self.y, 0, O, queues=queues))
        out = self.y.clone()
        cb.check(cb.clblasB200Orthogonalize(0, O, K, 1, 5, None, -0.02, BF16, self.gin, 0, K, 0, 0.99, self.w, 0, K, 0, queues=queues))
        self.xin.fill_(float("nan"))
        self.gin.fill_(float("nan"))
        return out


@pytest.mark.parametrize("T,O,K", [(1, 256, 384), (48, 512, 1024), (300, 1000, 264)])
def test_queued_steps_equal_waited_ones(T, O, K):
    """Kernels that may start before their predecessor has ended must not read or write early."""
    a, b = Layer(T, O, K, 1), Layer(T, O, K, 1)
    outs = [a.step(i) for i in range(12)]
    torch.cuda.synchronize()
    for i in range(12):
        want = b.step(i)
        torch.cuda.synchronize()
        assert torch.equal(outs[i], want), i
    assert torch.equal(a.w, b.w)


def test_one_step_against_64_bits():
    T, O, K = 40, 320, 512
    p = Layer(T, O, K, 2)
    w0 = p.w.double()
    y = p.step(0)
    total = p.qx.double() @ p.qw.double().t()
    want = total * p.sx.double()[:, None] * p.sw.double()[None, :]
    assert bool(((y.double() - want).abs() <= i8gemm_bound(total, p.sx.double(), p.sw.double(), 1.0, 0.0, want, "bf16")).all())
    q, s = quantize_reference(p.x[0], 1)
    assert torch.equal(p.qx.cpu(), q) and torch.equal(p.sx.cpu(), s)
    g = p.g[0].double()
    new = 0.99 * w0 - 0.02 * orth_exact(g, [QUINTIC] * 5)
    bound = 0.02 * orth_bound(g, [QUINTIC] * 5) + 2.0 ** -23 * float(new.norm())
    assert float((p.w.double() - new).norm()) <= bound + HALF_STEP["bf16"] * (float(new.norm()) + bound)


def test_threads_on_streams_of_their_own():
    layers = [Layer(16 + 5 * i, 256, 300, 3 + i) for i in range(4)]
    alone = []
    for i, p in enumerate(layers):
        alone.append([p.step(k) for k in range(3)][-1])
    torch.cuda.synchronize()
    again = [Layer(16 + 5 * i, 256, 300, 3 + i) for i in range(4)]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got[i] = [again[i].step(k) for k in range(3)][-1]
        s.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(torch.equal(a, b) for a, b in zip(got, alone))


FIRST = """
import torch, clblas_b200 as cb
a = torch.ones(300, 700, dtype=torch.int8, device='cuda'); b = torch.ones(700, 520, dtype=torch.int8, device='cuda')
c = torch.zeros(300, 520, device='cuda'); g = torch.eye(300, 500, device='cuda'); o = torch.zeros(300, 500, dtype=torch.bfloat16, device='cuda')
q = torch.zeros(300, 500, dtype=torch.int8, device='cuda'); s = torch.zeros(500, device='cuda')
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    r = [cb.clblasB200I8gemm(0, 0, 0, 300, 520, 700, 1.0, a, 0, 700, None, 0, b, 0, 520, None, 0, 0.0, 0, c, 0, 520),
         cb.clblasB200Orthogonalize(0, 300, 500, 1, 5, None, 1.0, 0, g, 0, 500, 0, 0.0, o, 0, 500, 0),
         cb.clblasB200QuantizeI8(0, 1, 300, 500, 0, g, 0, 500, q, 0, 500, s, 0)]
assert r == [0, 0, 0], r
graph.replay(); torch.cuda.synchronize()
assert bool((c == 700).all()) and int(q.sum()) == 300 * 127 and float(s[0]) > 0 and float(s[499]) == 0
x = 1 / (300 ** 0.5 + 1e-7)
for _ in range(5): x = x * (3.4445 - 4.775 * x ** 2 + 2.0315 * x ** 4)
d = o.float().diagonal()
assert float((d - x).abs().max()) < 0.01 * x and float((o.float().abs().sum() - d.abs().sum())) < 1.0
print('captured first')
"""


def test_first_call_of_a_process_may_be_captured():
    r = subprocess.run([sys.executable, "-c", FIRST], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stderr[-2000:]


def test_offsets_beyond_32_bits():
    """Small matrices behind 2^32 elements of their buffers."""
    far = (1 << 32) + 40
    M, N, K = 96, 160, 208
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.empty(far + 1 + M * K, dtype=torch.bfloat16, device="cuda")
    x[far + 1:] = torch.randn(M * K, generator=gen, device="cuda").bfloat16()
    q = torch.empty(far + M * K, dtype=torch.int8, device="cuda")
    s = torch.zeros(M, device="cuda")
    cb.check(cb.clblasB200QuantizeI8(0, cb.clblasLeft, M, K, BF16, x, far + 1, K, q, far, K, s, 0))
    want_q, want_s = quantize_reference(x[far + 1:].view(M, K), 1)
    got_q = q[far:].view(M, K)
    assert torch.equal(got_q.cpu(), want_q) and torch.equal(s.cpu(), want_s)
    b = torch.randint(-127, 128, (N, K), generator=gen, device="cuda", dtype=torch.int32).to(torch.int8)
    c = x                                                  # the product goes behind the large buffer's beginning, away from x's matrix
    off = 1 << 31
    cb.check(cb.clblasB200I8gemm(0, 0, 1, M, N, K, 1.0, q, far, K, s, 0, b, 0, K, None, 0, 0.0, BF16, c, off, N))
    total = got_q.double() @ b.double().t()
    want = total * s.double()[:, None]
    assert bool(((c[off:off + M * N].view(M, N).double() - want).abs()
                 <= i8gemm_bound(total, s.double(), torch.ones(N, dtype=torch.float64, device="cuda"), 1.0, 0.0, want, "bf16")).all())
    o = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    cb.check(cb.clblasB200Orthogonalize(0, M, K, 1, 5, None, 1.0, BF16, x, far + 1, K, 0, 0.0, o, 0, K, 0))
    g = x[far + 1:].view(M, K).double()
    ns, bound = orth_exact(g, [QUINTIC] * 5), orth_bound(g, [QUINTIC] * 5)
    assert float((o.double() - ns).norm()) <= bound + HALF_STEP["bf16"] * (float(ns.norm()) + bound)
    del x, q, c
    torch.cuda.empty_cache()


def test_result_beyond_32_bits():
    """More than 2^32 elements of C and of Q; a few lines of each against 64 bits."""
    n, K = 66000, 40
    gen = torch.Generator(device="cuda").manual_seed(6)
    a = torch.randint(-127, 128, (n, K), generator=gen, device="cuda", dtype=torch.int32).to(torch.int8)
    c = torch.empty(n, n, dtype=torch.bfloat16, device="cuda")
    cb.check(cb.clblasB200I8gemm(0, 0, 1, n, n, K, 1.0, a, 0, K, None, 0, a, 0, K, None, 0, 0.0, BF16, c, 0, n))
    q = torch.empty(n, n, dtype=torch.int8, device="cuda")
    s = torch.zeros(n, device="cuda")
    cb.check(cb.clblasB200QuantizeI8(0, cb.clblasLeft, n, n, BF16, c, 0, n, q, 0, n, s, 0))
    for rows in (slice(0, 3), slice(65070, 65075), slice(n - 3, n)):          # line 65075 lies behind element 2^32
        want = a[rows].double() @ a.double().t()
        assert torch.equal(c[rows].double(), want.bfloat16().double())
        wq, ws = quantize_reference(c[rows], 1)
        assert torch.equal(q[rows].cpu(), wq) and torch.equal(s[rows].cpu(), ws)
    t = torch.zeros(n, device="cuda")
    cb.check(cb.clblasB200QuantizeI8(0, cb.clblasRight, n, n, BF16, c, 0, n, q, 0, n, t, 0))
    top = torch.zeros(n, device="cuda")
    for i in range(0, n, 6000):
        top = torch.maximum(top, c[i:i + 6000].float().abs().amax(0))
    assert torch.equal(t, top / torch.full_like(top, 127.0))
    tail = c[n - 2:].float() * (torch.full_like(top, 127.0) / top)
    assert torch.equal(q[n - 2:], tail.round().to(torch.int8))
    del c, q
    torch.cuda.empty_cache()
    assert cb.lib.clblasB200DeviceFault() == 0
