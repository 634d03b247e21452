"""Buffers in memory that an allocator has mapped piece by piece (PyTorch's expandable segments): the driver knows such memory by its
pieces, but a buffer may span many."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import torch, clblas_b200 as cb
from tests.cases_narrow import quantize_reference, orth_exact, QUINTIC
assert cb.clblasSetup() == 0
for M, N in ((100, 1000), (3000, 9000), (16384, 8192)):                 # up to 268 MB; pieces are 2 and 20 MB
    x = torch.randn(M, N, device='cuda').bfloat16()
    q, s = torch.zeros(M, N, dtype=torch.int8, device='cuda'), torch.zeros(M, device='cuda')
    cb.check(cb.clblasB200QuantizeI8(0, 0, M, N, 2, x, 0, N, q, 0, N, s, 0))
    for rows in (slice(0, 2), slice(M - 2, M)):
        wq, ws = quantize_reference(x[rows], 1)
        assert torch.equal(q[rows].cpu(), wq) and torch.equal(s[rows].cpu(), ws)
    c = torch.zeros(M, 4000, device='cuda')
    cb.check(cb.clblasB200I8gemm(0, 0, 1, M, min(M, 4000), N, 1.0, q, 0, N, s, 0, q, 0, N, s, 0, 0.0, 0, c, 0, 4000))
    if M <= 4000:                                                       # the same product, its two scales in either order: three roundings each
        assert abs(float(c[M - 1, 0]) - float(c[0, M - 1])) <= 6 * 2.0 ** -24 * abs(float(c[0, M - 1]))
    assert float(c[M - 1].abs().sum()) > 0
    graph = torch.cuda.CUDAGraph()
    q.zero_()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        cb.check(cb.clblasB200QuantizeI8(0, 0, M, N, 2, x, 0, N, q, 0, N, s, 0))
    graph.replay()
    assert torch.equal(q[rows].cpu(), wq)
f, g = torch.randn(5000, 5000, device='cuda'), torch.randn(5000, 5000, device='cuda')
h = torch.zeros(5000, 5000, device='cuda')
cb.check(cb.clblasSgemm(0, 0, 0, 5000, 5000, 5000, 1.0, f, 0, 5000, g, 0, 5000, 0.0, h, 0, 5000))
assert float((h[4999].double() - f[4999].double() @ g.double()).abs().max()) < 0.05
b = torch.randn(300, 400, 500, device='cuda')                           # a batch of 240 MB
o = torch.zeros(300, 400, 500, dtype=torch.bfloat16, device='cuda')
cb.check(cb.clblasB200Orthogonalize(0, 400, 500, 300, 5, None, 1.0, 0, b, 0, 500, 200000, 0.0, o, 0, 500, 200000))
want = orth_exact(b[299].double(), [QUINTIC] * 5)
assert float((o[299].double() - want).norm()) < 5e-3 * float(want.norm())
# beyond everything that is mapped
far = 1 << 38
assert cb.clblasB200QuantizeI8(0, 0, 100, 1000, 2, x, far, 1000, q, 0, 1000, s, 0) == cb.clblasInsufficientMemMatA
assert cb.clblasB200Orthogonalize(0, 400, 500, 1 << 30, 5, None, 1.0, 0, b, 0, 500, 200000, 0.0, o, 0, 500, 200000) == cb.clblasInsufficientMemMatA
assert cb.clblasSgemm(0, 0, 0, 5000, 5000, 5000, 1.0, f, 0, 1 << 63, g, 0, 5000, 0.0, h, 0, 5000) == cb.clblasInsufficientMemMatA
torch.cuda.synchronize()
assert cb.device_fault() == 0
print('mapped memory ok')
"""


@pytest.mark.parametrize("setting", ["expandable_segments:True", "expandable_segments:False"])
def test_buffers_of_many_pieces(setting):
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=300,
                       env={**os.environ, "PYTORCH_CUDA_ALLOC_CONF": setting, "PYTORCH_ALLOC_CONF": setting})
    assert r.returncode == 0 and "mapped memory ok" in r.stdout, r.stderr[-2000:]
