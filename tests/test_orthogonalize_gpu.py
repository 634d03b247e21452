"""clblasB200Orthogonalize on a B200 against the definition in 64 bits, with the bound that its roundings give."""
import math

import pytest
import torch

import clblas_b200 as cb
from tests.cases_narrow import HALF_STEP, QUINTIC, TYPES, Stored, orth_bound, orth_exact, order_code

pytestmark = pytest.mark.gpu


class Problem:
    def __init__(self, order, M, N, batch=1, kind="bf16", pad=0, off=0, gap=0, seed=0, spectrum="normal"):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.order, self.M, self.N, self.kind = order, M, N, kind
        self.g = Stored(order, M, N, "n", pad, off, TYPES[kind][0], batch, gap)
        self.o = Stored(order, M, N, "n", pad, off, torch.bfloat16, batch, gap)
        self.o.buf.copy_(torch.randn(self.o.buf.shape, generator=gen, device="cuda"))
        self.g.buf.copy_(torch.randn(self.g.buf.shape, generator=gen, device="cuda"))
        if spectrum != "normal":
            r = min(M, N)
            for i in range(batch):
                u = torch.randn(M, r, generator=gen, device="cuda")
                v = torch.randn(r, N, generator=gen, device="cuda")
                w = {"decaying": 1.0 / torch.arange(1, r + 1, device="cuda") ** 2, "rank8": (torch.arange(r, device="cuda") < 8).float(),
                     "rank1": (torch.arange(r, device="cuda") < 1).float()}[spectrum]
                self.g.op()[i].copy_((u * w) @ v)

    def call(self, steps=5, coefficients=None, alpha=1.0, beta=0.0, **kw):
        g, o = self.g, self.o
        return cb.clblasB200Orthogonalize(order_code(self.order), self.M, self.N, g.batch, steps, coefficients, alpha, TYPES[self.kind][1],
                                          g.buf, g.off, g.ld, g.stride, beta, o.buf, o.off, o.ld, o.stride, **kw)

    def check(self, steps=5, coefficients=None, alpha=1.0, beta=0.0, **kw):
        chain = coefficients or [QUINTIC] * steps
        before, o0 = self.o.buf.clone(), self.o.op().double().clone()
        g0 = self.g.buf.clone()
        cb.check(self.call(steps, coefficients, alpha, beta, **kw), "orthogonalize")
        for i in range(self.g.batch):
            x = orth_exact(self.g.op()[i].double(), chain)
            want = alpha * x + (beta * o0[i] if beta else 0.0)
            err = float((self.o.op()[i].double() - want).norm())
            inner = abs(alpha) * orth_bound(self.g.op()[i], chain) + 2.0 ** -23 * (abs(alpha) * float(x.norm()) + abs(beta) * float(o0[i].norm()))
            bound = inner + HALF_STEP["bf16"] * (float(want.norm()) + inner)
            assert err <= bound, (self.M, self.N, i, err / float(want.norm()), bound / float(want.norm()))
        m = self.o.outside()
        assert torch.equal(self.o.buf[m], before[m]) and torch.equal(self.g.buf, g0)
        return err / max(float(want.norm()), 1e-30)


# one row or column; sizes round the tiles of 128 and 256; wide, tall, square
SIZES = [(1, 1), (1, 300), (17, 1), (5, 3), (64, 64), (127, 129), (128, 256), (130, 700), (700, 130), (256, 1024), (300, 300), (513, 511), (1003, 601)]


@pytest.mark.parametrize("M,N", SIZES)
@pytest.mark.parametrize("order", ["row", "col"])
def test_sizes(M, N, order):
    Problem(order, M, N, seed=M + N).check()


@pytest.mark.parametrize("M,N", [(2100, 2300), (2304, 4096), (3000, 1100)])
def test_large(M, N):
    """Enough tiles for the persistent kernels, one CTA and pairs of CTAs."""
    assert Problem("row", M, N, seed=1).check() < 4e-3


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("spectrum", ["normal", "decaying", "rank8", "rank1"])
@pytest.mark.parametrize("M,N", [(100, 130), (384, 1024), (600, 260)])
def test_types_and_spectra(kind, spectrum, M, N):
    Problem("row", M, N, kind=kind, spectrum=spectrum, seed=2).check()


@pytest.mark.parametrize("order", ["row", "col"])
@pytest.mark.parametrize("M,N", [(200, 333), (333, 200)])
@pytest.mark.parametrize("pad,off,gap", [(0, 0, 0), (3, 5, 11), (8, 8, 64)])
def test_batches_and_layouts(order, M, N, pad, off, gap):
    Problem(order, M, N, batch=5, kind="f32", pad=pad, off=off, gap=gap, seed=3).check(alpha=-0.02, beta=0.99)


@pytest.mark.parametrize("steps,coefficients", [(1, None), (2, None), (8, None), (3, [(1.5, -0.5, 0.0)] * 3), (4, [(4.0, -6.0, 2.8), (3.9, -5.6, 2.6), (3.0, -3.2, 1.2), (1.875, -1.25, 0.375)])])
@pytest.mark.parametrize("M,N", [(150, 260), (260, 150)])
def test_steps_and_coefficients(steps, coefficients, M, N):
    Problem("row", M, N, seed=5).check(steps, coefficients, alpha=2.0)


@pytest.mark.parametrize("M,N", [(90, 200), (200, 90)])
def test_zero_and_non_finite_matrices_stay_among_themselves(M, N):
    p = Problem("row", M, N, batch=5, kind="f32", seed=6)
    g = p.g.op()
    g[1] = 0
    g[2, 3, 4] = math.nan
    g[3, 5, 6] = -math.inf
    g[4] *= 1e36                                            # the squares leave FP32: the norm is taken in 64 bits
    p.o.buf.fill_(math.nan)                                 # beta == 0 never reads O
    cb.check(p.call(), "orthogonalize")
    o = p.o.op()
    assert not o[1].any() and bool(o[2].isnan().all()) and bool(o[3].isnan().all())
    for i in (0, 4):
        want = orth_exact(g[i].double(), [QUINTIC] * 5)
        bound = orth_bound(g[i], [QUINTIC] * 5)
        assert float((o[i].double() - want).norm()) <= bound + HALF_STEP["bf16"] * (float(want.norm()) + bound)


def test_in_place_and_side_by_side():
    """O on top of G, and the matrices of a batch as column blocks of one wide matrix."""
    p = Problem("row", 96, 160, batch=3, seed=7)
    p.o = p.g
    g0 = p.g.op().double().clone()
    cb.check(p.call(), "orthogonalize")
    for i in range(3):
        want = orth_exact(g0[i], [QUINTIC] * 5)
        bound = orth_bound(g0[i], [QUINTIC] * 5)
        assert float((p.g.op()[i].double() - want).norm()) <= bound + HALF_STEP["bf16"] * (float(want.norm()) + bound)
    M, N, batch = 60, 50, 4
    gen = torch.Generator(device="cuda").manual_seed(8)
    wide = torch.randn(M, N * batch, generator=gen, device="cuda")
    out = torch.zeros(M, N * batch, dtype=torch.bfloat16, device="cuda")
    cb.check(cb.clblasB200Orthogonalize(cb.clblasRowMajor, M, N, batch, 5, None, 1.0, cb.clblasB200Float32, wide, 0, N * batch, N, 0.0, out, 0, N * batch, N), "wide")
    for i in range(batch):
        g = wide[:, i * N:(i + 1) * N].double()
        want, bound = orth_exact(g, [QUINTIC] * 5), orth_bound(g, [QUINTIC] * 5)
        assert float((out[:, i * N:(i + 1) * N].double() - want).norm()) <= bound + HALF_STEP["bf16"] * (float(want.norm()) + bound)


def test_same_call_twice_is_identical():
    for M, N, batch in ((256, 1024, 1), (700, 701, 4)):
        p = Problem("row", M, N, batch=batch, seed=9)
        cb.check(p.call(), "first")
        first = p.o.buf.clone()
        for _ in range(5):
            cb.check(p.call(), "again")
        assert torch.equal(first, p.o.buf)


def test_two_streams_and_two_graphs():
    """Calls that overlap on two streams, and two captured calls replayed at once, keep their workspaces apart."""
    ps = [Problem("row", 300, 500 + 60 * i, seed=10 + i) for i in range(2)]
    want = []
    for p in ps:
        cb.check(p.call(), "alone")
        want.append(p.o.op().clone())
        p.o.buf.zero_()
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()
    for _ in range(3):
        for p, s in zip(ps, streams):
            cb.check(p.call(queues=[s]), "streams")
    torch.cuda.synchronize()
    assert all(torch.equal(p.o.op(), w) for p, w in zip(ps, want))
    graphs = []
    for p, s in zip(ps, streams):
        p.o.buf.zero_()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            cb.check(p.call(), "captured")
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p.o.op(), w) for p, w in zip(ps, want))


def test_refusals():
    p = Problem("row", 24, 40, batch=2)
    G, O = p.g.buf, p.o.buf
    def go(order=0, M=24, N=40, batch=2, steps=5, co=None, T=2, G=G, offG=0, ldg=40, sg=960, O=O, offO=0, ldo=40, so=960, **kw):
        return cb.clblasB200Orthogonalize(order, M, N, batch, steps, co, 1.0, T, G, offG, ldg, sg, 0.0, O, offO, ldo, so, **kw)
    assert go() == cb.clblasSuccess
    assert go(G=None) == cb.clblasInvalidMatA and go(O=None) == cb.clblasInvalidMatC
    assert go(order=2) == cb.clblasInvalidValue and go(T=3) == cb.clblasInvalidValue
    assert go(steps=0) == cb.clblasInvalidValue and go(steps=65) == cb.clblasInvalidValue
    assert go(steps=1, co=[(1.0, math.nan, 0.0)]) == cb.clblasInvalidValue and go(steps=1, co=[(math.inf, 1.0, 0.0)]) == cb.clblasInvalidValue
    assert go(M=0) == cb.clblasInvalidDim and go(N=0) == cb.clblasInvalidDim and go(batch=0) == cb.clblasInvalidDim
    assert go(ldg=39) == cb.clblasInvalidLeadDimA and go(ldo=39) == cb.clblasInvalidLeadDimC
    assert go(so=959) == cb.clblasInvalidLeadDimC and go(so=0) == cb.clblasInvalidLeadDimC
    big = 1 << 34
    assert go(offG=big) == cb.clblasInsufficientMemMatA and go(offO=big) == cb.clblasInsufficientMemMatC
    assert go(sg=big) == cb.clblasInsufficientMemMatA and go(so=big) == cb.clblasInsufficientMemMatC
    assert go(sg=(1 << 64) - 1) == cb.clblasInsufficientMemMatA
    assert go(sg=0) == cb.clblasSuccess                     # the same G for every O
    assert go(queues=[]) == cb.clblasInvalidCommandQueue
    with pytest.raises(ValueError):
        go(steps=2, co=[(1.0, 2.0, 3.0)])
    assert cb.lib.clblasB200DeviceFault() == 0


# The single kernel for small matrices: clusters of 1, 2, 4, 8 CTAs, widths of 64 to 256 columns per CTA, the sizes just beyond it.
SMALL = [(1, 64), (64, 64), (65, 65), (128, 128), (33, 257), (100, 500), (128, 640), (127, 1025), (90, 1600), (128, 2048), (128, 2049), (129, 2048)]


@pytest.mark.parametrize("n,m", SMALL)
@pytest.mark.parametrize("tall", [False, True])
def test_small_sizes(n, m, tall):
    Problem("row", *((m, n) if tall else (n, m)), kind="f32" if n % 2 else "bf16", seed=n + m).check()


@pytest.mark.parametrize("order", ["row", "col"])
@pytest.mark.parametrize("M,N,batch", [(70, 300, 5), (300, 70, 5), (120, 900, 17), (50, 60, 150)])
@pytest.mark.parametrize("kind,pad,off,gap", [("f32", 0, 0, 0), ("f32", 3, 5, 11), ("bf16", 8, 8, 64), ("f16", 2, 2, 6), ("bf16", 1, 3, 5)])
def test_small_batches_and_layouts(order, M, N, batch, kind, pad, off, gap):
    Problem(order, M, N, batch=batch, kind=kind, pad=pad, off=off, gap=gap, seed=4).check(alpha=-0.02, beta=0.99)


@pytest.mark.parametrize("steps,coefficients", [(1, None), (2, None), (64, [(1.5, -0.5, 0.0)] * 64), (3, [(1.5, -0.5, 0.0), (3.4445, -4.775, 2.0315), (1.875, -1.25, 0.375)])])
@pytest.mark.parametrize("M,N", [(100, 260), (260, 100)])
def test_small_steps_and_coefficients(steps, coefficients, M, N):
    Problem("row", M, N, seed=5).check(steps, coefficients, alpha=2.0)


def test_small_is_deterministic_on_streams_and_in_graphs():
    ps = [Problem("row", 100, 500 + 300 * i, batch=3, seed=20 + i) for i in range(3)]
    want = []
    for p in ps:
        cb.check(p.call(), "alone")
        want.append(p.o.op().clone())
        p.o.buf.zero_()
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()
    for _ in range(5):
        for p, s in zip(ps, streams):
            cb.check(p.call(queues=[s]), "streams")
    torch.cuda.synchronize()
    assert all(torch.equal(p.o.op(), w) for p, w in zip(ps, want))
    p, s = ps[0], streams[0]
    p.o.buf.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        cb.check(p.call(), "captured")
        cb.check(p.call(), "captured")
    g.replay()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(p.o.op(), want[0]) and cb.lib.clblasB200DeviceFault() == 0
