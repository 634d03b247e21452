"""clblasB200I8gemm on a B200 against 64-bit products of the same integers; the tolerance counts the roundings of the definition."""
import math

import pytest
import torch

import clblas_b200 as cb
from tests.cases_narrow import TYPES, Stored, i8gemm_bound, order_code, random_i8

pytestmark = pytest.mark.gpu

TR = {"n": cb.clblasNoTrans, "t": cb.clblasTrans, "c": cb.clblasConjTrans}


class Problem:
    def __init__(self, order, ta, tb, M, N, K, kind, pad=0, off=0, seed=0, scales=True, c_rms=100.0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.args = (order, ta, tb, M, N, K, kind)
        self.a = Stored(order, M, K, ta.replace("c", "t"), pad, off, torch.int8)
        self.b = Stored(order, K, N, tb.replace("c", "t"), pad, off, torch.int8)
        random_i8(self.a, gen)
        random_i8(self.b, gen)
        self.c = Stored(order, M, N, "n", pad, off, TYPES[kind][0])
        self.c.buf.copy_(torch.randn(self.c.buf.shape, generator=gen, device="cuda") * c_rms)
        self.sa = torch.exp(torch.randn(M, generator=gen, device="cuda")) * 1e-2 if scales else None
        self.sb = torch.exp(torch.randn(N, generator=gen, device="cuda")) * 1e-2 if scales else None

    def call(self, alpha=1.0, beta=0.0, **kw):
        order, ta, tb, M, N, K, kind = self.args
        a, b, c = self.a, self.b, self.c
        return cb.clblasB200I8gemm(order_code(order), TR[ta], TR[tb], M, N, K, alpha, a.buf, a.off, a.ld, self.sa, 0, b.buf, b.off, b.ld, self.sb, 0,
                                   beta, TYPES[kind][1], c.buf, c.off, c.ld, **kw)

    def check(self, alpha=1.0, beta=0.0, **kw):
        order, ta, tb, M, N, K, kind = self.args
        before = self.c.buf.clone()
        c0 = self.c.op()[0].double().clone()
        cb.check(self.call(alpha, beta, **kw), "i8gemm")
        got = self.c.op()[0].double()
        total = self.a.op()[0].double() @ self.b.op()[0].double()            # exact: below 2^53
        sa = self.sa.double() if self.sa is not None else torch.ones(M, dtype=torch.float64, device="cuda")
        sb = self.sb.double() if self.sb is not None else torch.ones(N, dtype=torch.float64, device="cuda")
        want = alpha * total * sa[:, None] * sb[None, :] + (beta * c0 if beta else 0.0)
        bound = i8gemm_bound(total, sa, sb, alpha, beta, c0, kind)
        off = (got - want).abs() - bound
        if kind == "f16":
            # Rounding to nearest takes every value of 65504 + half a step (16) or more to infinity: where the exact value may lie
            # there, an infinity of its sign is the rounded result.
            off = torch.where(got.isinf() & (got.sign() == want.sign()) & (want.abs() + bound >= 65520.0), torch.zeros_like(off), off)
        assert float(off.max()) <= 0, (self.args, float(off.max()))
        m = self.c.outside()
        assert torch.equal(self.c.buf[m], before[m])


# one token; few tokens; sizes round the tiles of 32, 64, 128 and 256; long and short k
SIZES = [(1, 1, 1), (1, 4096, 4096), (3, 130, 17), (32, 256, 128), (33, 1000, 300), (64, 512, 1024), (65, 640, 2056), (128, 129, 127), (129, 128, 129),
         (130, 300, 512), (257, 255, 64), (512, 512, 4096), (300, 20, 700), (1000, 64, 333), (2000, 2100, 140), (2304, 2560, 96)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("order", ["row", "col"])
def test_sizes(M, N, K, order):
    Problem(order, "n", "t", M, N, K, "bf16", seed=M + N + K).check()


@pytest.mark.parametrize("order", ["row", "col"])
@pytest.mark.parametrize("ta", ["n", "t", "c"])
@pytest.mark.parametrize("tb", ["n", "t", "c"])
@pytest.mark.parametrize("pad,off", [(0, 0), (5, 3), (16, 32)])
def test_layouts(order, ta, tb, pad, off):
    for M, N, K in ((40, 200, 272), (260, 390, 129), (1700, 1500, 65)):
        Problem(order, ta, tb, M, N, K, "f32", pad, off, seed=K).check()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("alpha,beta", [(1.0, 0.0), (-0.5, 1.0), (2.0, -0.75)])
@pytest.mark.parametrize("M,N,K", [(7, 500, 600), (200, 200, 2000), (500, 40, 300), (1800, 1555, 200)])
def test_types_alpha_beta(kind, alpha, beta, M, N, K):
    for order in ("row", "col"):
        Problem(order, "n", "t", M, N, K, kind, pad=8, seed=3).check(alpha, beta)


@pytest.mark.parametrize("M,N", [(1, 200), (300, 300), (1600, 1700)])
def test_extreme_sums_and_no_scales(M, N):
    """All operands -128 at the longest k: the sum is 131071 * 16384, just below 2^31, and no scale is given."""
    K = 131071
    p = Problem("row", "n", "t", M, N, K, "f32", scales=False)
    p.a.buf.fill_(-128)
    p.b.buf.fill_(-128)
    cb.check(p.call(), "i8gemm")
    assert bool((p.c.op() == float(torch.tensor(131071 * 16384, dtype=torch.int64).float())).all())


@pytest.mark.parametrize("M,N", [(5, 300), (200, 300), (1600, 1800)])
def test_nan_in_unread_c_and_scales(M, N):
    p = Problem("row", "n", "t", M, N, 256, "bf16")
    p.c.op().fill_(math.nan)                                # beta == 0 never reads C
    p.check()
    p.sa[M // 2] = math.nan                                 # the scale of a row that could not be quantised
    cb.check(p.call(), "i8gemm")
    got = p.c.op()[0]
    assert bool(got[M // 2].isnan().all()) and int(got.isnan().sum()) == N


def test_alpha_zero_and_k_zero():
    for K, alpha in ((64, 0.0), (0, 1.0)):
        for beta in (0.0, 0.5, 1.0):
            p = Problem("row", "n", "t", 70, 90, max(K, 1), "f16", pad=3)
            p.args = p.args[:5] + (K,) + p.args[6:]
            c0 = p.c.op()[0].clone()
            cb.check(p.call(alpha, beta), "i8gemm")
            want = (c0.float() * beta).half() if beta else torch.zeros_like(c0)
            assert torch.equal(p.c.op()[0], want)


def test_same_call_twice_is_identical():
    for M, N, K in ((1, 4096, 4096), (48, 1024, 8192), (300, 300, 3000)):
        p = Problem("row", "n", "t", M, N, K, "f32", seed=9)
        cb.check(p.call(), "i8gemm")
        first = p.c.buf.clone()
        for _ in range(5):
            cb.check(p.call(), "i8gemm")
        assert torch.equal(first, p.c.buf)


def test_streams_events_and_graph():
    """On a stream of its own behind an event, and captured (workspace and all) and replayed on new inputs."""
    p = Problem("row", "n", "n", 300, 520, 700, "bf16", pad=3, seed=4)
    side, ready, done = torch.cuda.Stream(), torch.cuda.Event(), torch.cuda.Event()
    ready.record()
    done.record()
    cb.check(p.call(queues=[side], wait=[ready], events=[done]), "i8gemm")
    done.synchronize()
    first = p.c.buf.clone()
    p.c.buf.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        cb.check(p.call(), "warm")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        cb.check(p.call(), "captured")
    p.a.buf.neg_()
    p.a.buf.clamp_(-127, 127)
    g.replay()
    torch.cuda.synchronize()
    second = p.c.op()[0].clone()
    p.check()
    assert torch.equal(second, p.c.op()[0]) and not torch.equal(first, p.c.buf)


def test_refusals():
    p = Problem("row", "n", "t", 16, 32, 48, "bf16")
    f = cb.clblasB200I8gemm
    a, b, c, sa, sb = p.a.buf, p.b.buf, p.c.buf, p.sa, p.sb
    def go(order=0, ta=0, tb=1, M=16, N=32, K=48, A=a, offA=0, lda=48, SA=sa, oSA=0, B=b, offB=0, ldb=48, SB=sb, oSB=0, T=2, C=c, offC=0, ldc=32, **kw):
        return f(order, ta, tb, M, N, K, 1.0, A, offA, lda, SA, oSA, B, offB, ldb, SB, oSB, 0.0, T, C, offC, ldc, **kw)
    assert go() == cb.clblasSuccess
    assert go(A=None) == cb.clblasInvalidMatA and go(B=None) == cb.clblasInvalidMatB and go(C=None) == cb.clblasInvalidMatC
    assert go(order=7) == cb.clblasInvalidValue and go(ta=3) == cb.clblasInvalidValue and go(T=5) == cb.clblasInvalidValue
    assert go(M=0) == cb.clblasInvalidDim and go(N=0) == cb.clblasInvalidDim
    assert go(lda=47) == cb.clblasInvalidLeadDimA and go(ldb=47) == cb.clblasInvalidLeadDimB and go(ldc=31) == cb.clblasInvalidLeadDimC
    big = 1 << 34
    assert go(offA=big) == cb.clblasInsufficientMemMatA and go(offB=big) == cb.clblasInsufficientMemMatB and go(offC=big) == cb.clblasInsufficientMemMatC
    assert go(oSA=big) == cb.clblasInsufficientMemVecX and go(oSB=big) == cb.clblasInsufficientMemVecY
    assert go(SA=1 << 20) == cb.clblasInvalidVecX and go(SB=1 << 20) == cb.clblasInvalidVecY
    assert go(queues=[]) == cb.clblasInvalidCommandQueue
    assert go(wait=[None]) == cb.clblasInvalidEventWaitList
    wide = torch.zeros(131072 * 4, dtype=torch.int8, device="cuda")
    assert f(0, 0, 1, 1, 1, 131072, 1.0, wide, 0, 131072, None, 0, wide, 0, 131072, None, 0, 0.0, 0, torch.zeros(1, device="cuda"), 0, 1) == cb.clblasInvalidDim
    assert cb.lib.clblasB200DeviceFault() == 0


@pytest.mark.parametrize("order", ["row", "col"])
def test_linear_layer_as_it_is_used(order):
    """Weights quantised per channel once, activations per token, then the product: within the quantisation's own error of the 64-bit layer."""
    T, O, K = 70, 384, 1024
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, w = (Stored(order, r, K, dtype=torch.bfloat16) for r in (T, O))
    for m in (x, w):
        m.buf.copy_(torch.randn(m.buf.shape, generator=gen, device="cuda"))
    qx, qw = (Stored(order, r, K, dtype=torch.int8) for r in (T, O))
    sx, sw = torch.zeros(T, device="cuda"), torch.zeros(O, device="cuda")
    for m, q, s, r in ((x, qx, sx, T), (w, qw, sw, O)):
        cb.check(cb.clblasB200QuantizeI8(order_code(order), cb.clblasLeft, r, K, cb.clblasB200Bfloat16, m.buf, 0, m.ld, q.buf, 0, q.ld, s, 0), "quantize")
    y = Stored(order, T, O, dtype=torch.float32)
    cb.check(cb.clblasB200I8gemm(order_code(order), cb.clblasNoTrans, cb.clblasTrans, T, O, K, 1.0, qx.buf, 0, qx.ld, sx, 0, qw.buf, 0, qw.ld, sw, 0,
                                 0.0, cb.clblasB200Float32, y.buf, 0, y.ld), "i8gemm")
    xd, wd = x.op()[0].double(), w.op()[0].double()
    # |x - s q| <= 0.51 s for both factors: |sum| is off by at most 0.51 (sx |w| + sw |x|) + 0.26 sx sw per term
    bound = 0.51 * (sx.double()[:, None] * wd.abs().sum(1)[None, :] + sw.double()[None, :] * xd.abs().sum(1)[:, None]) + K * 0.27 * sx.double()[:, None] * sw.double()[None, :]
    err = (y.op()[0].double() - xd @ wd.t()).abs()
    assert bool((err <= bound).all())
