"""clblasB200QuantizeI8 on a B200: the result is defined operation by operation in float32, so it is compared bit for bit with the
same operations on the CPU, and its distance from the values it stands for with the bound of a 64-bit evaluation."""
import math

import pytest
import torch

import clblas_b200 as cb
from tests.cases_narrow import TYPES, U32, Stored, order_code, quantize_reference

pytestmark = pytest.mark.gpu


def call(order, side, M, N, kind, x, q, scale, off_s=0, **kw):
    return cb.clblasB200QuantizeI8(order_code(order), cb.clblasLeft if side == "left" else cb.clblasRight, M, N, TYPES[kind][1],
                                   x.buf, x.off, x.ld, q.buf, q.off, q.ld, scale, off_s, **kw)


def build(order, M, N, kind, pad, off, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = Stored(order, M, N, pad=pad, off=off, dtype=TYPES[kind][0])
    v = torch.randn(x.buf.shape, generator=gen, device="cuda") * torch.exp(2 * torch.randn(x.buf.shape, generator=gen, device="cuda"))
    x.buf.copy_(v.clamp(-3e4, 3e4))
    q = Stored(order, M, N, pad=pad, off=off, dtype=torch.int8, fill=77)
    return x, q


SHAPES = [(1, 1), (1, 16), (3, 5), (16, 4096), (7, 4097), (5, 8192), (2, 20000), (300, 33), (129, 1000), (2000, 257)]


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("order", ["row", "col"])
@pytest.mark.parametrize("side", ["left", "right"])
@pytest.mark.parametrize("pad,off", [(0, 0), (8, 16), (3, 5)])
def test_against_the_definition(kind, order, side, pad, off):
    for M, N in SHAPES:
        x, q = build(order, M, N, kind, pad, off, seed=M * 31 + N)
        n = M if side == "left" else N
        scale = torch.full((n + 8,), 5.0, device="cuda")
        cb.check(call(order, side, M, N, kind, x, q, scale, off_s=4), "quantize")
        want_q, want_s = quantize_reference(x.op()[0], 1 if side == "left" else 0)
        got_q, got_s = q.op()[0].cpu(), scale[4:4 + n].cpu()
        assert torch.equal(got_q, want_q), (M, N)
        assert torch.equal(got_s, want_s), (M, N)
        assert bool((q.buf[q.outside()] == 77).all()) and bool((scale[:4] == 5).all()) and bool((scale[4 + n:] == 5).all())
        # |x - s q| <= s (1/2 + what three roundings move a value of at most 127)
        s64 = got_s.double()[:, None] if side == "left" else got_s.double()[None, :]
        off_by = (x.op()[0].cpu().double() - s64 * got_q.double()).abs()
        assert bool((off_by <= s64 * (0.5 + 127 * 4 * U32)).all())


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("pad,off", [(0, 0), (3, 5)])
def test_scales_across_many_lines(kind, pad, off):
    """More lines, or more elements, than a cluster keeps in registers: two passes, by 16-byte and by single accesses."""
    for M, N in ((4500, 40), (4500, 264), (5200, 520), (9000, 17), (4097, 2304), (8200, 3), (2048, 8320)):
        x, q = build("row", M, N, kind, pad, off, seed=M + N)
        scale = torch.full((N + 8,), 5.0, device="cuda")
        cb.check(call("row", "right", M, N, kind, x, q, scale, off_s=4), "quantize")
        want_q, want_s = quantize_reference(x.op()[0], 0)
        assert torch.equal(q.op()[0].cpu(), want_q) and torch.equal(scale[4:4 + N].cpu(), want_s), (M, N)
        assert bool((q.buf[q.outside()] == 77).all()) and bool((scale[:4] == 5).all()) and bool((scale[4 + N:] == 5).all())


@pytest.mark.parametrize("side", ["left", "right"])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_zero_tiny_and_non_finite_lines(side, kind):
    n = 12
    x, q = build("row", n, n, kind, 0, 0)
    v = x.op()[0]
    w = v if side == "left" else v.t()                     # w: lines that share a scale
    w[1] = 0
    w[2] = torch.full_like(w[2], 2.0 ** -101)              # below the smallest magnitude that is scaled
    w[3] = 0
    w[3, 5] = -(2.0 ** -100)                               # the smallest that is
    w[4, 2] = math.inf
    w[5, 7] = -math.inf
    w[6, 0] = math.nan
    w[7, 3] = math.nan
    w[7, 4] = math.inf
    scale = torch.full((n,), 5.0, device="cuda")
    cb.check(call("row", side, n, n, kind, x, q, scale), "quantize")
    got = q.op()[0] if side == "left" else q.op()[0].t()
    assert scale[1] == 0 and scale[2] == 0 and not got[1].any() and not got[2].any()
    assert scale[3].item() == torch.tensor(2.0 ** -100).div(torch.tensor(127.0)).item() and got[3, 5] == -127 and int(got[3].abs().sum()) == 127
    assert bool(scale[4:8].isnan().all()) and not got[4:8].any()
    rest = [0] + list(range(8, n))
    want_q, want_s = quantize_reference(w[rest], 1)
    assert torch.equal(got[rest].cpu(), want_q) and torch.equal(scale[rest].cpu(), want_s)


def test_refusals():
    x, q = build("row", 8, 32, "bf16", 0, 0)
    scale = torch.zeros(8, device="cuda")
    assert call("row", "left", 8, 32, "bf16", x, q, scale) == cb.clblasSuccess
    f = cb.clblasB200QuantizeI8
    assert f(0, 0, 8, 32, 2, None, 0, 32, q.buf, 0, 32, scale, 0) == cb.clblasInvalidMatA
    assert f(0, 0, 8, 32, 2, x.buf, 0, 32, None, 0, 32, scale, 0) == cb.clblasInvalidMatB
    assert f(0, 0, 8, 32, 2, x.buf, 0, 32, q.buf, 0, 32, None, 0) == cb.clblasInvalidVecX
    assert f(0, 0, 0, 32, 2, x.buf, 0, 32, q.buf, 0, 32, scale, 0) == cb.clblasInvalidDim
    assert f(0, 0, 8, 32, 2, x.buf, 0, 31, q.buf, 0, 32, scale, 0) == cb.clblasInvalidLeadDimA
    assert f(0, 0, 8, 32, 2, x.buf, 0, 32, q.buf, 0, 31, scale, 0) == cb.clblasInvalidLeadDimB
    assert f(0, 0, 8, 32, 3, x.buf, 0, 32, q.buf, 0, 32, scale, 0) == cb.clblasInvalidValue
    assert f(0, 2, 8, 32, 2, x.buf, 0, 32, q.buf, 0, 32, scale, 0) == cb.clblasInvalidValue
    big = 1 << 34
    assert f(0, 0, 8, 32, 2, x.buf, big, 32, q.buf, 0, 32, scale, 0) == cb.clblasInsufficientMemMatA
    assert f(0, 0, 8, 32, 2, x.buf, 0, 32, q.buf, big, 32, scale, 0) == cb.clblasInsufficientMemMatB
    assert f(0, 0, 8, 32, 2, x.buf, 0, 32, q.buf, 0, 32, scale, big) == cb.clblasInsufficientMemVecX
    assert cb.lib.clblasB200DeviceFault() == 0
