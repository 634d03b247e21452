"""clblasB200Orthogonalize over the range of FP32: gradients whose norm lies far below the 1e-7 of the definition, where X starts far below
one.  The result before its rounding to BF16 is held against 64 bits with the bound of the operator's roundings, which has no term
for the size of G: a result that loses bits with the norm fails."""
import pytest
import torch

import clblas_b200 as cb
from tests.cases_narrow import QUINTIC, TYPES, U32, orth_bound, orth_exact
from tests.cases_orth_rounding import before_rounding, gram_operand_bound

pytestmark = pytest.mark.gpu

NORMS = [3.0, 2e-7, 1e-9, 1e-12, 1e-14, 1e-16, 1e-22, 1e-36]


def gradients(lines, length, norms, kind, seed=0):
    """One matrix for each norm, as the type holds it."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    g = torch.randn(len(norms), lines, length, generator=gen, device="cuda").double()
    g *= torch.tensor(norms, device="cuda", dtype=torch.float64)[:, None, None] / torch.linalg.matrix_norm(g)[:, None, None]
    return g.to(TYPES[kind][0]).contiguous()


def check(g, chain, kind, order=cb.clblasRowMajor):
    exact = torch.stack([orth_exact(m.double(), chain) for m in g])
    got = before_rounding(g, exact, chain, TYPES[kind][1], order)
    for i, m in enumerate(g):
        size = float(exact[i].norm())
        bound = orth_bound(m, chain) + gram_operand_bound(m, chain) + 2 * U32 * size         # and the last operations in FP32
        # what before_rounding adds: FP32 sums with w (2^-24 of |NS| + |w|), and half a BF16 step of a difference of at most bound + 2^-8 |NS|
        bound += 3 * U32 * size + 2.0 ** -8 * (bound + 2.0 ** -8 * size)
        err = float((got[i] - exact[i]).norm())
        assert size > 0 and err <= bound, (i, float(m.double().norm()), err / size, bound / size)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("lines,length", [(64, 256), (300, 40), (90, 1500), (300, 300), (150, 700), (700, 260)])
def test_small_gradients(lines, length, kind):
    check(gradients(lines, length, NORMS, kind), [QUINTIC] * 5, kind)


def test_small_gradients_in_sixteen_bits():
    """FP16 ends at 6e-8: the norm of a matrix of its smallest numbers."""
    for lines, length in ((64, 96), (200, 260)):
        g = torch.zeros(1, lines, length, dtype=torch.float16, device="cuda")
        g[0, 3, 5:9] = 2.0 ** -24
        g[0, 7, 1:3] = -(2.0 ** -23)
        check(g, [QUINTIC] * 5, "f16")


@pytest.mark.parametrize("steps", [12, 20, 40])
@pytest.mark.parametrize("lines,length", [(96, 160), (200, 384), (256, 256)])
def test_small_gradients_over_many_steps(lines, length, steps):
    """X grows through the whole range and levels off: the exponent follows it down to zero.  (Cubic steps: they converge, and errors die out.)"""
    check(gradients(lines, length, [1e-8, 1e-13, 1e-16, 1e-18], "f32", seed=1), [(1.5, -0.5, 0.0)] * steps, "f32")
    check(gradients(lines, length, [1e-8, 1e-13, 1e-16, 1e-18], "f32", seed=2), [(1.875, -1.25, 0.375)] * steps, "f32")


@pytest.mark.parametrize("steps", [10, 20])
def test_the_default_coefficients_over_many_steps(steps):
    for lines, length in ((100, 130), (256, 384)):
        check(gradients(lines, length, [1e-10, 1e-13, 1e-16], "f32", seed=3), [QUINTIC] * steps, "f32")


@pytest.mark.parametrize("chain", [[(0.01, 0.0, 0.002)] * 3, [(0.0, 1.5, 0.0)], [(0.0, 1.0, 0.5)] * 2, [(40.0, -3.0, 1.0), (0.5, 0.25, 0.0)],
                                   [(1e-12, 0.0, 0.0), (1e12, 0.0, 0.0)], [(1e-3, 1.0, 1.0), (1e3, 0.1, 0.1)]])
@pytest.mark.parametrize("lines,length", [(80, 120), (200, 260)])
def test_coefficients_that_shrink_and_grow(lines, length, chain):
    """X may become small in the middle as well, and the polynomial may have no linear term."""
    check(gradients(lines, length, [1.0, 1e-6, 1e-9], "f32", seed=4), chain, "f32")


def test_column_major_and_one_row():
    g = gradients(260, 150, NORMS, "f32", seed=5)
    check(g, [QUINTIC] * 5, "f32", cb.clblasColumnMajor)
    check(gradients(1, 200, NORMS, "f32", seed=6), [QUINTIC] * 5, "f32")
    check(gradients(400, 1, NORMS, "f32", seed=7), [QUINTIC] * 5, "f32")
    check(gradients(1, 1, NORMS, "f32", seed=8), [QUINTIC] * 5, "f32")


def test_ordinary_gradients_beside_small_ones_keep_their_results():
    """A matrix of a batch has a power of two of its own: the ordinary one is the same, bit for bit, in any company."""
    for lines, length in ((96, 200), (256, 300)):
        g = gradients(lines, length, [2.0, 1e-15, 0.5], "f32", seed=9)
        outs = []
        for batch in (g, g[:1].contiguous(), g[2:].contiguous()):
            o = torch.zeros_like(batch, dtype=torch.bfloat16)
            cb.check(cb.clblasB200Orthogonalize(0, lines, length, len(batch), 5, None, 1.0, 0, batch, 0, length, lines * length, 0.0, o, 0, length, lines * length))
            outs.append(o)
        assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][2], outs[2][0])
    assert cb.lib.clblasB200DeviceFault() == 0
