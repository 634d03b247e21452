"""CPU-side refusals of the narrow-type entry points: what can be decided before any device work, in the order that the header
states (buffers, enums, sizes), as for the other routines (tests/test_abi.py)."""
import math

import pytest

import clblas_b200 as cb
from tests.cases_narrow import i8gemm_bound  # noqa: F401  (the helpers import without a GPU)

Q = [0]


def i8(order=0, ta=0, tb=1, M=16, N=32, K=48, A=8, lda=48, B=8, ldb=48, T=2, C=8, ldc=32, queues=Q):
    return cb.clblasB200I8gemm(order, ta, tb, M, N, K, 1.0, A, 0, lda, None, 0, B, 0, ldb, None, 0, 0.0, T, C, 0, ldc, queues=queues)


def quantize(order=0, side=0, M=8, N=32, T=2, X=8, ldx=32, Qm=8, ldq=32, S=8):
    return cb.clblasB200QuantizeI8(order, side, M, N, T, X, 0, ldx, Qm, 0, ldq, S, 0, queues=Q)


def orth(order=0, M=24, N=40, batch=2, steps=5, co=None, T=2, G=8, ldg=40, O=8, ldo=40):
    return cb.clblasB200Orthogonalize(order, M, N, batch, steps, co, 1.0, T, G, 0, ldg, 960, 0.0, O, 0, ldo, 960, queues=Q)


def test_null_buffers_and_enums():
    assert i8(A=None) == cb.clblasInvalidMatA and i8(B=None) == cb.clblasInvalidMatB and i8(C=None) == cb.clblasInvalidMatC
    assert i8(A=None, order=9) == cb.clblasInvalidMatA
    assert i8(order=9) == cb.clblasInvalidValue and i8(ta=3) == cb.clblasInvalidValue and i8(tb=-1) == cb.clblasInvalidValue
    assert i8(T=3) == cb.clblasInvalidValue and i8(T=-1) == cb.clblasInvalidValue
    assert quantize(X=None) == cb.clblasInvalidMatA and quantize(Qm=None) == cb.clblasInvalidMatB and quantize(S=None) == cb.clblasInvalidVecX
    assert quantize(side=2) == cb.clblasInvalidValue and quantize(T=7) == cb.clblasInvalidValue and quantize(order=2) == cb.clblasInvalidValue
    assert orth(G=None) == cb.clblasInvalidMatA and orth(O=None) == cb.clblasInvalidMatC
    assert orth(T=9) == cb.clblasInvalidValue and orth(order=3) == cb.clblasInvalidValue


@pytest.mark.parametrize("steps", [0, 65, 1 << 31])
def test_steps_out_of_range(steps):
    assert orth(steps=steps) == cb.clblasInvalidValue


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_coefficients_that_are_not_finite(bad):
    for at in range(3):
        triple = [1.0, 1.0, 1.0]
        triple[at] = bad
        assert orth(steps=2, co=[(1.5, -0.5, 0.0), tuple(triple)]) == cb.clblasInvalidValue
    with pytest.raises(ValueError):
        orth(steps=2, co=[(1.0, 1.0, 1.0)])


def test_sizes_and_leading_dimensions():
    assert i8(M=0) == cb.clblasInvalidDim and i8(lda=47) == cb.clblasInvalidLeadDimA
    assert i8(order=1, lda=15) == cb.clblasInvalidLeadDimA                   # column-major: lines of M
    assert quantize(M=0) == cb.clblasInvalidDim and quantize(N=0) == cb.clblasInvalidDim and quantize(ldx=31) == cb.clblasInvalidLeadDimA
    assert orth(M=0) == cb.clblasInvalidDim and orth(N=0) == cb.clblasInvalidDim and orth(batch=0) == cb.clblasInvalidDim
    assert orth(ldg=39) == cb.clblasInvalidLeadDimA


def test_type_codes_match_the_header():
    text = open(cb.__file__.replace("clblas_b200/__init__.py", "include/clblas_b200.h")).read()
    for name in ("clblasB200Float32", "clblasB200Float16", "clblasB200Bfloat16"):
        assert f"{name} = {getattr(cb, name)}" in text
