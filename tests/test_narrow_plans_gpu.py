"""Every plan of the 8-bit products, on random operands, with k long enough that a CTA's ring of slabs wraps inside a tile.  The plan that
ran is asserted, so that a change of the estimates cannot take a kernel out of the tests."""
import pytest

import clblas_b200 as cb
from tests.test_i8gemm_gpu import Problem

pytestmark = pytest.mark.gpu

# few lines (row) or few positions of a line (col); whole tiles in one round and in several
CASES = [("split32x1", 20, 20000, 2000), ("split32x2", 20, 12000, 2000), ("split32x4", 20, 6000, 2500), ("split32x8", 20, 3000, 6000),
         ("split64x1", 50, 20000, 2000), ("split64x2", 50, 12000, 2000), ("split64x4", 50, 6000, 2500), ("split64x8", 50, 3000, 6000),
         ("split128x1", 100, 10000, 3000), ("split128x2", 100, 6000, 3000), ("split128x4", 100, 3000, 3000),
         ("split128x1", 1400, 1400, 1500), ("split128x2", 900, 900, 1500), ("split128x4", 300, 900, 3000),
         ("pairs192", 1000, 5000, 2056), ("pairs256", 4096, 4096, 2048)]


@pytest.mark.parametrize("order", ["row", "col"])
@pytest.mark.parametrize("plan,M,N,K", CASES)
def test_plans(plan, M, N, K, order):
    p = Problem(order, "n", "t", M, N, K, "bf16", pad=16, seed=M + K)
    p.check()
    assert cb.last_gemm_variant() == f"i8gemm_tcgen05<{plan}>"
    p = Problem(order, "n", "t", M, N, K, "f16", pad=7, seed=M + K + 1, c_rms=1.0)      # C's lines unaligned, operands packed
    p.sa *= 0.1
    p.check(0.5, -0.75)
    assert cb.last_gemm_variant() == f"i8gemm_tcgen05<{plan}>"


@pytest.mark.parametrize("pad", [0, 5])
@pytest.mark.parametrize("order,M,N", [("row", 6321, 533), ("col", 533, 6321)])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_narrow_pairs(order, M, N, kind, pad):
    Problem(order, "n", "t", M, N, 1500, kind, pad=pad, seed=1).check(1.0, 0.5)
    assert cb.last_gemm_variant() == "i8gemm_tcgen05<pairs128>"


@pytest.mark.parametrize("plan,M,N,K", [c for c in CASES if c[0] != "pairs256"] + [("pairs256", 257, 7119, 2698), ("pairs192", 6274, 257, 1482)])
@pytest.mark.parametrize("pad", [0, 3])
def test_plans_with_32_bit_results(plan, M, N, K, pad):
    Problem("row", "n", "t", M, N, K, "f32", pad=pad, seed=N).check(-1.5, 0.25)
    assert cb.last_gemm_variant() == f"i8gemm_tcgen05<{plan}>"


def test_operands_in_other_layouts_take_the_same_plans():
    for ta in "nt":
        for tb in "nt":
            Problem("row", ta, tb, 1000, 5000, 2056, "bf16", seed=3).check()
            assert cb.last_gemm_variant() == "i8gemm_tcgen05<pairs192>"
    assert cb.lib.clblasB200DeviceFault() == 0
