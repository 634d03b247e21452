"""clblasB200Orthogonalize of very long matrices: the sums of the Gram product run over the larger side, and the tensor core cuts them
off, by 2^-25 for every 16 terms on average.  The error before the rounding to BF16 has to stay near that of the other roundings (E,
emulated with exact sums), whatever the length: a segment of 131072 terms falls 2^13 2^-25 = 2.4e-4 behind, of which the polynomial
makes twice as much."""
import pytest
import torch

import clblas_b200 as cb
from tests.cases_narrow import QUINTIC, orth_exact
from tests.cases_orth_rounding import before_rounding, orth_emulated

pytestmark = pytest.mark.gpu


# around one and two segments of 131072, odd ends, many segments; tall ones are transposed on the way
@pytest.mark.parametrize("lines,length,batch", [(8, 131072, 2), (8, 131073, 2), (5, 262144, 1), (300, 262145, 1), (262151, 140, 1), (3, 400009, 3), (200, 1 << 20, 1),
                                                (8, 1 << 20, 1), (1 << 22, 8, 1), (1, 1 << 24, 1), (2, (1 << 24) + 5, 1)])
def test_long_sums(lines, length, batch):
    gen = torch.Generator(device="cuda").manual_seed(length % 1000)
    g = torch.randn(batch, lines, length, generator=gen, device="cuda", dtype=torch.bfloat16)
    exact = torch.stack([orth_exact(m.double(), [QUINTIC] * 5) for m in g])
    got = before_rounding(g, exact, [QUINTIC] * 5, cb.clblasB200Bfloat16)
    for i in range(batch):
        E = float((orth_emulated(g[i], [QUINTIC] * 5) - exact[i]).norm())
        assert float((got[i] - exact[i]).norm()) <= 1.5 * E + 5e-4 * float(exact[i].norm()), i
    assert cb.lib.clblasB200DeviceFault() == 0
    del g, exact, got
    torch.cuda.empty_cache()


def test_long_sums_on_the_persistent_kernels():
    n, m = 2500, 262144
    g = torch.randn(n, m, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda", dtype=torch.bfloat16)
    chain = [QUINTIC] * 2
    exact = orth_exact(g.double(), chain)
    got = before_rounding(g[None], exact[None], chain, cb.clblasB200Bfloat16)[0]
    assert cb.last_gemm_variant().startswith("orthogonalize<pairs256,")
    assert float((got - exact).norm()) <= 1.5 * float((orth_emulated(g, chain) - exact).norm()) + 5e-4 * float(exact.norm())
    top = (got - exact).abs().max() / (got - exact).square().mean().sqrt()
    assert float(top) <= 20
    del g, exact, got
    torch.cuda.empty_cache()


def test_the_same_call_twice_is_identical():
    g = torch.randn(40, 300000, device="cuda")
    outs = []
    for _ in range(3):
        o = torch.zeros(40, 300000, dtype=torch.bfloat16, device="cuda")
        cb.check(cb.clblasB200Orthogonalize(0, 40, 300000, 1, 5, None, 1.0, 0, g, 0, 300000, 0, 0.0, o, 0, 300000, 0))
        outs.append(o)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
