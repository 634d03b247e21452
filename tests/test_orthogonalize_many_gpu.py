"""clblasB200Orthogonalize on more matrices than a grid has blocks along its second axis."""
import pytest
import torch

import clblas_b200 as cb
from tests.cases_narrow import HALF_STEP, QUINTIC, orth_bound, orth_exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,m,batch", [(130, 132, 65536), (131, 129, 70001), (3, 5, 200003)])
def test_batches_beyond_a_grid(n, m, batch):
    gen = torch.Generator(device="cuda").manual_seed(n)
    g = torch.randn(batch, n, m, generator=gen, device="cuda", dtype=torch.bfloat16)
    o = torch.full((batch * n * m + 64,), 7.0, device="cuda", dtype=torch.bfloat16)
    cb.check(cb.clblasB200Orthogonalize(0, n, m, batch, 5, None, 1.0, 2, g, 0, m, n * m, 0.0, o, 0, m, n * m), "orthogonalize")
    got = o[:-64].view(batch, n, m)
    for i in (0, 1, 32767, 32768, 65535, min(65536, batch - 1), batch - 1):
        want, bound = orth_exact(g[i].double(), [QUINTIC] * 5), orth_bound(g[i], [QUINTIC] * 5)
        assert float((got[i].double() - want).norm()) <= bound + HALF_STEP["bf16"] * (float(want.norm()) + bound), i
    assert bool((o[-64:] == 7).all())
    # every matrix has its place: the polynomial leaves the largest singular value between 0.68 and 1.21 and none above, so the size of a
    # result over sqrt(n) lies between 0.68 / sqrt(3), one value of three, and 1.21
    sizes = got.float().square().sum((1, 2)).sqrt() / min(n, m) ** 0.5
    assert 0.35 < float(sizes.min()) and float(sizes.max()) < 1.3
    assert cb.lib.clblasB200DeviceFault() == 0
    del g, o, got
    torch.cuda.empty_cache()


def test_one_gradient_for_many_weights():
    """strideG 0 and beta over the border between two parts."""
    n, m, batch = 40, 24, 40000
    gen = torch.Generator(device="cuda").manual_seed(1)
    g = torch.randn(n, m, generator=gen, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(batch, n, m, generator=gen, device="cuda", dtype=torch.bfloat16)
    w0 = w.float()
    one = torch.zeros(n, m, device="cuda", dtype=torch.bfloat16)
    cb.check(cb.clblasB200Orthogonalize(0, n, m, 1, 5, None, 1.0, 2, g, 0, m, 0, 0.0, one, 0, m, 0))
    cb.check(cb.clblasB200Orthogonalize(0, n, m, batch, 5, None, -0.5, 2, g, 0, m, 0, 0.25, w, 0, m, n * m))
    want = 0.25 * w0 - 0.5 * one.float()
    # `one` and w are rounded to BF16, half a step of either; the iterations may take their sums in another order, each within about 1e-3 of
    # the result's size: 8 times that of an element, sqrt(24 / 960) = 0.158, for two results times 0.5
    assert bool(((w.float() - want).abs() <= 2.0 ** -8 * (0.5 * one.float().abs() + want.abs()) + 8 * 1e-3 * 0.158).all())
