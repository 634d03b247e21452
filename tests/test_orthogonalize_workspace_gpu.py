"""Which calls of clblasB200Orthogonalize take a workspace: the rule that the header states, on both sides of its borders."""
import pytest
import torch

import clblas_b200 as cb
from tests.cases_narrow import HALF_STEP, QUINTIC, orth_bound, orth_exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tall", [False, True])
@pytest.mark.parametrize("n,m,batch,takes", [(128, 1024, 1, 0), (128, 1024, 100, 0), (128, 1025, 15, 0), (128, 1025, 16, 1), (128, 2048, 15, 0),
                                             (128, 2048, 16, 1), (128, 2049, 1, 1), (129, 200, 1, 1), (1, 2048, 15, 0), (5, 2048, 16, 1)])
def test_workspace_allocations(n, m, batch, takes, tall):
    M, N = (m, n) if tall else (n, m)
    gen = torch.Generator(device="cuda").manual_seed(n + m)
    g = torch.randn(batch, M, N, generator=gen, device="cuda", dtype=torch.bfloat16)
    o = torch.zeros_like(g)
    before = cb.lib.clblasB200WorkspaceAllocCount()
    cb.check(cb.clblasB200Orthogonalize(0, M, N, batch, 5, None, 1.0, 2, g, 0, N, M * N, 0.0, o, 0, N, M * N))
    assert cb.lib.clblasB200WorkspaceAllocCount() - before == takes
    for i in (0, batch - 1):
        want, bound = orth_exact(g[i].double(), [QUINTIC] * 5), orth_bound(g[i], [QUINTIC] * 5)
        assert float((o[i].double() - want).norm()) <= bound + HALF_STEP["bf16"] * (float(want.norm()) + bound)
