"""Leading dimensions and offsets whose products wrap round 2^64 are refused like any other extent beyond the buffer; nothing is launched."""
import pytest
import torch

import clblas_b200 as cb

pytestmark = pytest.mark.gpu


@pytest.fixture
def buffers():
    return [torch.zeros(4096, dtype=d, device="cuda") for d in (torch.float32, torch.int8, torch.bfloat16)]


@pytest.mark.parametrize("ld", [1 << 63, 1 << 62, (1 << 61) + 1, (1 << 64) - 1])
def test_leading_dimensions(lib, buffers, ld):
    f, i, h = buffers
    n = 9                                                    # eight steps of 2^61 and more wrap for every element size
    before = cb.launch_count()
    for order in (cb.clblasRowMajor, cb.clblasColumnMajor):
        for A, B, C, want in ((ld, n, n, cb.clblasInsufficientMemMatA), (n, ld, n, cb.clblasInsufficientMemMatB), (n, n, ld, cb.clblasInsufficientMemMatC)):
            assert cb.clblasSgemm(order, 0, 0, n, n, n, 1.0, f, 0, A, f, 0, B, 0.0, f, 0, C) == want
            assert cb.clblasB200I8gemm(order, 0, 0, n, n, n, 1.0, i, 0, A, None, 0, i, 0, B, None, 0, 0.0, 2, h, 0, C) == want
        assert cb.clblasB200QuantizeI8(order, 0, n, n, 0, f, 0, ld, i, 0, n, f, 0) == cb.clblasInsufficientMemMatA
        assert cb.clblasB200QuantizeI8(order, 0, n, n, 0, f, 0, n, i, 0, ld, f, 0) == cb.clblasInsufficientMemMatB
        assert cb.clblasB200Orthogonalize(order, n, n, 1, 5, None, 1.0, 2, h, 0, ld, 0, 0.0, h, 0, n, 0) == cb.clblasInsufficientMemMatA
        assert cb.clblasB200Orthogonalize(order, n, n, 1, 5, None, 1.0, 2, h, 0, n, 0, 0.0, h, 0, ld, 0) == cb.clblasInsufficientMemMatC
        assert cb.clblasStrsm(order, 0, 0, 0, 1, n, n, 1.0, f, 0, ld, f, 0, n) == cb.clblasInsufficientMemMatA
    assert cb.launch_count() == before and cb.lib.clblasB200DeviceFault() == 0


@pytest.mark.parametrize("off", [1 << 62, 1 << 63, (1 << 63) + 8, (1 << 64) - 4])
def test_offsets(buffers, off):
    f, i, h = buffers
    n, before = 9, cb.launch_count()
    assert cb.clblasSgemm(0, 0, 0, n, n, n, 1.0, f, off, n, f, 0, n, 0.0, f, 0, n) == cb.clblasInsufficientMemMatA
    assert cb.clblasSgemm(0, 0, 0, n, n, n, 1.0, f, 0, n, f, 0, n, 0.0, f, off, n) == cb.clblasInsufficientMemMatC
    assert cb.clblasB200I8gemm(0, 0, 0, n, n, n, 1.0, i, 0, n, None, 0, i, off, n, None, 0, 0.0, 2, h, 0, n) == cb.clblasInsufficientMemMatB
    assert cb.clblasB200I8gemm(0, 0, 0, n, n, n, 1.0, i, 0, n, f, off, i, 0, n, None, 0, 0.0, 2, h, 0, n) == cb.clblasInsufficientMemVecX
    assert cb.clblasB200QuantizeI8(0, 0, n, n, 0, f, 0, n, i, 0, n, f, off) == cb.clblasInsufficientMemVecX
    assert cb.clblasB200Orthogonalize(0, n, n, 1, 5, None, 1.0, 2, h, off, n, 0, 0.0, h, 0, n, 0) == cb.clblasInsufficientMemMatA
    assert cb.launch_count() == before


@pytest.mark.parametrize("ld", [9, 1 << 45, 1 << 63, (1 << 64) - 1])
def test_one_line_has_no_second(ld):
    """A matrix of one line may have any leading dimension: no element lies behind it."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(9, generator=gen, device="cuda").bfloat16()
    q, s, o, c = torch.zeros(9, dtype=torch.int8, device="cuda"), torch.zeros(1, device="cuda"), torch.zeros_like(x), torch.zeros(1, device="cuda")
    cb.check(cb.clblasB200QuantizeI8(0, 0, 1, 9, 2, x, 0, ld, q, 0, ld, s, 0))
    assert int(q.abs().max()) == 127
    cb.check(cb.clblasB200I8gemm(0, 0, 1, 1, 1, 9, 1.0, q, 0, ld, None, 0, q, 0, ld, None, 0, 0.0, 0, c, 0, ld))
    assert float(c) == float(q.double().square().sum())
    cb.check(cb.clblasB200Orthogonalize(0, 1, 9, 1, 5, None, 1.0, 2, x, 0, ld, 0, 0.0, o, 0, ld, 0))
    y = 1.0
    for _ in range(5):
        y *= 3.4445 - 4.775 * y ** 2 + 2.0315 * y ** 4
    want = x.double() / x.double().norm() * y
    assert float((o.double() - want).norm()) <= 5e-3 * abs(y) and cb.lib.clblasB200DeviceFault() == 0
