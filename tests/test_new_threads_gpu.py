"""Calls from threads that have not used CUDA before, as a C program's worker makes them: buffers are addresses, the queue is a handle, and
the thread's first CUDA call is the library's."""
import threading

import pytest
import torch

import clblas_b200 as cb
from tests.cases_narrow import quantize_reference

pytestmark = pytest.mark.gpu


def in_a_new_thread(work):
    t = threading.Thread(target=work)
    t.start()
    t.join()
    torch.cuda.synchronize()


def test_narrow_types():
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(300, 500, generator=gen, device="cuda")
    q, s = torch.zeros(300, 500, dtype=torch.int8, device="cuda"), torch.zeros(300, device="cuda")
    c, o = torch.zeros(300, 300, device="cuda"), torch.zeros(300, 500, dtype=torch.bfloat16, device="cuda")
    addresses = [t.data_ptr() for t in (x, q, s, c, o)]
    handle = torch.cuda.Stream().cuda_stream
    torch.cuda.synchronize()
    got = []

    def work():
        x, q, s, c, o = addresses
        got.append(cb.lib.clblasB200BufferDevice(q) - torch.cuda.current_device())
        got.append(cb.clblasB200QuantizeI8(0, cb.clblasLeft, 300, 500, 0, x, 0, 500, q, 0, 500, s, 0, queues=[handle]))
        got.append(cb.clblasB200I8gemm(0, 0, 1, 300, 300, 500, 1.0, q, 0, 500, s, 0, q, 0, 500, s, 0, 0.0, 0, c, 0, 300, queues=[handle]))
        got.append(cb.clblasB200Orthogonalize(0, 300, 500, 1, 5, None, 1.0, 0, x, 0, 500, 0, 0.0, o, 0, 500, 0, queues=[handle]))

    in_a_new_thread(work)
    assert got == [0, 0, 0, 0]
    ref_q, ref_s = quantize_reference(x, 1)
    assert torch.equal(q.cpu(), ref_q) and torch.equal(s.cpu(), ref_s)
    assert float(c.diagonal().min()) > 0 and 15 < float(o.float().norm()) < 21


@pytest.mark.parametrize("call", ["gemm", "trsm", "quantize", "i8gemm", "orthogonalize", "refused"])
def test_first_calls(lib, call):
    gen = torch.Generator(device="cuda").manual_seed(5)
    a = torch.randn(64, 64, generator=gen, device="cuda") + 16 * torch.eye(64, device="cuda")
    b, c = torch.randn(64, 64, generator=gen, device="cuda"), torch.zeros(64, 64, device="cuda")
    q, o = torch.zeros(64, 64, dtype=torch.int8, device="cuda"), torch.zeros(64, 64, dtype=torch.bfloat16, device="cuda")
    A, B, C, Q, O = (t.data_ptr() for t in (a, b, c, q, o))
    handle = [torch.cuda.Stream().cuda_stream]
    torch.cuda.synchronize()
    b0, got = b.clone(), []
    calls = {"gemm": lambda: cb.clblasSgemm(0, 0, 0, 64, 64, 64, 1.0, A, 0, 64, B, 0, 64, 0.0, C, 0, 64, queues=handle),
             "trsm": lambda: cb.clblasStrsm(0, 0, 1, 0, 1, 64, 64, 1.0, A, 0, 64, B, 0, 64, queues=handle),
             "quantize": lambda: cb.clblasB200QuantizeI8(0, 0, 64, 64, 0, A, 0, 64, Q, 0, 64, C, 0, queues=handle),
             "i8gemm": lambda: cb.clblasB200I8gemm(0, 0, 1, 64, 64, 64, 1.0, Q, 0, 64, None, 0, Q, 0, 64, None, 0, 0.0, 0, C, 0, 64, queues=handle),
             "orthogonalize": lambda: cb.clblasB200Orthogonalize(0, 64, 64, 1, 5, None, 1.0, 0, A, 0, 64, 0, 0.0, O, 0, 64, 0, queues=handle),
             "refused": lambda: cb.clblasSgemm(0, 0, 0, 64, 64, 64, 1.0, 1 << 20, 0, 64, B, 0, 64, 0.0, C, 0, 64, queues=handle)}
    in_a_new_thread(lambda: got.append(calls[call]()))
    assert got == [cb.clblasInvalidMatA if call == "refused" else 0]
    if call == "gemm":
        assert float((c.double() - a.double() @ b.double()).abs().max()) < 1e-3
    if call == "trsm":
        assert float((a.double().tril() @ b.double() - b0.double()).abs().max()) < 1e-3
    if call == "orthogonalize":
        assert 4 < float(o.float().norm()) < 10
    assert cb.lib.clblasB200DeviceFault() == 0
