"""Narrow-type kernels may start while the kernel before them on the stream drains.  Whatever else stands between two of them has to
end first all the same: an event, a copy from the host, the work of another stream that the default stream waits for."""
import ctypes

import pytest
import torch

import clblas_b200 as cb

pytestmark = pytest.mark.gpu

BF16 = cb.clblasB200Bfloat16
M, N = 64, 4096
LONG = 2_000_000                                             # clocks: a millisecond, far longer than the calls


class Pair:
    """x is made new in every round; the quantisation of `other` before it is the kernel that lets its successor start."""

    def __init__(self):
        gen = torch.Generator(device="cuda").manual_seed(7)
        self.new = [(torch.randn(M, N, generator=gen, device="cuda") * 2.0 ** i).bfloat16() for i in range(6)]
        self.x, self.other = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda"), self.new[0].clone()
        self.q, self.q2 = (torch.zeros(M, N, dtype=torch.int8, device="cuda") for _ in range(2))
        self.s, self.s2 = torch.zeros(M, device="cuda"), torch.zeros(M, device="cuda")
        self.o = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
        self.want = [v.float().abs().amax(1) / torch.full((M,), 127.0, device="cuda") for v in self.new]
        torch.cuda.synchronize()

    def before(self, queue):
        for _ in range(3):
            cb.check(cb.clblasB200QuantizeI8(0, cb.clblasLeft, M, N, BF16, self.other, 0, N, self.q2, 0, N, self.s2, 0, queues=[queue]))

    def after(self, queue, **kw):
        cb.check(cb.clblasB200QuantizeI8(0, cb.clblasLeft, M, N, BF16, self.x, 0, N, self.q, 0, N, self.s, 0, queues=[queue], **kw))

    def check(self, i):
        torch.cuda.synchronize()
        assert torch.equal(self.s, self.want[i]), i


def test_after_an_event_of_another_stream():
    p, a, b = Pair(), torch.cuda.Stream(), torch.cuda.Stream()
    for way in ("wait list", "stream wait"):
        for i in range(6):
            ready = torch.cuda.Event()
            with torch.cuda.stream(b):
                torch.cuda._sleep(LONG)
                p.x.copy_(p.new[i])
                ready.record(b)
            p.before(a)
            if way == "wait list":
                p.after(a, wait=[ready])
            else:
                a.wait_event(ready)
                p.after(a)
            p.check(i)


def test_after_a_copy_from_the_host():
    p, a = Pair(), torch.cuda.Stream()
    host = [v.cpu().pin_memory() for v in p.new]
    big = torch.zeros(64 << 20, dtype=torch.uint8).pin_memory()
    sink = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    for i in range(6):
        p.before(a)
        with torch.cuda.stream(a):
            sink.copy_(big, non_blocking=True)               # holds the copy engine for a millisecond
            p.x.copy_(host[i], non_blocking=True)
        p.after(a)
        p.check(i)


def test_after_a_fill_and_a_copy_on_the_device():
    p, a = Pair(), torch.cuda.Stream()
    for i in range(6):
        p.before(a)
        with torch.cuda.stream(a):
            torch.cuda._sleep(LONG)
            p.x.zero_()
            p.x.copy_(p.new[i])
        p.after(a)
        p.check(i)


def test_the_default_stream_after_a_blocking_one():
    """The default stream waits for the work of streams that were made to block."""
    cudart = ctypes.CDLL("libcudart.so.12")
    handle = ctypes.c_void_p()
    assert cudart.cudaStreamCreate(ctypes.byref(handle)) == 0
    p, b = Pair(), torch.cuda.ExternalStream(handle.value)
    for i in range(6):
        p.before(0)
        with torch.cuda.stream(b):
            torch.cuda._sleep(LONG)
            p.x.copy_(p.new[i])
        p.after(0)
        p.check(i)
    torch.cuda.synchronize()
    assert cudart.cudaStreamDestroy(handle) == 0


@pytest.mark.parametrize("between", ["event", "copy"])
def test_captured(between):
    p, a, b = Pair(), torch.cuda.Stream(), torch.cuda.Stream()
    host = [v.cpu().pin_memory() for v in p.new]
    staged = host[0].clone().pin_memory()
    source = p.new[0].clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=a):
        if between == "event":
            b.wait_stream(a)
            with torch.cuda.stream(b):
                torch.cuda._sleep(LONG)
                p.x.copy_(source)
            p.before(a)
            a.wait_stream(b)
        else:
            p.before(a)
            p.x.copy_(staged, non_blocking=True)
        p.after(a)
    for i in range(6):
        source.copy_(p.new[i])
        staged.copy_(host[i])
        torch.cuda.synchronize()
        graph.replay()
        p.check(i)
