"""The queue that the narrow-type calls take by default: torch's current stream of the device that holds the result, whatever device is
current (their work runs there).  Two devices are played by a library and by stream queries that only record what they are asked."""
import types

import pytest
import torch

import clblas_b200 as cb


class Recorder:
    """Stands in for the C library: keeps the queue that a call was given."""

    def __init__(self):
        self.queues = []

    def clblasB200BufferDevice(self, address):
        return {0x1000: 1, 0x2000: 2}.get(address, -1)

    def __getattr__(self, name):
        def call(*args):
            queue = next(a for a in args if hasattr(a, "_length_"))
            self.queues.append((name, queue[0] or 0))
            return 0
        return call


@pytest.fixture
def streams(monkeypatch):
    """Device 0 is current; device d's current stream has the handle 0x100 + d."""
    lib = Recorder()
    monkeypatch.setattr(cb, "lib", lib)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 0x100 + d, raising=False)
    return lib


def tensor(device):
    return types.SimpleNamespace(device=torch.device("cuda", device), data_ptr=lambda: 64)


def calls(result, **kw):
    x = tensor(0)
    assert cb.clblasB200QuantizeI8(0, 0, 4, 16, 2, x, 0, 16, result, 0, 16, x, 0, **kw) == 0
    assert cb.clblasB200I8gemm(0, 0, 1, 4, 4, 16, 1.0, x, 0, 16, None, 0, x, 0, 16, None, 0, 0.0, 2, result, 0, 4, **kw) == 0
    assert cb.clblasB200Orthogonalize(0, 4, 16, 1, 5, None, 1.0, 2, x, 0, 16, 0, 0.0, result, 0, 16, 0, **kw) == 0


@pytest.mark.parametrize("result,device", [(tensor(0), 0), (tensor(1), 1), (tensor(3), 3), (0x1000, 1), (0x2000, 2),
                                           (0x3000, 0), (torch.zeros(4), 0)])
def test_default_queue_is_the_result_devices(streams, result, device):
    calls(result)
    calls(result, wait=[0x55])
    assert [q for _, q in streams.queues] == [0x100 + device] * 6


def test_a_given_queue_stays(streams):
    calls(tensor(1), queues=[0x77])
    assert [q for _, q in streams.queues] == [0x77] * 3


def test_older_routines_keep_the_current_device(streams):
    x = tensor(1)
    assert cb.clblasSgemm(1, 0, 0, 4, 4, 4, 1.0, x, 0, 4, x, 0, 4, 0.0, x, 0, 4) == 0
    assert streams.queues == [("clblasSgemm", 0x100)]


def test_device_of_an_unknown_buffer():
    assert cb.lib.clblasB200BufferDevice(None) == -1


@pytest.mark.gpu
def test_device_of_a_buffer_and_calls_on_a_side_stream():
    """The current stream of the result's device, a side stream here, is the one the work is queued on, for tensors and for addresses."""
    x = torch.randn(64, 4096, device="cuda").bfloat16()
    q, s = torch.zeros(64, 4096, dtype=torch.int8, device="cuda"), torch.zeros(64, device="cuda")
    assert cb.lib.clblasB200BufferDevice(q.data_ptr()) == torch.cuda.current_device()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for result in (q, q.data_ptr()):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):           # work on any other stream would not be part of the graph
            cb.check(cb.clblasB200QuantizeI8(0, cb.clblasLeft, 64, 4096, cb.clblasB200Bfloat16, x, 0, 4096, result, 0, 4096, s, 0))
        q.zero_()
        torch.cuda.synchronize()
        assert not q.any()
        graph.replay()
        torch.cuda.synchronize()
        assert int(q.abs().max()) == 127
