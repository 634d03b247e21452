"""Results handed from one narrow-type call to the next with nothing between them: kernels that are resident before their predecessor has
ended must read what it writes only after the wait, and not as constants."""
import os
import re

import pytest
import torch

import clblas_b200 as cb

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16 = cb.clblasB200Bfloat16
FILES = ["i8gemm.cu", "quantize_i8.cu", "orthogonalize.cu", "orthogonalize_small.cu", "narrow_mma.cuh", "orthogonalize.cuh"]


def source(name):
    text = open(os.path.join(ROOT, "clblas_b200", "csrc", name)).read()
    return re.sub(r"//[^\n]*", "", text)


def kernels(text):
    """(parameters, body) of every kernel of a source file."""
    text = re.sub(r"__launch_bounds__\([^)]*\)", "", text)
    for m in re.finditer(r"__global__\s+void\s+(\w+)\(", text):
        depth, at = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[at], 0)
            at += 1
        yield m.group(1), text[m.end():at], text[text.index("{", at):text.index("\n}\n", at)]


def test_no_constant_loads_in_kernels_that_start_early():
    """`__ldg` and `const __restrict__` pointers ask for loads of data that is constant while the kernel lives; the predecessor of a
    kernel that waits for it (pdl_wait) may be writing it."""
    early = []
    for name in FILES:
        text = source(name)
        assert "__ldg(" not in text and "ld.global.nc" not in text, name
        for kernel, parameters, body in kernels(text):
            if "pdl_wait()" not in body:
                continue
            early.append(kernel)
            assert not re.search(r"const\s+\w+\s*\*\s*__restrict__", parameters), (name, kernel)
    assert {"quantize_lines_kernel", "quantize_across_kernel", "across_max_kernel", "across_quantize_kernel", "pack_kernel", "split_kernel",
            "narrow_persistent_kernel", "narrow_split_kernel", "orthogonalize_small_kernel"} <= set(early)


class Chain:
    """A layer whose buffers are used again by every step; only calls of the library between the first and the last."""

    def __init__(self, T, O, K, steps, side, seed=1):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
        self.T, self.O, self.K, self.steps, self.side = T, O, K, steps, side
        self.w = (r(O, K) / K ** 0.5).bfloat16()
        # inputs of very different sizes: a stale scale is off by a factor
        self.x = [(r(T, K) * 4.0 ** (i % 5 - 2)).bfloat16() for i in range(steps)]
        self.g = [r(O, K).bfloat16() for i in range(steps)]
        self.qw, self.qx = (torch.zeros(n, K, dtype=torch.int8, device="cuda") for n in (O, T))
        self.sw, self.sx = torch.zeros(O, device="cuda"), torch.zeros(T, device="cuda")
        self.y = torch.zeros(T, O, dtype=torch.bfloat16, device="cuda")
        self.qy = [torch.zeros(T, O, dtype=torch.int8, device="cuda") for _ in range(steps)]
        self.sy = [torch.zeros(T if side == cb.clblasLeft else O, device="cuda") for _ in range(steps)]
        self.qy2, self.sy2 = [torch.zeros_like(q) for q in self.qy], [torch.zeros_like(s) for s in self.sy]

    def run(self, wait):
        self.queue((lambda st: (cb.check(st), torch.cuda.synchronize())) if wait else cb.check)
        torch.cuda.synchronize()

    def queue(self, done=cb.check):
        T, O, K = self.T, self.O, self.K
        product = lambda: done(cb.clblasB200I8gemm(0, 0, 1, T, O, K, 1.0, self.qx, 0, K, self.sx, 0, self.qw, 0, K, self.sw, 0, 0.0, BF16, self.y, 0, O))  # noqa: E731
        left = cb.clblasLeft
        for i in range(self.steps):
            done(cb.clblasB200QuantizeI8(0, left, O, K, BF16, self.w, 0, K, self.qw, 0, K, self.sw, 0))
            done(cb.clblasB200QuantizeI8(0, left, T, K, BF16, self.x[i], 0, K, self.qx, 0, K, self.sx, 0))
            product()
            done(cb.clblasB200QuantizeI8(0, self.side, T, O, BF16, self.y, 0, O, self.qy[i], 0, O, self.sy[i], 0))
            product()
            done(cb.clblasB200QuantizeI8(0, left, T, K, BF16, self.x[(i + 1) % self.steps], 0, K, self.qx, 0, K, self.sx, 0))
            product()
            done(cb.clblasB200QuantizeI8(0, self.side, T, O, BF16, self.y, 0, O, self.qy2[i], 0, O, self.sy2[i], 0))
            done(cb.clblasB200Orthogonalize(0, O, K, 1, 5, None, -0.02, BF16, self.g[i], 0, K, 0, 0.99, self.w, 0, K, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("side", ["left", "right"])
@pytest.mark.parametrize("T,O,K", [(1, 256, 384), (48, 96, 512), (300, 1000, 264), (700, 1504, 1024)])
def test_queued_calls_with_nothing_between_equal_waited_ones(T, O, K, side):
    side = cb.clblasLeft if side == "left" else cb.clblasRight
    queued, waited = Chain(T, O, K, 25, side), Chain(T, O, K, 25, side)
    torch.cuda.synchronize()
    queued.run(wait=False)
    waited.run(wait=True)
    for i in range(25):
        assert torch.equal(queued.sy[i], waited.sy[i]) and torch.equal(queued.qy[i], waited.qy[i]), i
        assert torch.equal(queued.sy2[i], waited.sy2[i]) and torch.equal(queued.qy2[i], waited.qy2[i]), i
    assert torch.equal(queued.w, waited.w) and cb.lib.clblasB200DeviceFault() == 0
