"""Plain 64-bit restatements and input builders for the narrow-type operators (8-bit quantisation, 8-bit products with
scales, Newton-Schulz orthogonalisation), shared by their tests.  Matrices are kept as the caller of the C ABI keeps them:
a flat buffer of lines with a pitch, an element offset in front, and a guard pattern around what the call may write."""
import math

import torch

import clblas_b200 as cb

TYPES = {"f32": (torch.float32, cb.clblasB200Float32), "f16": (torch.float16, cb.clblasB200Float16),
         "bf16": (torch.bfloat16, cb.clblasB200Bfloat16)}
U32 = 2.0 ** -24                                              # half a step of float32, relative
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}     # half a step of the subnormal range


def order_code(order):
    return cb.clblasRowMajor if order == "row" else cb.clblasColumnMajor


class Stored:
    """op(X), rows x cols, as the ABI stores it: `buf` holds `lines` lines of `length` elements, pitch `ld`, after `off` elements."""

    def __init__(self, order, rows, cols, trans="n", pad=0, off=0, dtype=torch.float32, batch=1, gap=0, fill=None, device="cuda"):
        r, c = (cols, rows) if trans == "t" else (rows, cols)
        self.lines, self.length = (r, c) if order == "row" else (c, r)
        self.ld, self.off, self.batch = self.length + pad, off, batch
        self.stride = self.ld * self.lines + gap
        self.flip = (order == "row") != (trans == "n")
        n = off + self.stride * (batch - 1) + self.ld * (self.lines - 1) + self.length
        self.buf = torch.zeros(n + 64, dtype=dtype, device=device)          # 64 elements of guard behind the matrix
        if fill is not None:
            self.buf.fill_(fill)

    def lines_view(self):
        return torch.as_strided(self.buf, (self.batch, self.lines, self.length), (self.stride, self.ld, 1), self.off)

    def op(self):
        """batch x rows x cols view of op(X)."""
        v = self.lines_view()
        return v.transpose(1, 2) if self.flip else v

    def outside(self):
        """Mask of the elements no call may touch."""
        m = torch.ones_like(self.buf, dtype=torch.bool)
        torch.as_strided(m, (self.batch, self.lines, self.length), (self.stride, self.ld, 1), self.off).fill_(False)
        return m


def random_i8(st, gen, extremes=True):
    v = torch.randint(-127, 128, st.buf.shape, generator=gen, device=st.buf.device, dtype=torch.int32).to(torch.int8)
    if extremes:
        v[::7] = -128
    st.buf.copy_(v)


def i8gemm_bound(exact_sum, sa, sb, alpha, beta, c0, kind):
    """|computed - exact| of alpha sA S sB + beta C: S -> float32, alpha sA, its product with S and that with sB are one rounding each
    (the first order in 2^-24, the rest covered by a fifth), one for the final sum, one to the type of C."""
    prod = (alpha * exact_sum * sa[:, None] * sb[None, :]).abs()
    add = (beta * c0).abs() if beta else torch.zeros_like(prod)
    inner = 5 * U32 * prod + U32 * (prod + add)
    return inner + HALF_STEP[kind] * (prod + add + inner) + TINY[kind]


def quantize_reference(x, axis):
    """The definition, one IEEE float32 operation after the other, on the CPU: q (int8) and scale for a finite float32 matrix."""
    x = x.detach().cpu().float()
    top = x.abs().amax(axis, keepdim=True)
    live = top >= 2.0 ** -100
    full = torch.full_like(top, 127.0)
    scale = torch.where(live, top / full, torch.zeros_like(top))
    inv = torch.where(live, full / torch.where(live, top, full), torch.zeros_like(top))
    return (x * inv).round().to(torch.int8), scale.reshape(-1)
