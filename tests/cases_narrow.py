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


QUINTIC = (3.4445, -4.7750, 2.0315)


def orth_exact(g, coefficients):
    """NS(G) of the definition in 64 bits; g: rows x cols, float64."""
    x = g / (torch.linalg.matrix_norm(g) + 1e-7)
    for a, b, c in coefficients:
        q = x @ x.t() if x.shape[0] <= x.shape[1] else x.t() @ x
        p = a * torch.eye(q.shape[0], dtype=torch.float64, device=q.device) + b * q + c * (q @ q)
        x = p @ x if x.shape[0] <= x.shape[1] else x @ p
    return x


def orth_bound(g, coefficients):
    """First-order bound of |computed - exact|_F before the rounding to BF16, from the roundings the operator makes.

    In every step: the operands X, A = X X' - t I and P = (b + 2 c t) A + c A^2 are rounded to FP16 (u = 2^-11), X is kept in
    two FP16 numbers (2^-22), sums are FP32.  An error E of X after step k, in the basis of the singular vectors, reaches the
    result multiplied entry by entry by divided differences of the remaining polynomial F: (F_i - F_j) / (s_i - s_j) or
    (F_i + F_j) / (s_i + s_j).  A rounding of A or P is met by X, so its column j carries s_j; the rounding of the
    operand X is met by P, so its row i carries p_i; the rounding of the pair carries nothing."""
    u = 2.0 ** -11
    s = torch.linalg.svdvals(g.cpu().double())
    n, m = s.numel(), max(g.shape)
    s = s / (s.norm() + 1e-7)
    chain = [s]
    for a, b, c in coefficients:
        s = s * (a + b * s ** 2 + c * s ** 4)
        chain.append(s)
    last = chain[-1]

    def weights(k):
        """Largest factor with which an entry (i, j) of an error of X after step k reaches the result: n x n."""
        z = chain[k + 1]
        if k + 1 == len(coefficients):
            return torch.ones(n, n, dtype=torch.float64)
        d = z[:, None] - z[None, :]
        slope = torch.ones(n, dtype=torch.float64)
        y = z
        for a, b, c in coefficients[k + 1:]:
            slope = slope * (a + 3 * b * y ** 2 + 5 * c * y ** 4)
            y = y * (a + b * y ** 2 + c * y ** 4)
        minus = torch.where(d.abs() > 1e-6, (last[:, None] - last[None, :]) / torch.where(d.abs() > 1e-6, d, torch.ones_like(d)),
                            torch.maximum(slope.abs()[:, None], slope.abs()[None, :]))
        t = z[:, None] + z[None, :]
        plus = torch.where(t.abs() > 1e-12, (last[:, None] + last[None, :]) / torch.where(t.abs() > 1e-12, t, torch.ones_like(t)), slope.abs()[:, None])
        return torch.maximum(minus.abs(), plus.abs())

    total = 0.0
    for k, (a, b, c) in enumerate(coefficients):
        s = chain[k]
        w = weights(k)
        t = float((s ** 2).mean())
        t = t if t >= 0.2 else 0.0
        A = s ** 2 - t
        P = (b + 2 * c * t) * A + c * A ** 2
        # FP32 sums of tensor-core products, K / 16 of them, each within 2^-22 of the magnitudes (in norm at most |X|^2 and |A|^2, n-fold)
        dA = u * float(A.norm()) + (m / 16 + 1) * 2.0 ** -22 * float(s.norm()) ** 2
        dP = abs(b + 2 * c * t) * dA + 2 * abs(c) * float(A.abs().max()) * dA + u * float(P.norm()) + (n / 16 + 1) * 2.0 ** -22 * abs(c) * float(A.norm()) ** 2
        total += dP * float((w * s[None, :]).max())
        total += u * float(s.norm()) * float((w * P.abs()[:, None]).max())
        total += ((n / 16 + 1) * 2.0 ** -22 * float(P.norm()) + 2.0 ** -21 * (abs(a) + 1)) * float(s.norm()) * float(w.max())
    return total * 1.05                                     # the second order
