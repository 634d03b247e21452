"""The orthogonalisation with the roundings that the operator documents and everything else in 64 bits, and the operator's result before
its own rounding to BF16.  With both at hand a test sees the last bits that the design keeps, not only the final rounding."""
import math

import torch

import clblas_b200 as cb

SX, SA = 4096.0, 256.0                                        # scales of the stored X and of the stored Gram matrix and polynomial


def half(x):
    return x.to(torch.float16).double()


def exponent_of(v):
    """x with v = m 2^x, m in [0.5, 1)."""
    return math.frexp(v)[1]


def product(a, b):
    return a @ b


def truncating_product(a, b):
    """A sum in FP32 that is cut off after every 16 terms: no accumulator of a k = 16 instruction is worse."""
    acc = torch.zeros(a.shape[0], b.shape[1], dtype=torch.float64, device=a.device)
    for k in range(0, a.shape[1], 16):
        acc = ((acc + a[:, k:k + 16] @ b[k:k + 16]).view(torch.int64) & ~((1 << 29) - 1)).view(torch.float64)
    return acc


def orth_emulated(g, coefficients, shift=True, low=True, gram=half, scaled=True, spread=False, mul=product):
    """NS(G), rows x cols, as the operator rounds it: X = hi + lo in two FP16 numbers times 2^e, the products take hi, the Gram matrix
    minus its mean diagonal and the polynomial are FP16; what the shift takes from the polynomial goes to hi, and to lo in the steps after which
    |a| multiplies to 4 at most; sums are exact here.  The switches leave out what the design rests on (the shift, the low half, FP16
    for the Gram matrix, the power of two, the last rule), for tests of the tests; mul: how products are summed."""
    g = g.double()
    flip = g.shape[0] > g.shape[1]
    if flip:
        g = g.t()
    n = g.shape[0]
    eye = torch.eye(n, dtype=torch.float64, device=g.device)
    size = float(g.norm()) / (float(g.norm()) + 1e-7)
    e = max(0, -exponent_of(size)) if scaled and size > 0 else 0
    y = (g / (float(g.norm()) + 1e-7)) * 2.0 ** e * SX
    for k, (a, b, c) in enumerate(coefficients):
        hi = half(y)
        lo = half(y - hi) if low else torch.zeros_like(y)
        q2 = float((y / SX).square().sum())
        mean = q2 / n
        t = mean if shift and mean * 4.0 ** -e >= 0.2 else 0.0
        A = gram(mul(hi, hi.t()) * (SA / SX ** 2) - SA * t * eye)
        grown = abs(b) * q2 + abs(c) * q2 * q2 * 4.0 ** -e
        p = max(0, 2 * e - exponent_of(grown)) if scaled and grown > 0 else 0
        bk, ck = b * 4.0 ** -e, c * 16.0 ** -e
        P = half(2.0 ** p * ((bk + 2 * ck * t) * A + (ck / SA) * mul(A, A))) * 2.0 ** -p if c else bk * A
        bound = math.sqrt(q2) * (abs(a) + grown * 4.0 ** -e)
        after = max(0, e - exponent_of(bound)) if scaled and bound > 0 else e
        kappa = t * (bk + ck * t)
        growth = math.prod(abs(x[0]) for x in coefficients[k + 1:])
        y = ((a + kappa) * hi + (a + kappa if spread or growth <= 4 or n == 1 else a) * lo + mul(P, hi) / SA) * 2.0 ** (after - e)
        e = after
    x = y / SX * 2.0 ** -e
    return x.t() if flip else x


def before_rounding(g, want, coefficients, code, order=cb.clblasRowMajor):
    """The operator's NS(G) for the matrices of a batch (batch x lines x length, contiguous) before its rounding to BF16: with O = -w, w
    = `want` rounded to BF16, and beta = 1 the call returns NS(G) - w, computed in FP32 and rounded relative to the small difference."""
    batch, lines, length = g.shape
    w = want.bfloat16()
    o = (-w).contiguous()
    M, N = (lines, length) if order == cb.clblasRowMajor else (length, lines)
    cb.check(cb.clblasB200Orthogonalize(order, M, N, batch, len(coefficients), list(coefficients), 1.0, code, g, 0, length, lines * length,
                                        1.0, o, 0, length, lines * length), "orthogonalize")
    return w.double() + o.double()


def _reach(chain, coefficients, k):
    """n x n: the largest factor with which entry (i, j), in the basis of the singular vectors, of an error of X after step k reaches the
    result: the divided differences of the remaining polynomial (or its slope, where two values meet)."""
    z, last = chain[k + 1], chain[-1]
    n = z.numel()
    if k + 1 == len(coefficients):
        return torch.ones(n, n, dtype=torch.float64)
    slope, y = torch.ones(n, dtype=torch.float64), z
    for a, b, c in coefficients[k + 1:]:
        slope = slope * (a + 3 * b * y ** 2 + 5 * c * y ** 4)
        y = y * (a + b * y ** 2 + c * y ** 4)
    steep = torch.maximum(slope.abs()[:, None], slope.abs()[None, :])
    d, t = z[:, None] - z[None, :], z[:, None] + z[None, :]
    near = d.abs() <= 1e-6 * t
    minus = torch.where(near, steep, (last[:, None] - last[None, :]).abs() / torch.where(near, torch.ones_like(d), d.abs()))
    plus = torch.where(t > 0, (last[:, None] + last[None, :]).abs() / torch.where(t > 0, t, torch.ones_like(t)), steep)
    return torch.maximum(minus, plus)


def gram_operand_bound(g, coefficients):
    """First-order bound, in the Frobenius norm of the result, of what rounding the operand of the Gram product alone does.  With hi = X + D,
    |D_ij| <= u |x_ij|:  |hi hi' - X X'| = |X D' + D X'| <= 2 s_max |D| <= 2 u s_max |X|.  P follows with the factor |b + 2 c t| + 2 |c| |A|, and
    meets X: column j carries s_j."""
    u = 2.0 ** -11
    s = torch.linalg.svdvals(g.cpu().double())
    s = s / (s.norm() + 1e-7)
    chain = [s]
    for a, b, c in coefficients:
        s = s * (a + b * s ** 2 + c * s ** 4)
        chain.append(s)
    total = 0.0
    for k, (a, b, c) in enumerate(coefficients):
        s = chain[k].abs()
        t = float((s ** 2).mean())
        t = t if t >= 0.2 else 0.0
        dA = 2 * u * float(s.max()) * float(s.norm())
        total += (abs(b + 2 * c * t) + 2 * abs(c) * float((s ** 2 - t).abs().max())) * dA * float((_reach(chain, coefficients, k) * s[None, :]).max())
    return total * 1.05                                     # the second order
