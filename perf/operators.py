"""Workloads of the narrow-type operators: 8-bit products with scales, the quantisation that feeds them, and the
orthogonalisation of an update by Newton-Schulz products.

Three operators, each beside one that the library has in wider types:

  quantize   Q, s with X ~ diag(s) Q (one scale per row) or Q diag(s) (one per column), 8-bit integers
  i8gemm     C <- alpha diag(sA) op(A) op(B) diag(sB) + beta C, A and B in 8-bit integers
  orth       O <- alpha NS(G) + beta O, NS the matrix polynomial that pushes the singular values of G towards one

A case is a dict of plain values; `prepare` makes its inputs on the GPU, `run` is one pass (elementary torch operations, or
the library's own entry points where `own` is true), `exact` the same outputs from the definition in 64 bits.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}          # clblasB200Float32, clblasB200Float16, clblasB200Bfloat16
QUINTIC = (3.4445, -4.7750, 2.0315)              # the coefficients of the Muon optimiser, the library's default
EPS = 1e-7


def listed():
    return [
        # the activations of a decoding batch: a few long rows, where the call itself is what costs
        {"name": "quantize 16 tokens", "op": "quantize", "order": "row", "side": "left", "M": 16, "N": 4096, "pad": 0, "type": "bf16"},
        # the activations of a prompt
        {"name": "quantize a prompt", "op": "quantize", "order": "row", "side": "left", "M": 8192, "N": 8192, "pad": 0, "type": "bf16"},
        # a weight kept with its output channels along the contiguous axis: the maximum runs across the rows
        {"name": "quantize weight columns", "op": "quantize", "order": "row", "side": "right", "M": 4099, "N": 2300, "pad": 5, "type": "f32"},
        # a linear layer for one decoded token
        {"name": "i8gemm one token", "op": "i8gemm", "order": "row", "ta": "n", "tb": "t", "M": 1, "N": 4096, "K": 4096, "pad": 0, "type": "bf16", "beta": 0.0},
        # a linear layer for a decoding batch
        {"name": "i8gemm 48 tokens", "op": "i8gemm", "order": "row", "ta": "n", "tb": "t", "M": 48, "N": 8192, "K": 8192, "pad": 0, "type": "f16", "beta": 0.0},
        # packed prompts of no round length, added to the residual that stands in C, rows with a pitch of their own
        {"name": "i8gemm ragged residual", "op": "i8gemm", "order": "row", "ta": "n", "tb": "t", "M": 1000, "N": 5000, "K": 2056, "pad": 8, "type": "bf16", "beta": 0.5},
        # BLAS order, A as it is stored (contiguous along M), 32-bit result
        {"name": "i8gemm column-major n/n", "op": "i8gemm", "order": "col", "ta": "n", "tb": "n", "M": 2048, "N": 4096, "K": 2048, "pad": 0, "type": "f32", "beta": 0.0},
        # a linear layer over a long prompt
        {"name": "i8gemm a prompt", "op": "i8gemm", "order": "row", "ta": "n", "tb": "t", "M": 8192, "N": 8192, "K": 8192, "pad": 0, "type": "bf16", "beta": 0.0},
        # one small projection: a chain of short dependent products
        {"name": "orth one small matrix", "op": "orth", "order": "row", "M": 256, "N": 1024, "batch": 1, "pad": 0, "type": "bf16", "beta": 0.0},
        # the equal matrices of a dozen layers in one call, momentum kept in 32 bits
        {"name": "orth twelve layers", "op": "orth", "order": "row", "M": 768, "N": 768, "batch": 12, "pad": 0, "type": "f32", "beta": 0.0},
        # a tall matrix of odd sizes, its 16-bit weight decayed and updated in the same call
        {"name": "orth tall update", "op": "orth", "order": "col", "M": 2601, "N": 1003, "batch": 2, "pad": 3, "type": "bf16", "beta": 0.99},
        # the up projection of a wide feed-forward block
        {"name": "orth wide matrix", "op": "orth", "order": "row", "M": 4096, "N": 16384, "batch": 1, "pad": 0, "type": "bf16", "beta": 0.0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["quantize", "i8gemm", "i8gemm", "orth", "orth"])
    order, pad = rng.choice(["row", "row", "col"]), rng.choice([0, 0, rng.randint(1, 40)])
    if op == "quantize":
        M, N = _log(rng, 1, 16384), _log(rng, 16, 16384)
        M = min(M, (1 << 26) // N)
        return {"op": op, "order": order, "side": rng.choice(["left", "left", "right"]), "M": M, "N": N, "pad": pad, "type": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if op == "i8gemm":
        M, N, K = _log(rng, 1, 8192), _log(rng, 64, 16384), _log(rng, 64, 16384)
        while M * N * K > 8192 ** 3:
            M, N, K = (M + 1) // 2, N, (K + 1) // 2
        ta, tb = rng.choice([("n", "t"), ("n", "t"), ("t", "n"), ("n", "n"), ("t", "t")])
        return {"op": op, "order": order, "ta": ta, "tb": tb, "M": M, "N": N, "K": K, "pad": pad, "type": rng.choice(["bf16", "bf16", "f16", "f32"]), "beta": rng.choice([0.0, 0.0, 0.5])}
    M, N, batch = _log(rng, 32, 4096), _log(rng, 32, 8192), _log(rng, 1, 16)
    while batch * min(M, N) ** 2 * max(M, N) > 4096 ** 2 * 8192:
        batch = max(1, batch // 2)
    return {"op": op, "order": order, "M": M, "N": N, "batch": batch, "pad": pad, "type": rng.choice(["bf16", "bf16", "f32", "f16"]), "beta": rng.choice([0.0, 0.0, 0.99])}


def _stored(order, rows, cols, trans="n"):
    """(lines, length of a line) of a rows x cols matrix op(X) as it is stored."""
    if trans == "t":
        rows, cols = cols, rows
    return (rows, cols) if order == "row" else (cols, rows)


def _view(buf, order, rows, cols, trans="n"):
    """op(X), rows x cols, as a view of the stored lines (a batch in front where there is one)."""
    v = buf[..., : _stored(order, rows, cols, trans)[1]]
    return v if (order == "row") == (trans == "n") else v.transpose(-1, -2)


def _normal(gen, lines, length, ld):
    return torch.randn(lines, ld, generator=gen, device="cuda")


def _i8(gen, lines, length, ld):
    """What quantisation to the largest magnitude of a row gives: whole numbers, roughly normal, the extremes present."""
    x = torch.randn(lines, ld, generator=gen, device="cuda")
    return (x * (127.0 / 4.0)).round_().clamp_(-127, 127).to(torch.int8)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c, dt = dict(case), TYPES[case["type"]]
    M, N, order, pad = c["M"], c["N"], c["order"], c["pad"]
    s = {"case": c}
    if c["op"] == "quantize":
        lines, length = _stored(order, M, N)
        # activations: every column has a size of its own, a few are outliers; every row too
        x = _normal(gen, lines, length, length + pad)
        x *= torch.exp(0.5 * torch.randn(length + pad, generator=gen, device="cuda"))
        x *= torch.exp(0.5 * torch.randn(lines, 1, generator=gen, device="cuda"))
        s["x"] = x.to(dt)
        ldq = length + pad
        s["q"] = torch.zeros(lines, ldq, dtype=torch.int8, device="cuda")
        s["scale"] = torch.zeros(M if c["side"] == "left" else N, device="cuda")
    elif c["op"] == "i8gemm":
        K = c["K"]
        for name, rows, cols, t in (("a", M, K, c["ta"]), ("b", K, N, c["tb"])):
            lines, length = _stored(order, rows, cols, t)
            s[name] = _i8(gen, lines, length, length + pad)
        s["sa"] = 0.01 * torch.exp(0.3 * torch.randn(M, generator=gen, device="cuda"))
        s["sb"] = 0.002 * torch.exp(0.3 * torch.randn(N, generator=gen, device="cuda"))
        lines, length = _stored(order, M, N)
        rms = 0.01 * 0.002 * (127.0 / 4.0) ** 2 * math.sqrt(K)
        s["c"] = (_normal(gen, lines, length, length + pad) * rms).to(dt)
    else:
        lines, length = _stored(order, M, N)
        # a gradient: a few strong directions above a floor of noise, so that the singular values spread over two decades
        r = max(1, min(M, N) // 16)
        w = 1.0 / torch.arange(1, r + 1, device="cuda")
        g = torch.empty(c["batch"], lines, length + pad, device="cuda")
        for k in range(c["batch"]):
            u = torch.randn(lines, r, generator=gen, device="cuda") * w
            v = torch.randn(r, length + pad, generator=gen, device="cuda")
            g[k] = u @ v + 0.3 * torch.randn(lines, length + pad, generator=gen, device="cuda")
        s["g"] = (0.01 * g).to(dt)
        s["o"] = (torch.randn(c["batch"], lines, length + pad, generator=gen, device="cuda") / math.sqrt(N)).to(torch.bfloat16)
    return s


def _orth_coefficients(case):
    """alpha of the update: a step of 0.02 where the weight is kept (beta != 0), the orthogonal factor itself otherwise."""
    return -0.02 if case["beta"] else 1.0


def _run_own(s):
    import clblas_b200 as cb

    c = s["case"]
    order = cb.clblasRowMajor if c["order"] == "row" else cb.clblasColumnMajor
    M, N = c["M"], c["N"]
    code = CODES[c["type"]]
    if c["op"] == "quantize":
        x, q, scale = s["x"], s["q"], s["scale"]
        side = cb.clblasLeft if c["side"] == "left" else cb.clblasRight
        st = cb.clblasB200QuantizeI8(order, side, M, N, code, x, 0, x.stride(0), q, 0, q.stride(0), scale, 0)
        out = {"q": _view(q, c["order"], M, N), "scale": scale}
    elif c["op"] == "i8gemm":
        a, b, y = s["a"], s["b"], s["c"]
        st = cb.clblasB200I8gemm(order, cb.clblasTrans if c["ta"] == "t" else cb.clblasNoTrans, cb.clblasTrans if c["tb"] == "t" else cb.clblasNoTrans, M, N, c["K"], 1.0,
                                 a, 0, a.stride(0), s["sa"], 0, b, 0, b.stride(0), s["sb"], 0, c["beta"], code, y, 0, y.stride(0))
        out = {"c": _view(y, c["order"], M, N)}
    else:
        g, o = s["g"], s["o"]
        st = cb.clblasB200Orthogonalize(order, M, N, c["batch"], 5, None, _orth_coefficients(c), code, g, 0, g.stride(1), g.stride(0),
                                        c["beta"], o, 0, o.stride(1), o.stride(0))
        out = {"o": _view(o, c["order"], M, N)}
    cb.check(st, c["op"])
    return out


def _run_plain(s):
    c = s["case"]
    M, N = c["M"], c["N"]
    if c["op"] == "quantize":
        x = _view(s["x"], c["order"], M, N).float()
        top = x.abs().amax(1 if c["side"] == "left" else 0, keepdim=True)
        full = torch.full_like(top, 127.0)
        scale = top / full
        inv = torch.where(top > 0, full / top, torch.zeros_like(top))
        q = (x * inv).round().to(torch.int8)
        return {"q": q, "scale": scale.reshape(-1)}
    if c["op"] == "i8gemm":
        a = _view(s["a"], c["order"], M, c["K"], c["ta"]).float()
        b = _view(s["b"], c["order"], c["K"], N, c["tb"]).float()
        y = _view(s["c"], c["order"], M, N)
        r = (a @ b) * s["sa"][:, None] * s["sb"]
        if c["beta"]:
            r = r + c["beta"] * y.float()
        y.copy_(r)
        return {"c": y}
    g = _view(s["g"], c["order"], M, N).float()
    flip = M > N
    x = g.transpose(-1, -2) if flip else g
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + EPS)
    a, b, d = QUINTIC
    for _ in range(5):
        p = x @ x.transpose(-1, -2)
        x = a * x + (b * p + d * (p @ p)) @ x
    x = _orth_coefficients(c) * (x.transpose(-1, -2) if flip else x)
    o = _view(s["o"], c["order"], M, N)
    if c["beta"]:
        x = x + c["beta"] * o.float()
    o.copy_(x)
    return {"o": o}


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    c = case
    M, N = c["M"], c["N"]
    size = {"f32": 4, "f16": 2, "bf16": 2}[c["type"]]
    if c["op"] == "quantize":
        lines = M if c["side"] == "left" else N
        return {"bytes": M * N * (size + 1) + 4 * lines, "flops": 3 * M * N}
    if c["op"] == "i8gemm":
        K = c["K"]
        return {"bytes": M * K + K * N + 4 * (M + N) + M * N * size * (2 if c["beta"] else 1), "flops": 2 * M * N * K}
    n, m = min(M, N), max(M, N)
    # the Gram matrix and its square are symmetric: half of each product is enough
    step = n * (n + 1) * m + n * n * (n + 1) + 2 * n * n * m
    return {"bytes": c["batch"] * M * N * (size + 2 * (2 if c["beta"] else 1)), "flops": 5 * c["batch"] * step}


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    M, N = c["M"], c["N"]
    if c["op"] == "quantize":
        x = _view(s["x"], c["order"], M, N).to(torch.float64)
        return {"q": None, "scale": torch.linalg.vector_norm(x, math.inf, dim=1 if c["side"] == "left" else 0) / 127.0}
    if c["op"] == "i8gemm":
        K = c["K"]
        a = torch.einsum("ik,i->ik", _view(s["a"], c["order"], M, K, c["ta"]).to(torch.float64), s["sa"].to(torch.float64))
        b = torch.einsum("kj,j->kj", _view(s["b"], c["order"], K, N, c["tb"]).to(torch.float64), s["sb"].to(torch.float64))
        return {"c": torch.addmm(_view(s["c"], c["order"], M, N).to(torch.float64), a, b, beta=c["beta"])}
    g = _view(s["g"], c["order"], M, N).to(torch.float64)
    a, b, d = QUINTIC
    out = torch.empty(c["batch"], M, N, dtype=torch.float64, device=g.device)
    for k in range(c["batch"]):
        # X (a + b X'X + d (X'X)^2) or (a + b XX' + d (XX')^2) X, whichever square is the smaller
        x = g[k] / (torch.linalg.matrix_norm(g[k]) + EPS)
        for _ in range(5):
            q = x.T @ x if M > N else x @ x.T
            p = a * torch.eye(q.shape[0], dtype=torch.float64, device=q.device) + q @ (b * torch.eye(q.shape[0], dtype=torch.float64, device=q.device) + d * q)
            x = x @ p if M > N else p @ x
        out[k] = x
    return {"o": _orth_coefficients(c) * out + c["beta"] * _view(s["o"], c["order"], M, N).to(torch.float64)}
