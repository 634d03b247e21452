"""The last bits of the orthogonalisation.  The operator's result before its rounding to BF16 is held against 64 bits, and its error against
that of the documented roundings, emulated with exact sums (E).  The roundings of one input are as good as random, but their size is not: emulations with
sums cut to FP32 after every 16 terms, or with noise of 2^-24 in every sum, have 0.92 to 1.04 E (one direction only: 0.89 to 1.24), while
an operator without the shift has 1.7 E and more on matrices of full rank, one without the low half 37 E and more on the others, one with
BF16 in place of FP16 3 E.  The largest element of those errors is at most 11 (23) times their root mean square; a lost element is 1000."""
import pytest
import torch

import clblas_b200 as cb
from tests.cases_narrow import QUINTIC, TYPES, orth_exact
from tests.cases_orth_rounding import before_rounding, orth_emulated, truncating_product

# (error / E, largest element / root mean square)
# half: singular values of one in half the directions, of nothing in the others; fifth likewise: the shift is on, and empty directions must stay empty
LIMITS = {"half": (1.3, 20.0), "fifth": (1.3, 20.0), "normal": (1.15, 20.0), "noisy": (1.15, 20.0), "decaying": (1.3, 20.0), "rank8": (1.3, 20.0), "rank1": (1.8, 45.0)}


def gradients(lines, length, batch, spectrum, kind, seed, device="cuda"):
    gen = torch.Generator(device=device).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=device)  # noqa: E731
    if spectrum == "normal":
        return r(batch, lines, length).to(TYPES[kind][0])
    k = min(lines, length)
    if spectrum in ("half", "fifth"):
        some = max(1, k // 2 if spectrum == "half" else -(-k // 5))
        u, v = torch.linalg.qr(r(batch, lines, some).double())[0], torch.linalg.qr(r(batch, length, some).double())[0]
        return (u @ v.transpose(1, 2)).to(TYPES[kind][0])
    at = torch.arange(k, device=device)
    w = {"decaying": 1.0 / (at + 1) ** 2, "rank8": (at < 8).float(), "rank1": (at < 1).float(), "noisy": (at < max(1, k // 16)) / (at + 1.0)}[spectrum]
    g = (r(batch, lines, k) * w) @ r(batch, k, length)
    if spectrum == "noisy":
        g += 0.3 * r(batch, lines, length)
    # the rank is that of the 64-bit values: rounded to 16 bits a matrix of rank 8 has a floor of noise, which is as good a case
    return g.to(TYPES[kind][0])


def ratios(got, exact, emulated):
    err = got - exact
    return float(err.norm() / (emulated - exact).norm()), float(err.abs().max() / err.square().mean().sqrt())


def as_measured(x, want):
    """x through the same measurement: its difference from `want` in BF16 is rounded to BF16 (2^-18 of the result: one step alone errs as little)."""
    w = want.bfloat16().double()
    return w + (x - w).bfloat16().double()


def check(g, chain, kind, spectrum, order=cb.clblasRowMajor):
    exact = torch.stack([orth_exact(m.double(), chain) for m in g])
    got = before_rounding(g.contiguous(), exact, chain, TYPES[kind][1], order)
    limit, largest = LIMITS[spectrum]
    for i, m in enumerate(g):
        of_rms, top = ratios(got[i], exact[i], as_measured(orth_emulated(m, chain), exact[i]))
        assert of_rms <= limit and top <= largest, (i, of_rms, top)


def test_the_limits_see_what_the_design_rests_on():
    """On the CPU: the emulated operator with other sums stays within the limits, and loses them without the shift, the low half, FP16 or
    eight elements at an edge."""
    n, m, chain = 100, 130, [QUINTIC] * 5
    for spectrum, (limit, largest) in LIMITS.items():
        g = gradients(n, m, 1, spectrum, "f32", 3, "cpu")[0].double()
        exact, e = orth_exact(g, chain), orth_emulated(g, chain)
        of_rms, top = ratios(orth_emulated(g, chain, mul=truncating_product), exact, e)
        assert of_rms <= limit and top <= largest, spectrum
        broken = [orth_emulated(g, chain, gram=lambda x: x.to(torch.bfloat16).double())]
        if spectrum in ("normal", "noisy"):
            broken.append(orth_emulated(g, chain, shift=False))
        if spectrum not in ("normal", "half", "fifth"):
            broken.append(orth_emulated(g, chain, low=False))
        if spectrum in ("half", "fifth"):
            broken.append(orth_emulated(g, chain, spread=True))
        edge = e.clone()
        edge[n - 1, m - 8:] = 0
        for x in broken + [edge]:
            of_rms, top = ratios(x, exact, e)
            assert of_rms > limit or top > largest, spectrum


# n x m x batch: the plans of the Gram product, the square and the update (every one of each), or the CTAs of the single kernel
SHAPES = [(64, 64, 1, "_small<1>"), (100, 130, 3, "_small<4>"), (128, 512, 1, "_small<8>"), (90, 700, 40, "_small<4>"), (128, 2048, 2, "_small<8>"),
          (60, 200, 70, "_small<2>"), (120, 250, 200, "_small<1>"),
          (130, 131, 2, "<split128x2,split128x2,split128x2>"), (193, 196, 2, "<split128x4,split128x4,split128x4>"), (129, 194, 1, "<split128x4,split128x2,split128x2>"),
          (130, 132, 26, "<split128x1,split128x1,split128x1>"), (263, 266, 19, "<split128x1,split128x1,pairs128>"), (261, 540, 25, "<pairs256,split128x1,split128x1>"),
          (393, 402, 15, "<pairs256,pairs256,pairs256>"), (684, 1146, 5, "<split128x1,split128x1,pairs128>"), (768, 768, 12, "<pairs256,pairs256,pairs256>"),
          (256, 1024, 1, None), (1003, 2601, 2, "<split128x2,split128x2,pairs256>")]


@pytest.mark.gpu
@pytest.mark.parametrize("n,m,batch,plan", SHAPES)
@pytest.mark.parametrize("tall", [False, True])
@pytest.mark.parametrize("spectrum", ["normal", "noisy"])
def test_shapes(n, m, batch, plan, tall, spectrum):
    lines, length = (m, n) if tall else (n, m)
    kind = "f32" if tall == (spectrum == "normal") else "bf16"
    check(gradients(lines, length, batch, spectrum, kind, n + m), [QUINTIC] * 5, kind, spectrum, cb.clblasColumnMajor if tall else cb.clblasRowMajor)
    assert plan is None or cb.last_gemm_variant() == "orthogonalize" + plan


@pytest.mark.gpu
@pytest.mark.parametrize("n,m", [(100, 130), (300, 300), (256, 1024), (384, 700)])
@pytest.mark.parametrize("spectrum", sorted(LIMITS))
def test_spectra(n, m, spectrum):
    check(gradients(n, m, 3, spectrum, "f32", 5), [QUINTIC] * 5, "f32", spectrum)


@pytest.mark.gpu
@pytest.mark.parametrize("n,m", [(40, 90), (100, 130), (300, 300), (256, 1024)])
@pytest.mark.parametrize("spectrum", ["normal", "half", "fifth"])
@pytest.mark.parametrize("steps", [5, 7, 9])
def test_partial_rank_and_more_steps(n, m, spectrum, steps):
    """What is lost in the empty directions grows by 3.4 in every step: against 64 bits alone, with the error that the header states."""
    g, chain = gradients(n, m, 2, spectrum, "f32", 8), [QUINTIC] * steps
    exact = torch.stack([orth_exact(x.double(), chain) for x in g])
    got = before_rounding(g, exact, chain, TYPES["f32"][1])
    for i in range(2):
        assert float((got[i] - exact[i]).norm()) <= (3e-3 if steps == 5 else 1e-2) * float(exact[i].norm()), i


@pytest.mark.gpu
@pytest.mark.parametrize("chain", [[QUINTIC], [QUINTIC] * 2, [(1.5, -0.5, 0.0)] * 6, [(4.0, -6.0, 2.8), (3.9, -5.6, 2.6), (3.0, -3.2, 1.2), (1.875, -1.25, 0.375)]])
@pytest.mark.parametrize("n,m", [(120, 200), (300, 420)])
def test_steps_and_coefficients(n, m, chain):
    check(gradients(n, m, 3, "normal", "f32", 6), chain, "f32", "normal")
    assert cb.lib.clblasB200DeviceFault() == 0
