// Pieces shared by the two forms of the Newton-Schulz orthogonalisation: the chain of products (orthogonalize.cu) and the single
// kernel for small matrices (orthogonalize_small.cu).
#pragma once

#include "narrow_mma.cuh"

#include <cmath>

namespace cb200 {

// One cluster per matrix, everything on chip (orthogonalize_small.cu).
bool orthogonalize_small_applies(const OrthProblem& p);
template <typename T>
cudaError_t orthogonalize_small(const OrthProblem& p, cudaStream_t s);
unsigned orthogonalize_small_fault_flag();

namespace {

// Norm and roundings are described in orthogonalize.cu.
constexpr float SX = 4096.f, SA = 256.f;                  // scales of the stored X and of the stored A, P
constexpr double SUM_UNIT = 16777216.0;                    // sums of squares are counted in 2^-24
constexpr double EPS = 1e-7;

typedef unsigned long long u64;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ uint32_t pack(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ float2 unpack(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }

// Sum of the squares of eight elements.  They are added in FP32 (within 2^-21), since a conversion of every element to 64 bits would
// take longer than loading them; where the squares could leave FP32's range they are converted one by one.  NaN passes either way.
__device__ __forceinline__ double sum_of_squares(const float (&x)[8])
{
    float top = 0.f, low = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++) { top = fmaxf(top, fabsf(x[j])); low = fmaf(x[j], x[j], low); }
    double sum = low;
    if (top > 1e18f || (top < 1e-15f && top > 0.f)) {
        sum = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) sum = fma((double)x[j], (double)x[j], sum);
    }
    return sum;
}

// Powers of two.  X is held as Y = 2^e X (times SX), e >= 0 one per matrix and step: for gradients whose norm is far below the 1e-7 of the
// definition X starts far below one, grows by a factor of about a in a step, and would lose its bits among FP16's smallest numbers.
// e brings a bound of |X|_F between one half and one, and is 0 where that bound is larger already.  In terms of Y the polynomial has the
// coefficients a, 4^-e b, 16^-e c.  P, which is far smaller than X there, is held times 2^p in the same way.
constexpr int MAX_EXPONENT = 300;

// v = m 2^x with m in [0.5, 1): plus - x, within [0, MAX_EXPONENT]; 0 for 0 and for what is not finite.
__device__ __forceinline__ int raising(float v, int plus)
{
    int x = 0;
    if (!(v > 0.f && v < INFINITY)) return 0;
    frexpf(v, &x);
    return min(max(plus - x, 0), MAX_EXPONENT);
}

// v = m 2^x with m in [0.5, 1), for normal v (frexp and ldexp took 1 us of a small call).
__device__ __forceinline__ double mantissa(double v, int& x)
{
    const int top = __double2hiint(v);
    x = ((top >> 20) & 0x7ff) - 1022;
    return __hiloint2double((top & 0x000fffff) | 0x3fe00000, __double2loint(v));
}
__device__ __forceinline__ double power_of_two(int x) { return __hiloint2double((x + 1023) << 20, 0); }

// x * f0 * f1 = x * 2^e SX / (norm + eps): the factor may lie outside FP32, so it is divided between two (the norm of an FP32 matrix that
// is not zero lies between 2^-149 and 2^160).  NaN when the norm is not finite.  square: |Y0|_F^2.
__device__ __forceinline__ void norm_factors(double norm, float& f0, float& f1, double& square, int& e)
{
    const double f = 1.0 / (norm + EPS), size = norm * f;
    e = 0;
    if (!isfinite(norm)) { f0 = f1 = nanf(""); square = 0; return; }
    int x;
    if (size > 0 && size < 0.5) {
        mantissa(size, x);
        e = -x;
    }
    const double raise = power_of_two(e), m = mantissa(f * SX * raise, x);
    f0 = (float)power_of_two((x - 1) / 2);
    f1 = (float)(2.0 * m) * (float)power_of_two(x - 1 - (x - 1) / 2);
    square = size * raise * (size * raise);
}

// The shift: the mean diagonal of Y Y' once most singular values of X have come near one; 0 before (and for a matrix of NaN, whose sum says
// nothing).
__device__ __forceinline__ float shift(float mean, int e) { return (e == 0 ? mean : ldexpf(mean, -2 * e)) >= 0.2f ? mean : 0.f; }

// A step in terms of what is stored: P <- b A + f A A, Y <- w hi + v lo + g P hi (A in place of P when c == 0); next: the exponent of X after
// it.  Of w, kappa = b t + c t^2 is what the shift took from P.
struct StepFactors { float b, f, w, v, g; int next; };

// q2: |Y|^2, t: the shift.  The bounds, q = |X|_F: |X after the step|_F <= |a| q + |b| q^3 + |c| q^5, |P| <= 3 (|b| q^2 + |c| q^4) whatever t.
// Not inlined: the kernel for small matrices has no registers to spare for it.
__device__ __noinline__ StepFactors step_factors_scaled(float q2, float t, int e, float a, float b, float c, bool last, float scale, bool kappa_lo)
{
    const float grown = fabsf(b) * q2 + ldexpf(fabsf(c) * q2 * q2, -2 * e);                    // 4^e (|b| q^2 + |c| q^4)
    const float bound = sqrtf(q2) * (fabsf(a) + ldexpf(grown, -2 * e));                        // 2^e of the bound of X
    const int p = min(raising(grown, 2 * e), 2 * e + 40);                                      // c 2^(p - 4 e) stays in FP32's range
    StepFactors s;
    s.next = bound > 0.f ? raising(bound, e) : e;
    const float cp = ldexpf(c, p - 4 * e);
    s.b = ldexpf(b, p - 2 * e) + 2.f * cp * t;
    s.f = cp / SA;
    const int by = last ? -e : s.next - e;
    s.w = ldexpf(scale, by) * (a + t * (ldexpf(b, -2 * e) + ldexpf(c, -4 * e) * t));
    s.v = kappa_lo ? s.w : ldexpf(scale, by) * a;
    s.g = ldexpf(scale * ((c == 0.f ? b : 1.f) / SA), by - (c == 0.f ? 2 * e : p));
    return s;
}

// In the last step Y is left times `scale` (alpha / SX) and without its power of two.  kappa_lo: kappa multiplies lo too (orthogonalize.cu).
__device__ __forceinline__ StepFactors step_factors(float q2, float t, int e, float a, float b, float c, bool last, float scale, bool kappa_lo)
{
    if (!last) scale = 1.f;
    // The same without powers of two: the rule for gradients of ordinary size.
    const float grown = fabsf(b) * q2 + fabsf(c) * q2 * q2, sum = fabsf(a) + grown;
    if (e == 0 && grown >= 0.5f && q2 * sum * sum >= 0.25f)
        return {b + 2.f * c * t, c / SA, scale * (a + t * (b + c * t)), scale * (kappa_lo ? a + t * (b + c * t) : a), scale * ((c == 0.f ? b : 1.f) / SA), 0};
    return step_factors_scaled(q2, t, e, a, b, c, last, scale, kappa_lo);
}

// Whether a step may put kappa on lo (orthogonalize.cu): what it leaves in empty directions grows by |a| in every step after it.  A matrix
// of one row has none.
inline bool kappa_on_lo(size_t n, const float* coeffs, int step, int steps)
{
    if (n == 1) return true;
    float growth = 1.f;
    for (int k = step + 1; k < steps; k++) growth *= fabsf(coeffs ? coeffs[3 * k] : 3.4445f);
    return growth <= 4.f;
}

}  // namespace
}  // namespace cb200
