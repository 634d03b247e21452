// Pieces shared by the two forms of the Newton-Schulz orthogonalisation: the chain of products (orthogonalize.cu) and the single
// kernel for small matrices (orthogonalize_small.cu).
#pragma once

#include "narrow_mma.cuh"

namespace cb200 {

// One cluster per matrix, everything on chip (orthogonalize_small.cu).
bool orthogonalize_small_applies(const OrthProblem& p);
template <typename T>
cudaError_t orthogonalize_small(const OrthProblem& p, cudaStream_t s);
unsigned orthogonalize_small_fault_flag();

namespace {

// Scales, norm and roundings are described in orthogonalize.cu.
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

// x * f0 * f1 = x * SX / (norm + eps): the factor may lie outside FP32, so it is a power of two and a number in [1, 2).  NaN when the norm
// is not finite.  square: |X0|_F^2.
__device__ __forceinline__ void norm_factors(double norm, float& f0, float& f1, double& square)
{
    const double f = 1.0 / (norm + EPS);
    int e;
    const double m = frexp(f * SX, &e);
    f0 = isfinite(norm) ? (float)ldexp(1.0, e - 1) : nanf("");
    f1 = (float)(2.0 * m);
    square = isfinite(norm) ? norm * f * norm * f : 0;
}

// The shift t: the mean diagonal of X X', once most singular values have come near one; 0 before (and for a matrix of NaN, whose
// sum says nothing).  While X is dominated by a few directions the shift would put roundings of t on all the others
// (rank 8 of 100: 3e-3 with t from the first step on, 7e-4 from t = 0.2 on).
__device__ __forceinline__ float shift(float mean) { return mean >= 0.2f ? mean : 0.f; }

}  // namespace
}  // namespace cb200
