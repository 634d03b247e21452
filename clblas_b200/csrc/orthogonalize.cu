// Orthogonalisation of an update by Newton-Schulz products: with X0 = G / (|G|_F + 1e-7), k steps of
//     X <- a X + (b X X' + c (X X')^2) X
// push every singular value of G towards one and keep its singular vectors; O <- alpha X + beta O.  (No counterpart in the
// reference; the products are of its SYRK and SYMM families.  Optimisers that orthogonalise the momentum of a weight use it.)
//
// On the smaller side n of the matrix (n <= m) a step is three products: the Gram matrix (symmetric, n^2 m operations), its
// square (symmetric, n^3) and the update (2 n^2 m).  All run on the FP16 tensor-core tiles of narrow_mma.cuh, the symmetric ones on
// the tiles of one triangle, each result stored at both places.  (Matrices up to 128 x 1024, and up to 128 x 2048 where
// there are at most 15, take one kernel instead of the chain: orthogonalize_small.cu.)
//
// Measured, five steps: 4096 x 16384 BF16 4.1 to 4.3 ms back to back under the power cap (Gram 205 us, square 61, update 410: the
// tiles without their epilogues 329, the rest is the 8 bytes an element that X costs to read and write); twelve 768 x 768 FP32 264 us
// (15, 17, 29 us a step); two 2601 x 1003 256 us; 256 x 1024 96 us, of which launches and first loads are most.
//
// What is kept in how many bits, and why:
//   * X is a pair of FP16 numbers, hi + lo (22 bits); a X uses the pair, the products use hi.  Singular values far below the
//     others grow by a factor of about a in every step; a rounding of X itself would put noise on them that grows as
//     fast (rank-8 gradient, five steps: 4 % of the result with X in FP16 alone, 34 % in BF16).  A rounding inside the products
//     meets X once more and does not grow.
//   * The Gram matrix is stored as A = X X' - t I, t its mean diagonal, and P = (b + 2 c t) A + c A^2; X <- (a + b t + c t^2) X + P X is the
//     same polynomial.  Near the end X X' is close to I and b, c nearly cancel: rounding the small difference instead
//     halves the error of the result (normal 768 x 768: 1.5e-3 without, 7e-4 with t; the final rounding to BF16 is 1.7e-3).
//   * Of the coefficient of X in that form, kappa = b t + c t^2 stands for what the shift took from P, which meets hi alone.  On lo it is right
//     where the singular values are near one, and wrong by kappa lo where X has no component: the rounding of X would appear in empty
//     directions and grow by a in every step (rank 50 of 100: 5e-3 of the result after five steps, 6 % after seven, 70 % after nine).  So kappa
//     multiplies lo only in the steps after which |a| multiplies to 4 at most, the last two of the default ones: 1.8e-3, 3.2e-3, 2.4e-3
//     (and with it nowhere 1.8e-3, 3.3e-3, 2.4e-3, but 1.2e-3 instead of 7e-4 for a normal 256 x 1024).  Where all singular values lie close
//     together kappa on lo would be right throughout (a normal 64 x 8192: 2e-4 instead of 9e-4); asking |X X' - t I|_F^2 < t^2, which
//     tells those apart, cost 2 to 6 % of the kernel for small matrices and is hidden by the rounding to BF16, 1.7e-3.
//   * t comes from the sum of the squares of X, gathered in 64-bit integers (units of 2^-24), so the order of the atomic additions does
//     not change it.  Any t gives the same polynomial; it only has to be near.
//   * Accumulators and everything between accumulator and store are FP32.  The tensor core cuts its sums off instead of rounding them, so a
//     long one falls behind, by about 2^-25 for every 16 terms (8 x 2^20: 1.5e-3 of the result, 8 x 2^24: 2.3 %).  Beyond SEGMENT elements the Gram
//     product is therefore taken in segments, which are added up in ordinary FP32 (8 x 2^24: 1.9e-4).  X is held times 2^12, A and P times 2^8, so that the
//     entries of large matrices (about 1/sqrt(m)) stay far above FP16's smallest numbers, and times a power of two for each matrix where
//     the whole matrix is small (orthogonalize.cuh).  768 x 768, |G|_F = 1e-15: 32 % off without that power, 1e-7 with it (before BF16).
// The result is good to 3e-4 to 2e-3 after five steps and is therefore given in BF16 only.
#include "orthogonalize.cuh"

#include <algorithm>
#include <cstdio>
#include <type_traits>

namespace cb200 {

namespace {

using namespace narrow;

// ---- norm and split ---------------------------------------------------------------------------------------------------

// Eight consecutive elements, n of them valid, as loaded.  VEC: 16-byte loads (aligned lines, a whole piece).
template <typename T> struct alignas(16) Eight { T t[8]; };
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, unsigned n, Eight<T>& x)
{
    if (VEC && n == 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(Eight<T>) / 16; i++) reinterpret_cast<uint4*>(x.t)[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x.t[i] = i < (int)n ? p[i] : T(0.f);
    }
}

// Sums of squares in 64 bits, one per block; the blocks of a matrix share its pieces of eight elements evenly.  Clears the sums of the
// steps to come as well.  Bound by memory.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) sum_squares_kernel(const T* __restrict__ G, size_t lines, unsigned len, size_t ld, size_t stride,
                                                          double* __restrict__ part, u64* __restrict__ sums, int sums_pitch)
{
    pdl_launch_dependents();
    const T* g = G + blockIdx.y * stride;
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < sums_pitch; i += 256) sums[(size_t)blockIdx.y * sums_pitch + i] = 0;
    // Pieces of eight elements in the order of the matrix, the grid's threads apart; (line, piece of the line) is stepped by
    // (step / per_line, step % per_line), since a 64-bit division for every piece would bound the kernel.
    const unsigned per_line = (len + 7) / 8, step = gridDim.x * 256, at = blockIdx.x * 256 + threadIdx.x;
    const unsigned dl = step / per_line, dc = step % per_line;
    size_t l = at / per_line;
    unsigned c = at % per_line;
    double sum = 0;
    while (l < lines) {
        constexpr int AHEAD = 16 / sizeof(T);              // 128 bytes a thread in flight
        Eight<T> raw[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; k++) {
            load8<T, VEC>(g + l * ld + 8 * (size_t)c, l < lines ? min(8u, len - 8 * c) : 0, raw[k]);
            l += dl;
            c += dc;
            if (c >= per_line) { c -= per_line; l++; }
        }
#pragma unroll
        for (int k = 0; k < AHEAD; k++) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = to_f(raw[k].t[j]);
            sum += sum_of_squares(v);
        }
    }
    double all = sum;
    __shared__ double per_warp[8];
    for (int d = 16; d > 0; d >>= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
    if (threadIdx.x % 32 == 0) per_warp[threadIdx.x / 32] = all;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; w++) all += per_warp[w];
        part[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = all;
    }
}

// X0 = G / (|G| + eps), times 2^e SX, as hi + lo; FLIP: transposed on the way (G has more lines than elements per line).
// A matrix that holds a NaN or an infinity becomes NaN everywhere.  64 lines x 64 elements per CTA.  Bound by memory.  (`part` is written
// while this kernel is already resident: no `__restrict__`, which would allow loads as of constants.)
template <typename T, bool VEC, bool FLIP>
__global__ void __launch_bounds__(256) split_kernel(const T* G, size_t lines, size_t len, size_t ld, size_t stride, const double* part,
                                                    int parts, __half* __restrict__ hi, __half* __restrict__ lo, size_t ldx, size_t stride_x,
                                                    u64* __restrict__ sums, int* __restrict__ exps, int sums_pitch, unsigned tiles_len)
{
    __shared__ float factors[2];
    __shared__ float tile[FLIP ? 64 : 1][65];
    pdl_launch_dependents();
    const unsigned z = blockIdx.y;
    const size_t l0 = (size_t)(blockIdx.x / tiles_len) * 64, i0 = (size_t)(blockIdx.x % tiles_len) * 64;
    const T* g = G + z * stride;
    // A thread's two pieces of eight elements: lines k and k + 32 of the tile.  (Read before the norm is known.)
    const int piece = threadIdx.x % 8;
    const size_t i = i0 + 8 * piece;
    const unsigned n = i < len ? (unsigned)min((size_t)8, len - i) : 0;
    Eight<T> raw[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const size_t l = l0 + threadIdx.x / 8 + 32 * h;
        load8<T, VEC>(g + l * ld + i, l < lines ? n : 0, raw[h]);
    }
    pdl_wait();
    if (threadIdx.x < 32) {
        double sum = 0;
        for (int k = threadIdx.x; k < parts; k += 32) sum += part[(size_t)z * parts + k];
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (threadIdx.x == 0) {
            double square;
            int e;
            norm_factors(sqrt(sum), factors[0], factors[1], square, e);
            if (blockIdx.x == 0) {
                sums[(size_t)z * sums_pitch] = (u64)(square * SUM_UNIT);
                exps[(size_t)z * sums_pitch] = e;
            }
        }
    }
    __syncthreads();
    const float f0 = factors[0], f1 = factors[1];
    float x[2][8];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int j = 0; j < 8; j++) x[h][j] = to_f(raw[h].t[j]) * f0 * f1;
    size_t out_line[2], out_at;
    bool write[2];
    if (!FLIP) {
        out_at = i;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            out_line[h] = l0 + threadIdx.x / 8 + 32 * h;
            write[h] = out_line[h] < lines && n > 0;
        }
    } else {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int j = 0; j < 8; j++) tile[threadIdx.x / 8 + 32 * h][8 * piece + j] = x[h][j];
        __syncthreads();
        out_at = l0 + 8 * piece;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int c = threadIdx.x / 8 + 32 * h;
            out_line[h] = i0 + c;
            write[h] = out_line[h] < len && out_at < lines;
#pragma unroll
            for (int j = 0; j < 8; j++) x[h][j] = tile[8 * piece + j][c];
        }
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        if (!write[h]) continue;
        uint32_t a[4], r[4];                               // the pitch is a multiple of 8: what lies beyond the matrix is padding
#pragma unroll
        for (int j = 0; j < 4; j++) {
            a[j] = pack(x[h][2 * j], x[h][2 * j + 1]);
            const float2 t = unpack(a[j]);
            r[j] = pack(x[h][2 * j] - t.x, x[h][2 * j + 1] - t.y);
        }
        const size_t at = z * stride_x + out_line[h] * ldx + out_at;
        *reinterpret_cast<uint4*>(hi + at) = make_uint4(a[0], a[1], a[2], a[3]);
        *reinterpret_cast<uint4*>(lo + at) = make_uint4(r[0], r[1], r[2], r[3]);
    }
}

// ---- epilogues ----------------------------------------------------------------------------------------------------------

// What the Gram product of a step finds and leaves for the others.
struct Sizes {
    const u64* sums; int* exps;                            // sum of squares and exponent of every matrix before the step, `pitch` apart
    float4* factors;                                       // of the step, two each: (b, f) and (w, v, g) (StepFactors)
    int pitch;
    float n, a, b, c;
    bool last, kappa_lo;
    float scale;
};

// The workspaces have a pitch of a multiple of 8 elements: every row piece is aligned.
__device__ __forceinline__ uint16_t* bits(__half* p) { return reinterpret_cast<uint16_t*>(p); }
__device__ __forceinline__ const uint16_t* bits(const __half* p) { return reinterpret_cast<const uint16_t*>(p); }

// The product of one segment of X: S <- X X' or S + X X', on the tiles of the triangle.
struct EpiGramPart {
    static constexpr bool kHeavy = false;
    static constexpr bool kTriangle = true;
    struct State {};
    template <int G> struct Pre {};
    float* S; size_t ld, stride;
    bool first;
    // x += what S holds at its place (the same in all kernels: each element is read and written by one thread)
    template <int G>
    __device__ static void add(const float* S, size_t ld, const Shape& s, unsigned u0, unsigned v0, float (&x)[4][G][2])
    {
        const int lane = threadIdx.x & 31;
        float2 old[4][G];
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int k = 0; k < G; k++) {
                const unsigned u = u0 + 8 * g + lane / 4, v = v0 + 8 * k + 2 * (lane & 3);
                old[g][k] = u < s.U && v < s.V ? *reinterpret_cast<const float2*>(S + (size_t)u * ld + v) : make_float2(0.f, 0.f);
            }
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int k = 0; k < G; k++) {
                x[g][k][0] += old[g][k].x;
                x[g][k][1] += old[g][k].y;
            }
    }
    __device__ void begin(State&, const Shape&, unsigned, unsigned, unsigned) const {}
    template <int G> __device__ void fetch(Pre<G>&, const Shape&, unsigned, unsigned, unsigned) const {}
    template <int G>
    __device__ void chunk(State&, Pre<G>&, const Shape& s, unsigned z, unsigned u0, unsigned v0, unsigned, int where, float (&x)[4][G][2]) const
    {
        if (where == PART_ABOVE) return;
        float* to = S + z * stride;
        if (!first) add<G>(to, ld, s, u0, v0, x);
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int k = 0; k < G; k++) {
                const unsigned u = u0 + 8 * g + lane / 4, v = v0 + 8 * k + 2 * (lane & 3);      // the pitch is even: v + 1 is padding at most
                if (u < s.U && v < s.V) *reinterpret_cast<float2*>(to + (size_t)u * ld + v) = make_float2(x[g][k][0], x[g][k][1]);
            }
    }
    __device__ void end(State&, unsigned, unsigned) const {}
};

template <bool JOIN>                                       // JOIN: of the last segment, S holds the sum of the others
struct EpiGram {                                           // A <- X X' - t I
    static constexpr bool kHeavy = false;
    static constexpr bool kTriangle = true;
    struct State { float t; };
    template <int G> struct Pre {};
    __half* A; size_t ld, stride;
    Sizes sizes;
    const float* S;
    __device__ void begin(State& st, const Shape&, unsigned z, unsigned u0, unsigned v0) const
    {
        const size_t at = (size_t)z * sizes.pitch;         // read past L1: a neighbour is written meanwhile
        const float mean = (float)((double)__ldcg(sizes.sums + at) * (1.0 / SUM_UNIT)) * (1.f / sizes.n);
        const int e = __ldcg(sizes.exps + at);
        const float t = shift(mean, e);
        st.t = SA * t;
        // Once for a matrix: evaluated by every tile of the products that need them they took 0.35 us a kernel.
        if (u0 == 0 && v0 == 0 && (threadIdx.x & 31) == 0) {
            const StepFactors k = step_factors(mean * sizes.n, t, e, sizes.a, sizes.b, sizes.c, sizes.last, sizes.scale, sizes.kappa_lo);
            sizes.factors[2 * at] = make_float4(k.b, k.f, 0.f, 0.f);
            sizes.factors[2 * at + 1] = make_float4(k.w, k.v, k.g, 0.f);
            sizes.exps[at + 1] = k.next;
        }
    }
    template <int G> __device__ void fetch(Pre<G>&, const Shape&, unsigned, unsigned, unsigned) const {}
    template <int G>
    __device__ void chunk(State& st, Pre<G>&, const Shape& s, unsigned z, unsigned u0, unsigned v0, unsigned, int where, float (&x)[4][G][2]) const
    {
        if (JOIN && where != PART_ABOVE) EpiGramPart::add<G>(S + z * stride, ld, s, u0, v0, x);
        const int lane = threadIdx.x & 31;
        const int off = (int)(u0 + lane / 4) - (int)(v0 + 2 * (lane & 3));      // row - column of x[0][0][0]
        Bits16<G> o;
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int k = 0; k < G; k++) {
                float a = x[g][k][0] * (SA / (SX * SX)), b = x[g][k][1] * (SA / (SX * SX));
                const int d = off + 8 * (g - k);
                if (d == 0) a -= st.t;
                if (d == 1) b -= st.t;
                o.h[g][k] = pack(a, b);
            }
        if (where == PART_BELOW) store_columns16<G>(o, bits(A + z * stride), ld, u0, v0, s.U, s.V, PADDED);
        if (where != PART_ABOVE) store_rows16<G>(o, bits(A + z * stride), ld, u0, v0, s.U, s.V, PADDED);
    }
    __device__ void end(State&, unsigned, unsigned) const {}
};

struct EpiSquare {                                         // P <- (b + 2 c t) A + c A^2, times 2^p
    static constexpr bool kHeavy = false;
    static constexpr bool kTriangle = true;
    struct State { float b, f; };
    template <int G> struct Pre { Bits16<G> a; };
    const __half* A; __half* P; size_t ld, stride;
    const float4* factors; int pitch;
    __device__ void begin(State& st, const Shape&, unsigned z, unsigned, unsigned) const
    {
        const float4 k = __ldcg(factors + 2 * (size_t)z * pitch);
        st.b = k.x;
        st.f = k.y;
    }
    template <int G>
    __device__ void fetch(Pre<G>& p, const Shape& s, unsigned z, unsigned u0, unsigned v0) const
    {
        load_rows16<G>(p.a, bits(A + z * stride), ld, u0, v0, s.U, s.V, PADDED);
    }
    template <int G>
    __device__ void chunk(State& st, Pre<G>& p, const Shape& s, unsigned z, unsigned u0, unsigned v0, unsigned v_next, int where, float (&x)[4][G][2]) const
    {
        rows_to_fragments<G>(p.a, v0, s.V, PADDED);
        Bits16<G> o;
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int k = 0; k < G; k++) {
                const float2 a = unpack(p.a.h[g][k]);
                o.h[g][k] = pack(fmaf(st.b, a.x, st.f * x[g][k][0]), fmaf(st.b, a.y, st.f * x[g][k][1]));
            }
        if (v_next != ~0u) fetch<G>(p, s, z, u0, v_next);
        if (where == PART_BELOW) store_columns16<G>(o, bits(P + z * stride), ld, u0, v0, s.U, s.V, PADDED);
        if (where != PART_ABOVE) store_rows16<G>(o, bits(P + z * stride), ld, u0, v0, s.U, s.V, PADDED);
    }
    __device__ void end(State&, unsigned, unsigned) const {}
};

// Common part of the two updates: y = (a + b t + c t^2) X + P X.  P is P, or A with factor b when c == 0.
struct UpdateTerm {
    const __half* hi; const __half* lo; size_t ld, stride;
    const float4* factors; int pitch;
    template <int G> struct Pre { Bits16<G> h, l; };
    struct Factors { float w, v, g; };                     // of hi, of lo and of the product
    template <int G>
    __device__ void fetch(Pre<G>& p, const Shape& s, unsigned z, unsigned u0, unsigned v0) const
    {
        load_rows16<G>(p.h, bits(hi + z * stride), ld, u0, v0, s.U, s.V, PADDED);
        load_rows16<G>(p.l, bits(lo + z * stride), ld, u0, v0, s.U, s.V, PADDED);
    }
    __device__ Factors of(unsigned z) const
    {
        const float4 k = __ldcg(factors + 2 * (size_t)z * pitch + 1);
        return {k.x, k.y, k.z};
    }
    template <int G>
    __device__ void add(Pre<G>& p, const Shape& s, unsigned v0, const Factors& by, float (&x)[4][G][2]) const
    {
        rows_to_fragments<G>(p.h, v0, s.V, PADDED);
        rows_to_fragments<G>(p.l, v0, s.V, PADDED);
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int k = 0; k < G; k++) {
                const float2 h = unpack(p.h.h[g][k]), l = unpack(p.l.h[g][k]);
                x[g][k][0] = fmaf(by.w, h.x, fmaf(by.v, l.x, by.g * x[g][k][0]));
                x[g][k][1] = fmaf(by.w, h.y, fmaf(by.v, l.y, by.g * x[g][k][1]));
            }
    }
};

struct EpiUpdate {
    static constexpr bool kHeavy = true;
    static constexpr bool kTriangle = false;
    struct State { UpdateTerm::Factors by; float sum; };
    template <int G> using Pre = UpdateTerm::Pre<G>;
    UpdateTerm t;
    __half* hi; __half* lo;                                // lo may be the one that is read: each place is read, then written, by one thread
    u64* next;                                             // sums of the new X
    __device__ void begin(State& st, const Shape&, unsigned z, unsigned, unsigned) const
    {
        st.by = t.of(z);
        st.sum = 0.f;
    }
    template <int G> __device__ void fetch(Pre<G>& p, const Shape& s, unsigned z, unsigned u0, unsigned v0) const { t.fetch<G>(p, s, z, u0, v0); }
    template <int G>
    __device__ void chunk(State& st, Pre<G>& p, const Shape& s, unsigned z, unsigned u0, unsigned v0, unsigned v_next, int, float (&x)[4][G][2]) const
    {
        t.add<G>(p, s, v0, st.by, x);
        if (v_next != ~0u) fetch<G>(p, s, z, u0, v_next);
        const int lane = threadIdx.x & 31;
        Bits16<G> h, l;
        float sum = 0.f;
        const bool whole = u0 + 32 <= s.U && v0 + 8 * G <= s.V;
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int k = 0; k < G; k++) {
                const float a = x[g][k][0], b = x[g][k][1];
                h.h[g][k] = pack(a, b);
                const float2 r = unpack(h.h[g][k]);
                l.h[g][k] = pack(a - r.x, b - r.y);
                // outside the matrix the accumulators are zero but the fetched values may be anything: chosen, not multiplied by zero
                const unsigned v = v0 + 8 * k + 2 * (lane & 3);
                const bool in = whole || u0 + 8 * g + lane / 4 < s.U;
                sum += in && (whole || v < s.V) ? a * a : 0.f;
                sum += in && (whole || v + 1 < s.V) ? b * b : 0.f;
            }
        st.sum += sum;
        store_rows16<G>(h, bits(hi + z * t.stride), t.ld, u0, v0, s.U, s.V, PADDED);
        store_rows16<G>(l, bits(lo + z * t.stride), t.ld, u0, v0, s.U, s.V, PADDED);
    }
    __device__ void end(State& st, unsigned z, unsigned) const
    {
        float s = st.sum;
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (threadIdx.x % 32 == 0) {
            const double q = (double)s * (SUM_UNIT / ((double)SX * SX));
            if (q >= 0.5 && q < 1e18) atomicAdd(next + (size_t)z * t.pitch, (u64)(q + 0.5));
        }
    }
};

struct EpiOut {                                            // O <- alpha X + beta O
    static constexpr bool kHeavy = true;
    static constexpr bool kTriangle = false;
    struct State { UpdateTerm::Factors by; };
    template <int G> struct Pre { UpdateTerm::Pre<G> x; Bits16<G> o; };
    UpdateTerm t;
    uint16_t* O; size_t ldo, stride_o;                     // BF16
    float beta;                                            // (alpha is in the factors)
    bool flip;                                             // element (u, v) at O[v * ldo + u]
    int align;                                             // of O's lines
    __device__ void begin(State& st, const Shape&, unsigned z, unsigned, unsigned) const { st.by = t.of(z); }
    template <int G>
    __device__ void fetch(Pre<G>& p, const Shape& s, unsigned z, unsigned u0, unsigned v0) const
    {
        t.fetch<G>(p.x, s, z, u0, v0);
        if (beta == 0.f) return;
        if (flip) load_columns16<G>(p.o, O + z * stride_o, ldo, u0, v0, s.U, s.V, align);
        else load_rows16<G>(p.o, O + z * stride_o, ldo, u0, v0, s.U, s.V, align);
    }
    template <int G>
    __device__ void chunk(State& st, Pre<G>& p, const Shape& s, unsigned z, unsigned u0, unsigned v0, unsigned v_next, int, float (&x)[4][G][2]) const
    {
        t.add<G>(p.x, s, v0, st.by, x);
        uint16_t* o = O + z * stride_o;
        if (beta != 0.f) {
            if (flip) columns_to_fragments<G>(p.o);
            else rows_to_fragments<G>(p.o, v0, s.V, align);
#pragma unroll
            for (int g = 0; g < 4; g++)
#pragma unroll
                for (int k = 0; k < G; k++) {
                    const float2 old = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&p.o.h[g][k]));
                    x[g][k][0] = fmaf(beta, old.x, x[g][k][0]);
                    x[g][k][1] = fmaf(beta, old.y, x[g][k][1]);
                }
        }
        if (v_next != ~0u) fetch<G>(p, s, z, u0, v_next);
        Bits16<G> r;
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int k = 0; k < G; k++) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(x[g][k][0], x[g][k][1]);
                r.h[g][k] = *reinterpret_cast<const uint32_t*>(&b);
            }
        if (flip) store_columns16<G>(r, o, ldo, u0, v0, s.U, s.V, align);
        else store_rows16<G>(r, o, ldo, u0, v0, s.U, s.V, align);
    }
    __device__ void end(State&, unsigned, unsigned) const {}
};

// Longest sum of a Gram product: an error of up to 2.5e-4 on its diagonal, half of what rounding A to FP16 costs.
constexpr size_t SEGMENT = 1 << 17;

// ---- the chain ----------------------------------------------------------------------------------------------------------

template <typename T>
cudaError_t orthogonalize_typed(const OrthProblem& p, cudaStream_t s)
{
    if (orthogonalize_small_applies(p)) return orthogonalize_small<T>(p, s);
    const bool flip = p.lines > p.len;
    const size_t n = flip ? p.len : p.lines, m = flip ? p.lines : p.len, batch = p.batch;
    if (m >= (1u << 31)) return cudaErrorNotSupported;
    auto up = [](size_t v, size_t q) { return (v + q - 1) / q * q; };
    const size_t ldx = up(m, 8), ldn = up(n, 8), xs = n * ldx, as = n * ldn;
    const int pitch = p.steps + 1;
    // Blocks of the norm: about 8 pieces a thread, at most two blocks per SM over the batch.
    const size_t blocks = (p.lines * ((p.len + 7) / 8) + 2047) / 2048, most = std::max<size_t>(1, 2 * (size_t)sm_count() / batch);
    const size_t parts = std::min(blocks, most);
    // workspace: hi (two of them, read and written in turn), lo, A, P, sums of squares, exponents, factors, partial norms, sums of segments
    const size_t x_bytes = up(batch * xs * 2, 256), a_bytes = up(batch * as * 2, 256), sum_bytes = up(batch * pitch * 8, 256), exp_bytes = up(batch * pitch * 4, 256), factor_bytes = up(batch * pitch * 32, 256),
                 part_bytes = up(batch * parts * 8, 256), join_bytes = m > SEGMENT ? batch * as * 4 : 0;
    unsigned char* ws = nullptr;
    cudaError_t e = ws_alloc(reinterpret_cast<void**>(&ws), 3 * x_bytes + 2 * a_bytes + sum_bytes + exp_bytes + factor_bytes + part_bytes + join_bytes, s);
    if (e != cudaSuccess) return e;
    __half* hi[2] = {reinterpret_cast<__half*>(ws), reinterpret_cast<__half*>(ws + x_bytes)};
    __half* lo = reinterpret_cast<__half*>(ws + 2 * x_bytes);
    __half* A = reinterpret_cast<__half*>(ws + 3 * x_bytes);
    __half* P = reinterpret_cast<__half*>(ws + 3 * x_bytes + a_bytes);
    u64* sums = reinterpret_cast<u64*>(ws + 3 * x_bytes + 2 * a_bytes);
    int* exps = reinterpret_cast<int*>(ws + 3 * x_bytes + 2 * a_bytes + sum_bytes);
    float4* factors = reinterpret_cast<float4*>(ws + 3 * x_bytes + 2 * a_bytes + sum_bytes + exp_bytes);
    double* part = reinterpret_cast<double*>(ws + 3 * x_bytes + 2 * a_bytes + sum_bytes + exp_bytes + factor_bytes);
    float* S = reinterpret_cast<float*>(ws + 3 * x_bytes + 2 * a_bytes + sum_bytes + exp_bytes + factor_bytes + part_bytes);
    const T* G = static_cast<const T*>(p.G) + p.offG;

    const size_t tl = (p.len + 63) / 64, tiles = tl * ((p.lines + 63) / 64);
    if (tiles >= (1u << 31)) e = cudaErrorNotSupported;
    if (e == cudaSuccess) {
        const bool vec = aligned16(G) && p.ldg * sizeof(T) % 16 == 0 && (batch == 1 || p.strideG * sizeof(T) % 16 == 0);
        const dim3 g1((unsigned)parts, (unsigned)batch), g2((unsigned)tiles, (unsigned)batch);
        auto prepare = [&](auto is_vec, auto is_flip) {
            constexpr bool V = decltype(is_vec)::value, F = decltype(is_flip)::value;
            sum_squares_kernel<T, V><<<g1, 256, 0, s>>>(G, p.lines, (unsigned)p.len, p.ldg, p.strideG, part, sums, pitch);
            count_launch(2);
            return launch_chained(split_kernel<T, V, F>, g2, 256, s, G, p.lines, p.len, p.ldg, p.strideG, (const double*)part, (int)parts, hi[0], lo, ldx, xs, sums, exps, pitch, (unsigned)tl);
        };
        if (vec) e = flip ? prepare(std::true_type{}, std::true_type{}) : prepare(std::true_type{}, std::false_type{});
        else     e = flip ? prepare(std::false_type{}, std::true_type{}) : prepare(std::false_type{}, std::false_type{});
    }
    const char* plans[2] = {"", "none"};                   // of the last step's products
    for (int k = 0; k < p.steps && e == cudaSuccess; k++) {
        const float a = p.coeffs ? p.coeffs[3 * k] : 3.4445f, b = p.coeffs ? p.coeffs[3 * k + 1] : -4.7750f, c = p.coeffs ? p.coeffs[3 * k + 2] : 2.0315f;
        const Sizes sizes{sums + k, exps + k, factors + 2 * k, pitch, (float)n, a, b, c, k + 1 == p.steps, kappa_on_lo(n, p.coeffs, k, p.steps), p.alpha / SX};
        __half* x = hi[k & 1];
        const Operand ox{x, m, n, ldx, xs}, oa{A, n, n, ldn, as}, op{P, n, n, ldn, as};
        Shape sq = {};
        sq.U = sq.V = (unsigned)n; sq.batch = (unsigned)batch; sq.tri = 1;
        for (size_t at = 0; at < m && e == cudaSuccess; at += SEGMENT) {
            const size_t length = std::min(SEGMENT, m - at);
            const Operand part{x + at, length, n, ldx, xs};
            sq.K = (unsigned)length;
            if (m <= SEGMENT) e = run_planned<KIND_F16, false>(part, part, sq, EpiGram<false>{A, ldn, as, sizes, nullptr}, s);
            else if (at + length < m) e = run_planned<KIND_F16, false>(part, part, sq, EpiGramPart{S, ldn, as, at == 0}, s);
            else e = run_planned<KIND_F16, false>(part, part, sq, EpiGram<true>{A, ldn, as, sizes, S}, s);
        }
        plans[0] = last_plan();
        if (e == cudaSuccess && c != 0.f) {
            sq.K = (unsigned)n;
            e = run_planned<KIND_F16, false>(oa, oa, sq, EpiSquare{A, P, ldn, as, factors + 2 * k, pitch}, s);
            plans[1] = last_plan();
        }
        if (e != cudaSuccess) break;
        Shape up_ = {};
        up_.U = (unsigned)n; up_.V = (unsigned)m; up_.K = (unsigned)n; up_.batch = (unsigned)batch;
        const UpdateTerm t{x, lo, ldx, xs, factors + 2 * k, pitch};
        if (k + 1 < p.steps) {
            e = run_planned<KIND_F16, true>(c != 0.f ? op : oa, ox, up_, EpiUpdate{t, hi[(k + 1) & 1], lo, sums + k + 1}, s);
        } else {
            uint16_t* O = static_cast<uint16_t*>(p.O) + p.offO;
            const int align = line_alignment(O, p.ldo, batch > 1 ? p.strideO : 0);
            e = run_planned<KIND_F16, true>(c != 0.f ? op : oa, ox, up_, EpiOut{t, O, p.ldo, p.strideO, p.beta, flip, align}, s);
        }
    }
    if (e == cudaSuccess) {
        char name[96];
        std::snprintf(name, sizeof(name), "orthogonalize<%s,%s,%s>", plans[0], plans[1], last_plan());
        set_last_variant(name);
    }
    const cudaError_t e2 = ws_free(ws, s);
    return e == cudaSuccess ? e2 : e;
}

}  // namespace

cudaError_t orthogonalize(const OrthProblem& p, cudaStream_t s)
{
    // A grid has 65535 blocks along y, the matrices of a batch: larger batches in parts, which share a workspace in turn.
    constexpr size_t MOST = 32768;
    for (size_t i = 0; i < p.batch; i += MOST) {
        OrthProblem part = p;
        part.batch = std::min(MOST, p.batch - i);
        part.offG += i * p.strideG;
        part.offO += i * p.strideO;
        cudaError_t e;
        switch (p.type) {
            case clblasB200Float32: e = orthogonalize_typed<float>(part, s); break;
            case clblasB200Float16: e = orthogonalize_typed<__half>(part, s); break;
            default: e = orthogonalize_typed<__nv_bfloat16>(part, s);
        }
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

unsigned orthogonalize_fault_flag() { return read_wait_timeout_flag() | orthogonalize_small_fault_flag(); }

}  // namespace cb200
