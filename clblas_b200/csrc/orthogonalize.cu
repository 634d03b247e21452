// Orthogonalisation of an update by Newton-Schulz products: with X0 = G / (|G|_F + 1e-7), k steps of
//     X <- a X + (b X X' + c (X X')^2) X
// push every singular value of G towards one and keep its singular vectors; O <- alpha X + beta O.  (No counterpart in the
// reference; the products are of its SYRK and SYMM families.  Optimisers that orthogonalise the momentum of a weight use it.)
//
// On the smaller side n of the matrix (n <= m) a step is three products: the Gram matrix (symmetric, n^2 m operations), its
// square (symmetric, n^3) and the update (2 n^2 m).  All run on the FP16 tensor-core tiles of narrow_mma.cuh, the symmetric ones on
// the tiles of one triangle, each result stored at both places.
//
// What is kept in how many bits, and why:
//   * X is a pair of FP16 numbers, hi + lo (22 bits); a X uses the pair, the products use hi.  Singular values far below the
//     others grow by a factor of about a in every step; a rounding of X itself would put noise on them that grows as
//     fast (rank-8 gradient, five steps: 4 % of the result with X in FP16 alone, 34 % in BF16).  A rounding inside the products
//     meets X once more and does not grow.
//   * The Gram matrix is stored as A = X X' - t I, t its mean diagonal, and P = (b + 2 c t) A + c A^2; X <- (a + b t + c t^2) X + P X is the
//     same polynomial.  Near the end X X' is close to I and b, c nearly cancel: rounding the small difference instead
//     halves the error of the result (normal 768 x 768: 1.5e-3 without, 7e-4 with t; the final rounding to BF16 is 1.7e-3).
//   * t comes from the sum of the squares of X, gathered in 64-bit integers (units of 2^-24), so the order of the atomic additions does
//     not change it.  Any t gives the same polynomial; it only has to be near.
//   * Accumulators and everything between accumulator and store are FP32.  X is held times 2^12, A and P times 2^8, so that the
//     entries of large matrices (about 1/sqrt(m)) stay far above FP16's smallest numbers.
// The result is good to about 1e-3 and is therefore given in BF16 only.
#include "narrow_mma.cuh"

namespace cb200 {

namespace {

using namespace narrow;

constexpr float SX = 4096.f, SA = 256.f;                  // scales of the stored X and of the stored A, P
constexpr double SUM_UNIT = 16777216.0;                    // sums of squares are counted in 2^-24
constexpr double EPS = 1e-7;
constexpr int SUM_BLOCKS = 296;

typedef unsigned long long u64;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

struct alignas(16) Half8 { __half2 h[4]; };
__device__ __forceinline__ void load8(const __half* p, float (&x)[8])
{
    const Half8 v = *reinterpret_cast<const Half8*>(p);
#pragma unroll
    for (int i = 0; i < 4; i++) { const float2 f = __half22float2(v.h[i]); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
}
__device__ __forceinline__ void store8(__half* p, const float (&x)[8])
{
    Half8 v;
#pragma unroll
    for (int i = 0; i < 4; i++) v.h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<Half8*>(p) = v;
}

// ---- norm and split ---------------------------------------------------------------------------------------------------

// Sum of squares of one matrix of the batch, in 64 bits: block b takes lines b, b + blocks, ...
template <typename T>
__global__ void __launch_bounds__(256) sum_squares_kernel(const T* __restrict__ G, size_t lines, size_t len, size_t ld, size_t stride, double* __restrict__ part)
{
    const T* g = G + blockIdx.y * stride;
    double sum = 0;
    for (size_t l = (size_t)blockIdx.x * 8 + threadIdx.x / 32; l < lines; l += (size_t)gridDim.x * 8) {
        const T* x = g + l * ld;
#pragma unroll 4
        for (size_t i = threadIdx.x % 32; i < len; i += 32) {
            const double v = to_f(x[i]);
            sum = fma(v, v, sum);
        }
    }
    __shared__ double sums[8];
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (threadIdx.x % 32 == 0) sums[threadIdx.x / 32] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; w++) sum += sums[w];
        part[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = sum;
    }
}

// X0 = G / (|G| + eps), times SX, as hi + lo; FLIP: transposed on the way (G has more lines than elements per line).
// A matrix that holds a NaN or an infinity becomes NaN everywhere.  64 x 64 elements per CTA.
template <typename T, bool FLIP>
__global__ void __launch_bounds__(256) split_kernel(const T* __restrict__ G, size_t lines, size_t len, size_t ld, size_t stride, const double* __restrict__ part,
                                                    int parts, __half* __restrict__ hi, __half* __restrict__ lo, size_t ldx, size_t stride_x,
                                                    u64* __restrict__ sums, int sums_pitch, unsigned tiles_len)
{
    __shared__ double factor;
    __shared__ float tile[FLIP ? 64 : 1][65];
    const unsigned z = blockIdx.y;
    if (threadIdx.x < 32) {
        double sum = 0;
        for (int i = threadIdx.x; i < parts; i += 32) sum += part[(size_t)z * parts + i];
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (threadIdx.x == 0) {
            const double norm = sqrt(sum), f = 1.0 / (norm + EPS);
            factor = isfinite(norm) ? f * SX : nan("");
            if (blockIdx.x == 0) sums[(size_t)z * sums_pitch] = isfinite(norm) ? (u64)(norm * f * norm * f * SUM_UNIT) : 0;
        }
    }
    __syncthreads();
    const double f = factor;
    const size_t l0 = (size_t)(blockIdx.x / tiles_len) * 64, i0 = (size_t)(blockIdx.x % tiles_len) * 64;
    const T* g = G + z * stride;
    __half* h = hi + z * stride_x;
    __half* w = lo + z * stride_x;
    if (!FLIP) {
        for (int k = threadIdx.x / 32; k < 64; k += 8) {
            const size_t l = l0 + k, i = i0 + 2 * (threadIdx.x % 32);      // pairs: the pitch of X is even
            if (l >= lines || i >= len) continue;
            const float a = (float)(to_f(g[l * ld + i]) * f), b = i + 1 < len ? (float)(to_f(g[l * ld + i + 1]) * f) : 0.f;
            const __half2 t = __floats2half2_rn(a, b);
            const float2 r = __half22float2(t);
            *reinterpret_cast<__half2*>(h + l * ldx + i) = t;
            *reinterpret_cast<__half2*>(w + l * ldx + i) = __floats2half2_rn(a - r.x, b - r.y);
        }
    } else {
        for (int k = threadIdx.x / 32; k < 64; k += 8)
            for (int j = threadIdx.x % 32; j < 64; j += 32) {
                const size_t l = l0 + k, i = i0 + j;
                tile[k][j] = l < lines && i < len ? (float)(to_f(g[l * ld + i]) * f) : 0.f;
            }
        __syncthreads();
        for (int j = threadIdx.x / 32; j < 64; j += 8) {
            const int k = 2 * (threadIdx.x % 32);
            const size_t l = l0 + k, i = i0 + j;
            if (l >= lines || i >= len) continue;
            const float a = tile[k][j], b = tile[k + 1][j];
            const __half2 t = __floats2half2_rn(a, b);
            const float2 r = __half22float2(t);
            *reinterpret_cast<__half2*>(h + i * ldx + l) = t;
            *reinterpret_cast<__half2*>(w + i * ldx + l) = __floats2half2_rn(a - r.x, b - r.y);
        }
    }
}

// ---- epilogues ----------------------------------------------------------------------------------------------------------
// Segments are eight aligned columns here (slices of at least 8 columns, workspaces with a pitch of a multiple of 8): pieces of the
// workspaces are read and written whole, what lies beyond V is padding that no product reads.

// The shift t: the mean diagonal of X X', once most singular values have come near one; 0 before (and for a matrix of NaN, whose
// sum says nothing).  While X is dominated by a few directions the shift would put roundings of t on all the others
// (rank 8 of 100: 3e-3 with t from the first step on, 7e-4 from t = 0.2 on).
__device__ __forceinline__ float shift_of(const u64* sums, size_t at, float inv_n)
{
    const float t = (float)((double)sums[at] * (1.0 / SUM_UNIT)) * inv_n;
    return t >= 0.2f ? t : 0.f;
}

struct EpiGram {                                           // A <- X X' - t I
    static constexpr bool kMirror = true;
    struct State { float t; };
    __half* A; size_t ld, stride;
    const u64* sums; int pitch;
    float inv_n;
    __device__ bool transposed() const { return false; }
    __device__ float begin(State& st, unsigned z, unsigned) const
    {
        st.t = SA * shift_of(sums, (size_t)z * pitch, inv_n);
        return SA / (SX * SX);
    }
    template <int CH> __device__ void combine(State&, unsigned, unsigned, unsigned, unsigned, float (&)[CH]) const {}
    __device__ void column(State&, unsigned z, unsigned u, unsigned v, float x) const { A[z * stride + (size_t)v * ld + u] = __float2half_rn(x); }
    __device__ void segment(State& st, unsigned z, unsigned u, unsigned v, unsigned n, float (&x)[8]) const
    {
#pragma unroll
        for (int i = 0; i < 8; i++) if (u == v + i) x[i] -= st.t;
        store8(A + z * stride + (size_t)u * ld + v, x);
    }
    __device__ void end(State&, unsigned, unsigned) const {}
};

struct EpiSquare {                                         // P <- (b + 2 c t) A + c A^2
    static constexpr bool kMirror = true;
    struct State { float b; };
    const __half* A; __half* P; size_t ld, stride;
    const u64* sums; int pitch;
    float inv_n, b, c;
    __device__ bool transposed() const { return false; }
    __device__ float begin(State& st, unsigned z, unsigned) const
    {
        st.b = b + 2.f * c * shift_of(sums, (size_t)z * pitch, inv_n);
        return c / SA;
    }
    template <int CH> __device__ void combine(State&, unsigned, unsigned, unsigned, unsigned, float (&)[CH]) const {}
    __device__ void column(State& st, unsigned z, unsigned u, unsigned v, float x) const
    {
        const size_t at = z * stride + (size_t)v * ld + u;
        P[at] = __float2half_rn(fmaf(st.b, __half2float(A[at]), x));
    }
    __device__ void segment(State& st, unsigned z, unsigned u, unsigned v, unsigned n, float (&x)[8]) const
    {
        const size_t at = z * stride + (size_t)u * ld + v;
        float a[8];
        load8(A + at, a);
#pragma unroll
        for (int i = 0; i < 8; i++) a[i] = fmaf(st.b, a[i], x[i]);
        store8(P + at, a);
    }
    __device__ void end(State&, unsigned, unsigned) const {}
};

// Common part of the two updates: y = (a + b t + c t^2) X + P X, times SX.  P is P, or A with factor b when c == 0.
struct UpdateTerm {
    const __half* hi; const __half* lo; size_t ldx, stride_x;
    const u64* sums; int pitch;
    float inv_n, a, b, c;
    __device__ float coefficient(unsigned z) const
    {
        const float t = shift_of(sums, (size_t)z * pitch, inv_n);
        return a + t * (b + c * t);
    }
    __device__ float factor() const { return (c == 0.f ? b : 1.f) / SA; }
};

struct EpiUpdate {
    static constexpr bool kMirror = false;
    struct State { float a, sum; };
    UpdateTerm t;
    __half* hi; __half* lo;                                // lo may be the one that is read: each place is read and written by one thread
    u64* next;                                             // sums of the new X
    __device__ bool transposed() const { return false; }
    __device__ float begin(State& st, unsigned z, unsigned) const
    {
        st.a = t.coefficient(z);
        st.sum = 0.f;
        return t.factor();
    }
    template <int CH> __device__ void combine(State&, unsigned, unsigned, unsigned, unsigned, float (&)[CH]) const {}
    __device__ void column(State&, unsigned, unsigned, unsigned, float) const {}
    __device__ void segment(State& st, unsigned z, unsigned u, unsigned v, unsigned n, float (&x)[8]) const
    {
        const size_t at = z * t.stride_x + (size_t)u * t.ldx + v;
        float h[8], l[8];
        load8(t.hi + at, h);
        load8(t.lo + at, l);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x[i] = fmaf(st.a, h[i] + l[i], x[i]);
            h[i] = __half2float(__float2half_rn(x[i]));
            l[i] = x[i] - h[i];
            if (i < (int)n) st.sum = fmaf(x[i], x[i], st.sum);
        }
        store8(hi + at, h);
        store8(lo + at, l);
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
    static constexpr bool kMirror = false;
    struct State { float a; };
    UpdateTerm t;
    __nv_bfloat16* O; size_t ldo, stride_o;
    float alpha, beta;
    bool flip, vec;                                        // flip: element (u, v) at O[v * ldo + u]
    __device__ bool transposed() const { return flip; }
    __device__ float begin(State& st, unsigned z, unsigned) const
    {
        st.a = t.coefficient(z) * (alpha / SX);
        return t.factor() * (alpha / SX);
    }
    template <int CH>
    __device__ void combine(State& st, unsigned z, unsigned u, unsigned v0, unsigned V, float (&x)[CH]) const
    {
        const size_t at = z * t.stride_x + (size_t)u * t.ldx + v0;
#pragma unroll
        for (int j = 0; j < CH; j += 8) {
            if (v0 + j >= V) break;
            float h[8], l[8];
            load8(t.hi + at + j, h);
            load8(t.lo + at + j, l);
#pragma unroll
            for (int i = 0; i < 8; i++) x[j + i] = fmaf(st.a, h[i] + l[i], x[j + i]);
        }
    }
    __device__ void column(State&, unsigned z, unsigned u, unsigned v, float x) const
    {
        __nv_bfloat16* o = O + z * stride_o + (size_t)v * ldo + u;
        if (beta != 0.f) x = fmaf(beta, __bfloat162float(*o), x);
        *o = __float2bfloat16_rn(x);
    }
    __device__ void segment(State& st, unsigned z, unsigned u, unsigned v, unsigned n, float (&x)[8]) const
    {
        const size_t at = z * t.stride_x + (size_t)u * t.ldx + v;
        __nv_bfloat16* o = O + z * stride_o + (size_t)u * ldo + v;
        float h[8], l[8];
        load8(t.hi + at, h);
        load8(t.lo + at, l);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = fmaf(st.a, h[i] + l[i], x[i]);
        if (vec && n == 8) {
            uint4 raw;
            __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&raw);
            if (beta != 0.f) {
                raw = *reinterpret_cast<const uint4*>(o);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float2 f = __bfloat1622float2(p[i]);
                    x[2 * i] = fmaf(beta, f.x, x[2 * i]);
                    x[2 * i + 1] = fmaf(beta, f.y, x[2 * i + 1]);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) p[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            *reinterpret_cast<uint4*>(o) = raw;
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (i >= (int)n) break;
            float y = x[i];
            if (beta != 0.f) y = fmaf(beta, __bfloat162float(o[i]), y);
            o[i] = __float2bfloat16_rn(y);
        }
    }
    __device__ void end(State&, unsigned, unsigned) const {}
};

// ---- the chain ----------------------------------------------------------------------------------------------------------

template <typename T>
cudaError_t orthogonalize_typed(const OrthProblem& p, cudaStream_t s)
{
    const bool flip = p.lines > p.len;
    const size_t n = flip ? p.len : p.lines, m = flip ? p.lines : p.len, batch = p.batch;
    if (m >= (1u << 31) || batch >= 65536) return cudaErrorNotSupported;
    auto up = [](size_t v, size_t q) { return (v + q - 1) / q * q; };
    const size_t ldx = up(m, 8), ldn = up(n, 8), xs = n * ldx, as = n * ldn;
    const int pitch = p.steps + 1;
    const size_t lines_blocks = (p.lines + 7) / 8, parts = lines_blocks < SUM_BLOCKS ? lines_blocks : SUM_BLOCKS;
    // workspace: hi (two of them, read and written in turn), lo, A, P, sums of squares, partial norms
    const size_t x_bytes = up(batch * xs * 2, 256), a_bytes = up(batch * as * 2, 256), sum_bytes = up(batch * pitch * 8, 256);
    unsigned char* ws = nullptr;
    cudaError_t e = ws_alloc(reinterpret_cast<void**>(&ws), 3 * x_bytes + 2 * a_bytes + sum_bytes + batch * parts * 8, s);
    if (e != cudaSuccess) return e;
    __half* hi[2] = {reinterpret_cast<__half*>(ws), reinterpret_cast<__half*>(ws + x_bytes)};
    __half* lo = reinterpret_cast<__half*>(ws + 2 * x_bytes);
    __half* A = reinterpret_cast<__half*>(ws + 3 * x_bytes);
    __half* P = reinterpret_cast<__half*>(ws + 3 * x_bytes + a_bytes);
    u64* sums = reinterpret_cast<u64*>(ws + 3 * x_bytes + 2 * a_bytes);
    double* part = reinterpret_cast<double*>(ws + 3 * x_bytes + 2 * a_bytes + sum_bytes);
    const T* G = static_cast<const T*>(p.G) + p.offG;

    e = cudaMemsetAsync(sums, 0, batch * pitch * 8, s);
    if (e == cudaSuccess) {
        sum_squares_kernel<T><<<dim3((unsigned)parts, (unsigned)batch), 256, 0, s>>>(G, p.lines, p.len, p.ldg, p.strideG, part);
        const size_t tl = (p.len + 63) / 64, tiles = tl * ((p.lines + 63) / 64);
        if (tiles >= (1u << 31)) e = cudaErrorNotSupported;
        else if (flip)
            split_kernel<T, true><<<dim3((unsigned)tiles, (unsigned)batch), 256, 0, s>>>(G, p.lines, p.len, p.ldg, p.strideG, part, (int)parts, hi[0], lo, ldx, xs, sums, pitch, (unsigned)tl);
        else
            split_kernel<T, false><<<dim3((unsigned)tiles, (unsigned)batch), 256, 0, s>>>(G, p.lines, p.len, p.ldg, p.strideG, part, (int)parts, hi[0], lo, ldx, xs, sums, pitch, (unsigned)tl);
        count_launch(2);
        if (e == cudaSuccess) e = cudaGetLastError();
    }
    const float inv_n = 1.f / (float)n;
    for (int k = 0; k < p.steps && e == cudaSuccess; k++) {
        const float a = p.coeffs ? p.coeffs[3 * k] : 3.4445f, b = p.coeffs ? p.coeffs[3 * k + 1] : -4.7750f, c = p.coeffs ? p.coeffs[3 * k + 2] : 2.0315f;
        __half* x = hi[k & 1];
        const Operand ox{x, m, n, ldx, xs}, oa{A, n, n, ldn, as}, op{P, n, n, ldn, as};
        Shape sq = {};
        sq.U = sq.V = (unsigned)n; sq.K = (unsigned)m; sq.batch = (unsigned)batch; sq.tri = 1;
        e = run_planned<KIND_F16, false>(ox, ox, sq, EpiGram{A, ldn, as, sums + k, pitch, inv_n}, s);
        if (e == cudaSuccess && c != 0.f) {
            sq.K = (unsigned)n;
            e = run_planned<KIND_F16, false>(oa, oa, sq, EpiSquare{A, P, ldn, as, sums + k, pitch, inv_n, b, c}, s);
        }
        if (e != cudaSuccess) break;
        Shape up_ = {};
        up_.U = (unsigned)n; up_.V = (unsigned)m; up_.K = (unsigned)n; up_.batch = (unsigned)batch;
        const UpdateTerm t{x, lo, ldx, xs, sums + k, pitch, inv_n, a, b, c};
        if (k + 1 < p.steps) {
            e = run_planned<KIND_F16, true>(c != 0.f ? op : oa, ox, up_, EpiUpdate{t, hi[(k + 1) & 1], lo, sums + k + 1}, s);
        } else {
            __nv_bfloat16* O = static_cast<__nv_bfloat16*>(p.O) + p.offO;
            const bool vec = aligned16(O) && p.ldo % 8 == 0 && (batch == 1 || p.strideO % 8 == 0);
            e = run_planned<KIND_F16, true>(c != 0.f ? op : oa, ox, up_, EpiOut{t, O, p.ldo, p.strideO, p.alpha, p.beta, flip, vec}, s);
        }
    }
    const cudaError_t e2 = ws_free(ws, s);
    return e == cudaSuccess ? e2 : e;
}

}  // namespace

cudaError_t orthogonalize(const OrthProblem& p, cudaStream_t s)
{
    set_last_kernel("orthogonalize_tcgen05");
    switch (p.type) {
        case clblasB200Float32: return orthogonalize_typed<float>(p, s);
        case clblasB200Float16: return orthogonalize_typed<__half>(p, s);
        default: return orthogonalize_typed<__nv_bfloat16>(p, s);
    }
}

unsigned orthogonalize_fault_flag() { return read_wait_timeout_flag(); }

}  // namespace cb200
