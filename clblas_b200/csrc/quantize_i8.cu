// Symmetric 8-bit quantisation with one scale per row or column (the operands of the 8-bit product):
//   s = max|x| / 127,  q = rint(x * (127 / max|x|)),  x ~ s q.
// Every operation is one IEEE FP32 operation, so the result does not depend on the launch.  Lines whose largest magnitude is below
// 2^-100 (where 127 / max|x| would leave the range of FP32) count as zero: s = 0, q = 0.  A line that holds a NaN or an
// infinity gets s = NaN, q = 0: the product with it is NaN, as the product with the line itself would be.
//
// Bound by memory: each element is read once and one byte written.
#include "common.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace cb200 {

namespace {

constexpr float kSmallest = 7.888609052210118e-31f;       // 2^-100

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

// Magnitudes are compared as integers: for non-negative floats the order is the same, and an infinity or a NaN, whose
// pattern is larger than that of every finite number, wins.
__device__ __forceinline__ unsigned magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

struct LineScale { float s, inv; };
__device__ __forceinline__ LineScale line_scale(unsigned top)
{
    const float m = __uint_as_float(top);
    if (top >= 0x7f800000u) return {__uint_as_float(0x7fffffffu), 0.f};
    if (m < kSmallest) return {0.f, 0.f};
    return {__fdiv_rn(m, 127.f), __fdiv_rn(127.f, m)};
}
__device__ __forceinline__ signed char quant(float x, const LineScale& l)
{
    return l.inv == 0.f ? (signed char)0 : (signed char)__float2int_rn(__fmul_rn(x, l.inv));
}

// One line (contiguous elements, one scale) per CTA of THREADS threads; V elements per access.
template <typename T, int THREADS, int V>
__global__ void __launch_bounds__(THREADS) quantize_lines_kernel(const T* __restrict__ X, size_t ldx, signed char* __restrict__ Q, size_t ldq,
                                                                 float* __restrict__ scale, size_t len)
{
    constexpr int KEEP = 32 / V;                          // accesses a thread keeps in registers (32 elements)
    struct alignas(sizeof(T) * V) In { T t[V]; };
    struct alignas(V) Out { signed char q[V]; };
    __shared__ unsigned tops[THREADS / 32];
    const T* x = X + (size_t)blockIdx.x * ldx;
    signed char* q = Q + (size_t)blockIdx.x * ldq;
    const size_t pieces = len / V;
    In kept[KEEP];
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < KEEP; k++) {
        const size_t i = (size_t)k * THREADS + threadIdx.x;
        if (i < pieces) {
            kept[k] = *reinterpret_cast<const In*>(x + i * V);
        } else {
#pragma unroll
            for (int j = 0; j < V; j++) kept[k].t[j] = T(0.f);
        }
    }
#pragma unroll
    for (int k = 0; k < KEEP; k++)
#pragma unroll
        for (int j = 0; j < V; j++) top = max(top, magnitude(to_f(kept[k].t[j])));
    for (size_t i = (size_t)KEEP * THREADS + threadIdx.x; i < pieces; i += THREADS) {
        const In v = *reinterpret_cast<const In*>(x + i * V);
#pragma unroll
        for (int j = 0; j < V; j++) top = max(top, magnitude(to_f(v.t[j])));
    }
    for (size_t i = pieces * V + threadIdx.x; i < len; i += THREADS) top = max(top, magnitude(to_f(x[i])));
    top = __reduce_max_sync(0xffffffffu, top);
    if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, tops[threadIdx.x % (THREADS / 32)]);
    const LineScale l = line_scale(top);
    if (threadIdx.x == 0) scale[blockIdx.x] = l.s;
#pragma unroll
    for (int k = 0; k < KEEP; k++) {
        const size_t i = (size_t)k * THREADS + threadIdx.x;
        if (i >= pieces) continue;
        Out o;
#pragma unroll
        for (int j = 0; j < V; j++) o.q[j] = quant(to_f(kept[k].t[j]), l);
        *reinterpret_cast<Out*>(q + i * V) = o;
    }
    for (size_t i = (size_t)KEEP * THREADS + threadIdx.x; i < pieces; i += THREADS) {
        const In v = *reinterpret_cast<const In*>(x + i * V);
        Out o;
#pragma unroll
        for (int j = 0; j < V; j++) o.q[j] = quant(to_f(v.t[j]), l);
        *reinterpret_cast<Out*>(q + i * V) = o;
    }
    for (size_t i = pieces * V + threadIdx.x; i < len; i += THREADS) q[i] = quant(to_f(x[i]), l);
}

// One scale per position of the lines: the maximum runs across the lines.  First pass: every CTA takes the maximum of
// its lines for 256 positions and joins it to the others' (integer maximum: the order does not matter).
constexpr int ACROSS_LINES = 64;
template <typename T>
__global__ void __launch_bounds__(256) across_max_kernel(const T* __restrict__ X, size_t ldx, unsigned* __restrict__ top, size_t lines, size_t len)
{
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= len) return;
    const size_t l0 = (size_t)blockIdx.y * ACROSS_LINES, l1 = min(lines, l0 + ACROSS_LINES);
    unsigned m = 0;
#pragma unroll 8
    for (size_t l = l0; l < l1; l++) m = max(m, magnitude(to_f(X[l * ldx + i])));
    atomicMax(top + i, m);
}

template <typename T>
__global__ void __launch_bounds__(256) across_quantize_kernel(const T* __restrict__ X, size_t ldx, signed char* __restrict__ Q, size_t ldq,
                                                              const unsigned* __restrict__ top, float* __restrict__ scale, size_t lines, size_t len)
{
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= len) return;
    const LineScale s = line_scale(top[i]);
    if (blockIdx.y == 0) scale[i] = s.s;
    const size_t l0 = (size_t)blockIdx.y * ACROSS_LINES, l1 = min(lines, l0 + ACROSS_LINES);
#pragma unroll 8
    for (size_t l = l0; l < l1; l++) Q[l * ldq + i] = quant(to_f(X[l * ldx + i]), s);
}

template <typename T>
cudaError_t quantize_typed(bool per_line, const T* X, size_t ldx, signed char* Q, size_t ldq, float* scale, size_t lines, size_t len, cudaStream_t s)
{
    if (per_line) {
        if (lines >= (1u << 31)) return cudaErrorNotSupported;
        constexpr int V = 16 / sizeof(T);
        const unsigned grid = (unsigned)lines;
        if (aligned16(X) && (ldx * sizeof(T)) % 16 == 0 && (reinterpret_cast<uintptr_t>(Q) | ldq) % V == 0)
            quantize_lines_kernel<T, 256, V><<<grid, 256, 0, s>>>(X, ldx, Q, ldq, scale, len);
        else
            quantize_lines_kernel<T, 256, 1><<<grid, 256, 0, s>>>(X, ldx, Q, ldq, scale, len);
        count_launch();
        return cudaGetLastError();
    }
    const size_t rows = (lines + ACROSS_LINES - 1) / ACROSS_LINES;
    if (len >= (1u << 31) || rows > 65535) return cudaErrorNotSupported;
    unsigned* top = nullptr;
    cudaError_t e = ws_alloc(reinterpret_cast<void**>(&top), len * sizeof(unsigned), s);
    if (e != cudaSuccess) return e;
    e = cudaMemsetAsync(top, 0, len * sizeof(unsigned), s);
    if (e == cudaSuccess) {
        const dim3 grid((unsigned)((len + 255) / 256), (unsigned)rows);
        across_max_kernel<T><<<grid, 256, 0, s>>>(X, ldx, top, lines, len);
        across_quantize_kernel<T><<<grid, 256, 0, s>>>(X, ldx, Q, ldq, top, scale, lines, len);
        count_launch(2);
        e = cudaGetLastError();
    }
    const cudaError_t e2 = ws_free(top, s);
    return e == cudaSuccess ? e2 : e;
}

}  // namespace

cudaError_t quantize_i8(int type, bool per_line, const void* X, size_t offX, size_t ldx, signed char* Q, size_t ldq, float* scale, size_t lines,
                        size_t len, cudaStream_t s)
{
    switch (type) {
        case clblasB200Float32: return quantize_typed(per_line, static_cast<const float*>(X) + offX, ldx, Q, ldq, scale, lines, len, s);
        case clblasB200Float16: return quantize_typed(per_line, static_cast<const __half*>(X) + offX, ldx, Q, ldq, scale, lines, len, s);
        default: return quantize_typed(per_line, static_cast<const __nv_bfloat16*>(X) + offX, ldx, Q, ldq, scale, lines, len, s);
    }
}

}  // namespace cb200
