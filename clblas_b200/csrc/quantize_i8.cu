// Symmetric 8-bit quantisation with one scale per row or column (the operands of the 8-bit product):
//   s = max|x| / 127,  q = rint(x * (127 / max|x|)),  x ~ s q.
// Every operation is one IEEE FP32 operation, so the result does not depend on the launch.  Lines whose largest magnitude is below
// 2^-100 count as zero: s = 0, q = 0.  (127 / max|x| stays finite down to 2^-121; the limit is part of the operator's definition,
// chosen with room to that.)  A line that holds a NaN or an
// infinity gets s = NaN, q = 0: the product with it is NaN, as the product with the line itself would be.
//
// Bound by memory: each element is read once and one byte written.
//
// The kernels start while the one before them, which may write X, still runs.  X is therefore no `const __restrict__` pointer: that
// would allow loads through the cache for constants, which may be taken ahead of the wait.
#include "common.h"
#include "tma_pipeline.cuh"

#include <algorithm>

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
// V values, packed.  rint by adding 3 * 2^22, which leaves the integer (two's complement) in the low mantissa bits: a quarter-rate
// conversion for every element would take half as long as the memory traffic.
template <int V> struct Bytes;
template <> struct Bytes<1> { typedef unsigned char Type; };
template <> struct Bytes<4> { typedef uint32_t Type; };
template <> struct Bytes<8> { typedef uint2 Type; };
__device__ __forceinline__ uint32_t quant_bits(float x, const LineScale& l) { return __float_as_uint(__fadd_rn(__fmul_rn(x, l.inv), 12582912.f)); }
__device__ __forceinline__ uint32_t quant4(const float* x, const LineScale& l)
{
    const uint32_t a = __byte_perm(quant_bits(x[0], l), quant_bits(x[1], l), 0x0040), b = __byte_perm(quant_bits(x[2], l), quant_bits(x[3], l), 0x0040);
    return l.inv == 0.f ? 0u : __byte_perm(a, b, 0x5410);
}
__device__ __forceinline__ unsigned char quantize(const float (&x)[1], const LineScale& l) { return l.inv == 0.f ? 0 : (unsigned char)quant_bits(x[0], l); }
__device__ __forceinline__ uint32_t quantize(const float (&x)[4], const LineScale& l) { return quant4(x, l); }
__device__ __forceinline__ uint2 quantize(const float (&x)[8], const LineScale& l) { return make_uint2(quant4(x, l), quant4(x + 4, l)); }

template <typename T, int V> struct alignas(sizeof(T) * V) Word { T t[V]; };
template <typename T, int V>
__device__ __forceinline__ unsigned magnitude(const Word<T, V>& w, unsigned top)
{
#pragma unroll
    for (int j = 0; j < V; j++) top = max(top, magnitude(to_f(w.t[j])));
    return top;
}
template <typename T, int V>
__device__ __forceinline__ void put(signed char* q, const Word<T, V>& w, const LineScale& l)
{
    float x[V];
#pragma unroll
    for (int j = 0; j < V; j++) x[j] = to_f(w.t[j]);
    *reinterpret_cast<typename Bytes<V>::Type*>(q) = quantize(x, l);
}

// One line (contiguous elements, one scale) per CTA of THREADS threads; V elements per access.  A thread keeps its first KEEP
// accesses in registers between the maximum and the quantisation; longer lines are read again from there on.
template <typename T, int THREADS, int V, int KEEP>
__global__ void __launch_bounds__(THREADS) quantize_lines_kernel(const T* X, size_t ldx, signed char* __restrict__ Q, size_t ldq,
                                                                 float* __restrict__ scale, size_t len)
{
    typedef Word<T, V> W;
    __shared__ unsigned tops[THREADS / 32];
    const T* x = X + (size_t)blockIdx.x * ldx;
    signed char* q = Q + (size_t)blockIdx.x * ldq;
    const size_t pieces = len / V;
    pdl_launch_dependents();
    pdl_wait();
    W kept[KEEP];
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < KEEP; k++) {
        const size_t i = (size_t)k * THREADS + threadIdx.x;
        if (i < pieces) kept[k] = *reinterpret_cast<const W*>(x + i * V);
    }
#pragma unroll
    for (int k = 0; k < KEEP; k++)
        if ((size_t)k * THREADS + threadIdx.x < pieces) top = magnitude(kept[k], top);
    for (size_t i = (size_t)KEEP * THREADS + threadIdx.x; i < pieces; i += THREADS) top = magnitude(*reinterpret_cast<const W*>(x + i * V), top);
    if (V > 1)
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
        if (i < pieces) put<T, V>(q + i * V, kept[k], l);
    }
    for (size_t i = (size_t)KEEP * THREADS + threadIdx.x; i < pieces; i += THREADS) put<T, V>(q + i * V, *reinterpret_cast<const W*>(x + i * V), l);
    if (V > 1)
        for (size_t i = pieces * V + threadIdx.x; i < len; i += THREADS) {
            const Word<T, 1> w = {x[i]};
            put<T, 1>(q + i, w, l);
        }
}

// One scale per position of the lines: the maximum runs across the lines.
//
// Up to 5120 lines, unless the matrix is large and aligned: a cluster takes a strip of 32 positions, its CTAs share the lines, a warp a line at a time.  Each
// thread keeps its elements in registers, the maxima meet in distributed shared memory and every CTA quantises its own lines:
// one launch, each element read once.  KEEP elements a thread: 64, or the 80 that two CTAs per SM have room for when that saves a pass.
template <typename T, int KEEP>
__global__ void __launch_bounds__(256) quantize_across_kernel(const T* X, size_t ldx, signed char* __restrict__ Q, size_t ldq,
                                                              float* __restrict__ scale, size_t lines, size_t len)
{
    __shared__ unsigned tops[8][32], joined[32];
    uint32_t rank, ranks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const size_t i = (size_t)(blockIdx.x / ranks) * 32 + lane;
    const bool in = i < len;
    const size_t l0 = lines * rank / ranks, n = lines * (rank + 1) / ranks - l0;
    pdl_launch_dependents();
    pdl_wait();
    // This lane's lines: l0 + warp, + 8, ...  Addresses are stepped and the count is 32-bit: the kernel is bound by instructions as
    // much as by memory (55 of them per access took 30 us where 22 took 20).
    const int mine = in && n > (size_t)warp ? (int)((n - warp + 7) / 8) : 0;        // at most KEEP
    const size_t step = 8 * ldx, qstep = 8 * ldq;
    const T* x = X + (l0 + warp) * ldx + i;
    signed char* q = Q + (l0 + warp) * ldq + i;
    T kept[KEEP];
#pragma unroll
    for (int k = 0; k < KEEP; k++, x += step)
        if (k < mine) kept[k] = *x;
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < KEEP; k++)
        if (k < mine) top = max(top, magnitude(to_f(kept[k])));
    tops[warp][lane] = top;
    __syncthreads();
    if (warp == 0) {
#pragma unroll
        for (int w = 1; w < 8; w++) top = max(top, tops[w][lane]);
        joined[lane] = top;
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    unsigned m = 0;
    const uint32_t here = static_cast<uint32_t>(__cvta_generic_to_shared(&joined[lane]));
    for (uint32_t r = 0; r < ranks; r++) {
        uint32_t there, v;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(r));
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(there) : "memory");
        m = max(m, v);
    }
    const LineScale s = line_scale(m);
    if (rank == 0 && warp == 0 && in) scale[i] = s.s;
    // A CTA's maxima stay where they are until every other CTA has read them.
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    const uint32_t mask = s.inv == 0.f ? 0u : 0xffu;
#pragma unroll
    for (int k = 0; k < KEEP; k++, q += qstep)
        if (k < mine) *q = (signed char)(quant_bits(to_f(kept[k]), s) & mask);
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Everything larger: two passes, the second one mostly from L2.  A CTA takes COLS V positions and a block of lines, a warp 32 / COLS
// lines at a time, AHEAD accesses in flight.  First the maxima of every block, then the maximum over the blocks and the quantisation.
template <typename T, int V, int COLS>
struct AcrossBlock {
    typedef Word<T, V> W;
    static constexpr int RPW = 32 / COLS, AHEAD = V == 1 ? 16 : 8;
    size_t i, l0;
    int mine;                                                  // this lane's lines: l0, + 8 RPW, ...
    __device__ AcrossBlock(size_t lines, size_t len, unsigned blocks)
    {
        const int lane = threadIdx.x % 32, line = (int)(threadIdx.x / 32) * RPW + lane / COLS;
        i = ((size_t)blockIdx.x * COLS + lane % COLS) * V;
        const size_t first = lines * blockIdx.y / blocks, n = lines * (blockIdx.y + 1) / blocks - first;
        l0 = first + line;
        mine = i < len && n > (size_t)line ? (int)((n - line + 8 * RPW - 1) / (8 * RPW)) : 0;
    }
};

template <typename T, int V, int COLS>
__global__ void __launch_bounds__(256) across_max_kernel(const T* X, size_t ldx, unsigned* __restrict__ tops, size_t lines, size_t len)
{
    typedef AcrossBlock<T, V, COLS> B;
    __shared__ unsigned per_warp[8][COLS * V];
    pdl_launch_dependents();
    pdl_wait();
    const B b(lines, len, gridDim.y);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const T* x = X + b.l0 * ldx + b.i;
    const size_t step = 8 * B::RPW * ldx;
    unsigned top[V] = {};
    for (int k = 0; k < b.mine; k += B::AHEAD) {
        typename B::W v[B::AHEAD];
#pragma unroll
        for (int j = 0; j < B::AHEAD; j++, x += step)
            if (k + j < b.mine) v[j] = *reinterpret_cast<const typename B::W*>(x);
#pragma unroll
        for (int j = 0; j < B::AHEAD; j++)
            if (k + j < b.mine) {
#pragma unroll
                for (int e = 0; e < V; e++) top[e] = max(top[e], magnitude(to_f(v[j].t[e])));
            }
    }
#pragma unroll
    for (int e = 0; e < V; e++) {
#pragma unroll
        for (int d = 16; d >= COLS; d >>= 1) top[e] = max(top[e], __shfl_xor_sync(0xffffffffu, top[e], d));
        if (lane < COLS) per_warp[warp][lane * V + e] = top[e];
    }
    __syncthreads();
    for (int j = threadIdx.x; j < COLS * V; j += 256) {
        const size_t at = (size_t)blockIdx.x * COLS * V + j;
        unsigned m = per_warp[0][j];
#pragma unroll
        for (int w = 1; w < 8; w++) m = max(m, per_warp[w][j]);
        if (at < len) tops[(size_t)blockIdx.y * len + at] = m;
    }
}

template <typename T, int V, int COLS>
__global__ void __launch_bounds__(256) across_quantize_kernel(const T* X, size_t ldx, signed char* __restrict__ Q, size_t ldq,
                                                              const unsigned* tops, float* __restrict__ scale, size_t lines, size_t len)
{
    typedef AcrossBlock<T, V, COLS> B;
    __shared__ unsigned joined[COLS * V];
    pdl_launch_dependents();
    pdl_wait();
    const B b(lines, len, gridDim.y);
    for (int j = threadIdx.x; j < COLS * V; j += 256) {
        const size_t at = (size_t)blockIdx.x * COLS * V + j;
        unsigned m = 0;
        if (at < len) {
#pragma unroll 8
            for (unsigned y = 0; y < gridDim.y; y++) m = max(m, __ldcg(tops + (size_t)y * len + at));
            if (blockIdx.y == 0) scale[at] = line_scale(m).s;
        }
        joined[j] = m;
    }
    __syncthreads();
    LineScale s[V];
    uint32_t mask[(V + 3) / 4] = {};                           // bytes of the positions that are not all zero
#pragma unroll
    for (int e = 0; e < V; e++) {
        s[e] = line_scale(joined[(threadIdx.x % COLS) * V + e]);
        mask[e / 4] |= s[e].inv == 0.f ? 0u : 0xffu << (8 * (e % 4));
    }
    const T* x = X + b.l0 * ldx + b.i;
    signed char* q = Q + b.l0 * ldq + b.i;
    const size_t step = 8 * B::RPW * ldx, qstep = 8 * B::RPW * ldq;
    for (int k = 0; k < b.mine; k += B::AHEAD) {
        typename B::W v[B::AHEAD];
#pragma unroll
        for (int j = 0; j < B::AHEAD; j++, x += step)
            if (k + j < b.mine) v[j] = *reinterpret_cast<const typename B::W*>(x);
#pragma unroll
        for (int j = 0; j < B::AHEAD; j++, q += qstep) {
            if (k + j >= b.mine) continue;
            uint32_t r[V];
#pragma unroll
            for (int e = 0; e < V; e++) r[e] = quant_bits(to_f(v[j].t[e]), s[e]);
            auto four = [&](int e) { return __byte_perm(__byte_perm(r[e], r[e + 1], 0x0040), __byte_perm(r[e + 2], r[e + 3], 0x0040), 0x5410) & mask[e / 4]; };
            if constexpr (V == 1) *q = (signed char)(r[0] & mask[0]);
            else if constexpr (V == 4) *reinterpret_cast<uint32_t*>(q) = four(0);
            else *reinterpret_cast<uint2*>(q) = make_uint2(four(0), four(4));
        }
    }
}

template <typename T, int KEEP>
cudaError_t launch_across(const T* X, size_t ldx, signed char* Q, size_t ldq, float* scale, size_t lines, size_t len, unsigned ranks, cudaStream_t s)
{
    const size_t strips = (len + 31) / 32;
    if (strips * ranks >= (1u << 31)) return cudaErrorNotSupported;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(strips * ranks));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    count_launch();
    return cudaLaunchKernelEx(&cfg, quantize_across_kernel<T, KEEP>, X, ldx, Q, ldq, scale, lines, len);
}

template <typename T, int V, int COLS>
cudaError_t launch_across_passes(const T* X, size_t ldx, signed char* Q, size_t ldq, float* scale, size_t lines, size_t len, cudaStream_t s)
{
    const size_t strips = (len + COLS * V - 1) / (COLS * V), at_least = 8 * (32 / COLS);
    if (strips >= (1u << 31)) return cudaErrorNotSupported;
    // Blocks of lines: four CTAs per SM, 64 blocks at most (every CTA of the second pass reads their maxima).
    size_t blocks = ((size_t)sm_count() * 4 + strips - 1) / strips;
    blocks = std::min(std::min<size_t>(blocks, 64), (lines + at_least - 1) / at_least);
    unsigned* tops = nullptr;
    cudaError_t e = ws_alloc(reinterpret_cast<void**>(&tops), blocks * len * sizeof(unsigned), s);
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)strips, (unsigned)blocks);
    e = launch_chained(across_max_kernel<T, V, COLS>, grid, 256, s, X, ldx, tops, lines, len);
    if (e == cudaSuccess) e = launch_chained(across_quantize_kernel<T, V, COLS>, grid, 256, s, X, ldx, Q, ldq, (const unsigned*)tops, scale, lines, len);
    count_launch(2);
    const cudaError_t e2 = ws_free(tops, s);
    return e == cudaSuccess ? e2 : e;
}

template <typename T>
cudaError_t quantize_typed(bool per_line, const T* X, size_t ldx, signed char* Q, size_t ldq, float* scale, size_t lines, size_t len, cudaStream_t s)
{
    constexpr int V = 16 / sizeof(T);
    if (!per_line) {
        const size_t strips = (len + 31) / 32;
        unsigned ranks = 1;
        while (ranks < 8 && lines > (size_t)8 * ranks && (lines > (size_t)8 * 64 * ranks || strips * ranks < 2 * (size_t)sm_count())) ranks *= 2;
        const bool vec = aligned16(X) && (ldx * sizeof(T)) % 16 == 0 && len % V == 0 && (reinterpret_cast<uintptr_t>(Q) | ldq) % V == 0;
        // us, one kernel / two passes: 300 x 16000 BF16 12 / 14, 4096 x 1024 FP32 6.5 / 12, 4096 x 4096 FP32 24.2 / 24.6 (unaligned 25 / 45),
        // 4096 x 11008 BF16 117 / 57 (unaligned 118 / 114).
        if (!(vec && lines * len > (1u << 24))) {
            if (lines <= (size_t)8 * 64 * ranks) return launch_across<T, 64>(X, ldx, Q, ldq, scale, lines, len, ranks, s);
            if (lines <= (size_t)8 * 80 * ranks) return launch_across<T, 80>(X, ldx, Q, ldq, scale, lines, len, ranks, s);
        }
        if (vec && len >= 8 * V) return len >= 32 * V ? launch_across_passes<T, V, 32>(X, ldx, Q, ldq, scale, lines, len, s)
                                                      : launch_across_passes<T, V, 8>(X, ldx, Q, ldq, scale, lines, len, s);
        return launch_across_passes<T, 1, 32>(X, ldx, Q, ldq, scale, lines, len, s);
    }
    if (lines >= (1u << 31)) return cudaErrorNotSupported;
    count_launch();
    const unsigned grid = (unsigned)lines;
    // 64 elements a thread in registers.  8192 x 8192 BF16: 34 to 36 us in a row with 128 threads a line (5.6 to 5.9 TB/s, 87 to 91 % of a
    // copy's rate), 3 more with 64 or 256 of 32 elements each, 9 more with 512; so as few threads as hold the line.
    if (aligned16(X) && (ldx * sizeof(T)) % 16 == 0 && (reinterpret_cast<uintptr_t>(Q) | ldq) % V == 0) {
        if (len <= 128 * 64) return launch_chained(quantize_lines_kernel<T, 128, V, 64 / V>, dim3(grid), 128, s, X, ldx, Q, ldq, scale, len);
        return launch_chained(quantize_lines_kernel<T, 256, V, 64 / V>, dim3(grid), 256, s, X, ldx, Q, ldq, scale, len);
    }
    return launch_chained(quantize_lines_kernel<T, 256, 1, 32>, dim3(grid), 256, s, X, ldx, Q, ldq, scale, len);
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
