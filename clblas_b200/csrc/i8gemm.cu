// C <- alpha * diag(sA) * op(A) * op(B) * diag(sB) + beta * C, A and B signed 8-bit integers, C in FP32, FP16 or BF16.
// (No counterpart in the reference, whose products are FP32 / FP64: the linear layer of a language model with one scale per
// token and per output channel.)
//
// The products are exact: tcgen05.mma.kind::i8 accumulates in 32-bit integers, |sum| <= K * 2^14 < 2^31 for the K <= 131071 the
// front end admits, in any order and over any split of K.  The sum is rounded once to FP32, scaled in FP32 (three
// roundings) and rounded once to the type of C.
//
// Both operands are read k-contiguous with 128-byte slabs (narrow_mma.cuh); an operand stored the other way, or not 16-byte
// aligned, is transposed / copied once into a workspace.
#include "narrow_mma.cuh"

#include <cstdio>

namespace cb200 {

namespace {

using namespace narrow;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }

template <typename T> __device__ __forceinline__ uint32_t pack16(float a, float b);
template <> __device__ __forceinline__ uint32_t pack16<__half>(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
template <> __device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float a, float b) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
template <typename T> __device__ __forceinline__ float2 unpack16(uint32_t h);
template <> __device__ __forceinline__ float2 unpack16<__half>(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }
template <> __device__ __forceinline__ float2 unpack16<__nv_bfloat16>(uint32_t h) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&h)); }

// C[u, v] <- alpha su[u] sv[v] acc + beta C[u, v].
template <typename T>
struct EpiScaled {
    static constexpr bool kHeavy = sizeof(T) == 4;
    static constexpr bool kTriangle = false;
    struct State { float factor[4]; };
    template <int G> struct Pre { Bits16<G> c; };
    // Scales of the rows u and the columns v; nullptr: ones.  Read by ordinary loads after pdl_wait() and not as constants (__ldg): the
    // quantisation before may still write them while this kernel is already resident, next to a product that has the old ones cached.
    const float* su;
    const float* sv;
    float alpha, beta;
    T* C;
    size_t ld;
    bool trans;                     // element (u, v) at C[v * ld + u] instead of C[u * ld + v]
    int align;                      // of C's lines: 16, 4 or 2 bytes (16-bit C); 8-byte accesses allowed when 8 or more (32-bit C)

    __device__ void begin(State& st, const Shape& s, unsigned, unsigned u0, unsigned) const
    {
        const unsigned u = u0 + (threadIdx.x & 31) / 4;
#pragma unroll
        for (int g = 0; g < 4; g++) st.factor[g] = su && u + 8 * g < s.U ? alpha * su[u + 8 * g] : alpha;
    }
    template <int G>
    __device__ void fetch(Pre<G>& p, const Shape& s, unsigned, unsigned u0, unsigned v0) const
    {
        if (sizeof(T) == 4 || beta == 0.f) return;
        if (trans) load_columns16<G>(p.c, reinterpret_cast<const uint16_t*>(C), ld, u0, v0, s.U, s.V, align);
        else load_rows16<G>(p.c, reinterpret_cast<const uint16_t*>(C), ld, u0, v0, s.U, s.V, align);
    }
    template <int G>
    __device__ void chunk(State& st, Pre<G>& p, const Shape& s, unsigned z, unsigned u0, unsigned v0, unsigned v_next, int, float (&x)[4][G][2]) const
    {
        const int lane = threadIdx.x & 31, q = lane & 3;
        const unsigned u = u0 + lane / 4;
#pragma unroll
        for (int k = 0; k < G; k++) {
            const unsigned v = v0 + 8 * k + 2 * q;
            const float w0 = sv && v < s.V ? sv[v] : 1.f, w1 = sv && v + 1 < s.V ? sv[v + 1] : 1.f;
#pragma unroll
            for (int g = 0; g < 4; g++) {
                x[g][k][0] = x[g][k][0] * st.factor[g] * w0;
                x[g][k][1] = x[g][k][1] * st.factor[g] * w1;
            }
        }
        if (sizeof(T) == 4 && beta != 0.f) {
            T old[4][G][2];
#pragma unroll
            for (int g = 0; g < 4; g++)
#pragma unroll
                for (int k = 0; k < G; k++)
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        if (u + 8 * g < s.U && v0 + 8 * k + 2 * q + e < s.V) old[g][k][e] = C[at(u + 8 * g, v0 + 8 * k + 2 * q + e)];
#pragma unroll
            for (int g = 0; g < 4; g++)
#pragma unroll
                for (int k = 0; k < G; k++)
#pragma unroll
                    for (int e = 0; e < 2; e++) x[g][k][e] = fmaf(beta, to_f(old[g][k][e]), x[g][k][e]);
        }
        if constexpr (sizeof(T) == 2) {
            if (beta != 0.f) {
                if (trans) columns_to_fragments<G>(p.c);
                else rows_to_fragments<G>(p.c, v0, s.V, align);
#pragma unroll
                for (int g = 0; g < 4; g++)
#pragma unroll
                    for (int k = 0; k < G; k++) {
                        const float2 c = unpack16<T>(p.c.h[g][k]);
                        x[g][k][0] = fmaf(beta, c.x, x[g][k][0]);
                        x[g][k][1] = fmaf(beta, c.y, x[g][k][1]);
                    }
            }
            if (v_next != ~0u) fetch<G>(p, s, z, u0, v_next);
            Bits16<G> o;
#pragma unroll
            for (int g = 0; g < 4; g++)
#pragma unroll
                for (int k = 0; k < G; k++) o.h[g][k] = pack16<T>(x[g][k][0], x[g][k][1]);
            if (trans) store_columns16<G>(o, reinterpret_cast<uint16_t*>(C), ld, u0, v0, s.U, s.V, align);
            else store_rows16<G>(o, reinterpret_cast<uint16_t*>(C), ld, u0, v0, s.U, s.V, align);
        } else {                                                    // 32-bit: a quad's fragments fill 32 bytes of a row, eight lanes' 32 bytes of a column
#pragma unroll
            for (int g = 0; g < 4; g++)
#pragma unroll
                for (int k = 0; k < G; k++) {
                    const unsigned v = v0 + 8 * k + 2 * q;
                    if (u + 8 * g >= s.U) continue;
                    float* c = reinterpret_cast<float*>(C) + at(u + 8 * g, v);
                    if (!trans && align >= 8 && v + 2 <= s.V) *reinterpret_cast<float2*>(c) = make_float2(x[g][k][0], x[g][k][1]);
                    else {
                        if (v < s.V) *c = x[g][k][0];
                        if (v + 1 < s.V) c[trans ? ld : 1] = x[g][k][1];
                    }
                }
        }
    }
    __device__ size_t at(unsigned u, unsigned v) const { return trans ? (size_t)v * ld + u : (size_t)u * ld + v; }
    __device__ void end(State&, unsigned, unsigned) const {}
};

// C <- beta * C (K == 0 or alpha == 0): lines of `len` contiguous elements.
template <typename T>
__global__ void scale_lines_kernel(T* C, size_t lines, size_t len, size_t ld, float beta)
{
    const size_t total = lines * len;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (size_t)gridDim.x * blockDim.x) {
        T* c = C + (i / len) * ld + i % len;
        *c = from_f<T>(beta == 0.f ? 0.f : beta * to_f(*c));
    }
}

// An operand on its way to k-contiguous lines of pitch ldd (a multiple of 16, so whole 16-byte words of a line may be written).
struct PackJob {
    unsigned char* dst; size_t ldd;
    const unsigned char* src; size_t lds;
    size_t rows, K;
    bool transpose;                 // src[k][r] instead of src[r][k]
    bool words;                     // transpose: base and pitch allow 4-byte loads
    unsigned tiles_r;               // transpose: tiles of 128 rows
    unsigned blocks;
};

// dst[r][k] <- src[k][r].  128 x 128 bytes per CTA: words of four r are read along r, 4 x 4 bytes are exchanged in registers,
// words of four k go to shared memory (word w of row r at w ^ (r / 4), free of bank conflicts both ways) and leave as 128-byte rows.
__device__ __forceinline__ void transpose_tile(const PackJob& j, unsigned block, uint32_t* tile)
{
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const size_t r0 = (size_t)(block % j.tiles_r) * 128, k0 = (size_t)(block / j.tiles_r) * 128, r = r0 + 4 * lane;
    uint32_t w[4][4];
#pragma unroll
    for (int g = 0; g < 4; g++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const size_t k = k0 + 4 * (warp * 4 + g) + i;
            const unsigned char* p = j.src + k * j.lds + r;
            w[g][i] = 0;
            if (k >= j.K) continue;
            if (j.words && r + 4 <= j.rows) {
                w[g][i] = *reinterpret_cast<const uint32_t*>(p);
            } else {
#pragma unroll
                for (int b = 0; b < 4; b++)
                    if (r + b < j.rows) w[g][i] |= (uint32_t)p[b] << (8 * b);
            }
        }
#pragma unroll
    for (int g = 0; g < 4; g++) {
        const int kw = warp * 4 + g;                       // word of four k
        const uint32_t a = __byte_perm(w[g][0], w[g][1], 0x5140), b = __byte_perm(w[g][2], w[g][3], 0x5140);      // bytes 0, 1 of each pair
        const uint32_t c = __byte_perm(w[g][0], w[g][1], 0x7362), d = __byte_perm(w[g][2], w[g][3], 0x7362);      // bytes 2, 3
        const uint32_t o[4] = {__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632), __byte_perm(c, d, 0x5410), __byte_perm(c, d, 0x7632)};
#pragma unroll
        for (int i = 0; i < 4; i++) tile[(4 * lane + i) * 32 + (kw ^ lane)] = o[i];
    }
    __syncthreads();
    for (int i = warp; i < 128; i += 8) {
        const size_t row = r0 + i, k = k0 + 4 * lane;
        if (row < j.rows && k < j.K) *reinterpret_cast<uint32_t*>(j.dst + row * j.ldd + k) = tile[i * 32 + (lane ^ (i / 4))];
    }
}

// dst[r][k] <- src[r][k] for a source of any alignment, 16 bytes of dst a thread.  They are cut out of the five aligned words that
// hold them when all of those lie inside the row, and collected byte by byte at its ends.
__device__ __forceinline__ void copy_piece(const PackJob& j, unsigned block)
{
    const unsigned per_row = (unsigned)((j.K + 15) / 16);
    const size_t i = (size_t)block * 256 + threadIdx.x, row = i / per_row;
    const unsigned k = (unsigned)(i - row * per_row) * 16;
    if (row >= j.rows) return;
    const unsigned char* line = j.src + row * j.lds;
    const unsigned char* p = line + k;
    const unsigned mis = (unsigned)(reinterpret_cast<uintptr_t>(p) & 3u);
    const unsigned char* q = p - mis;
    uint32_t o[4] = {};
    if (q >= line && q + (mis ? 20 : 16) <= line + j.K) {
        uint32_t w[5];
#pragma unroll
        for (int b = 0; b < 4; b++) w[b] = reinterpret_cast<const uint32_t*>(q)[b];
        w[4] = mis ? reinterpret_cast<const uint32_t*>(q)[4] : 0;
#pragma unroll
        for (int b = 0; b < 4; b++) o[b] = __funnelshift_r(w[b], w[b + 1], 8 * mis);
    } else {
#pragma unroll
        for (int b = 0; b < 16; b++)
            if (k + b < j.K) o[b / 4] |= (uint32_t)p[b] << (8 * (b % 4));
    }
    *reinterpret_cast<uint4*>(j.dst + row * j.ldd + k) = make_uint4(o[0], o[1], o[2], o[3]);
}

// Both operands of a product in one launch (either may have no blocks).
__global__ void __launch_bounds__(256) pack_kernel(const PackJob a, const PackJob b)
{
    __shared__ uint32_t tile[128 * 32];
    pdl_launch_dependents();
    pdl_wait();
    const bool first = blockIdx.x < a.blocks;
    const PackJob& j = first ? a : b;
    const unsigned block = first ? blockIdx.x : blockIdx.x - a.blocks;
    if (j.transpose) transpose_tile(j, block, tile);
    else copy_piece(j, block);
}

PackJob pack_job(unsigned char* dst, size_t ldd, const signed char* src, size_t lds, size_t rows, size_t K, bool transpose)
{
    PackJob j{dst, ldd, reinterpret_cast<const unsigned char*>(src), lds, rows, K, transpose, ((reinterpret_cast<uintptr_t>(src) | lds) & 3u) == 0, (unsigned)((rows + 127) / 128), 0};
    const size_t blocks = transpose ? j.tiles_r * ((K + 127) / 128) : (rows * ((K + 15) / 16) + 255) / 256;
    j.blocks = blocks < (1u << 30) ? (unsigned)blocks : 0;
    return j;
}

template <typename T>
cudaError_t multiply(const Operand& lines, const Operand& len, const float* s_lines, const float* s_len, float alpha, float beta, T* C,
                     size_t ldc, cudaStream_t st)
{
    // C is `lines.rows` lines of `len.rows` contiguous elements.
    const size_t L = lines.rows, W = len.rows, K = lines.inner;
    const int align = sizeof(T) == 2 ? line_alignment(C, ldc, 0) : (reinterpret_cast<uintptr_t>(C) | (ldc * 4)) % 8 == 0 ? 8 : 4;
    const unsigned nk = (unsigned)((K + slab_k(KIND_I8) - 1) / slab_k(KIND_I8));
    const unsigned sms = (unsigned)sm_count();
    Shape s = {};
    s.K = (unsigned)K;
    s.batch = 1;
    auto normal = [&] {
        s.U = (unsigned)L; s.V = (unsigned)W;
        return EpiScaled<T>{s_lines, s_len, alpha, beta, C, ldc, false, align};
    };
    // Few columns: k over as many CTAs as the machine has room for, two slabs each at least.
    auto split_for = [&](unsigned bn, unsigned per_sm) {
        const size_t tiles = ((s.U + BM - 1) / BM) * (size_t)((s.V + bn - 1) / bn);
        unsigned split = 1;
        while (split < (bn == 128 ? 4u : 8u) && tiles * split * 2 <= (size_t)sms * per_sm && split * 2 * 2 <= nk) split *= 2;
        return split;
    };
    if (L <= 128 && W > L) {
        // Few lines (decoding): the contiguous dimension supplies the 128 rows of the instruction, the lines its columns.
        s.U = (unsigned)W; s.V = (unsigned)L;
        const EpiScaled<T> epi{s_len, s_lines, alpha, beta, C, ldc, true, align};
        if (L <= 32) return run_split_by<KIND_I8, 32, false>(split_for(32, 2), len, lines, s, epi, st);
        if (L <= 64) return run_split_by<KIND_I8, 64, false>(split_for(64, 2), len, lines, s, epi, st);
        return run_split_by<KIND_I8, 128, false>(split_for(128, 1), len, lines, s, epi, st);
    }
    const EpiScaled<T> epi = normal();
    if (W <= 32) return run_split_by<KIND_I8, 32, false>(split_for(32, 2), lines, len, s, epi, st);
    if (W <= 64) return run_split_by<KIND_I8, 64, false>(split_for(64, 2), lines, len, s, epi, st);
    return run_planned<KIND_I8, false>(lines, len, s, epi, st);
}

template <typename T>
cudaError_t i8gemm_typed(const I8GemmProblem& p, cudaStream_t s)
{
    T* C = static_cast<T*>(p.C) + p.offC;
    if (p.K == 0 || p.alpha == 0.f) {
        if (p.beta == 1.f) return cudaSuccess;
        const size_t want = (p.lines * p.len + 255) / 256, most = (size_t)sm_count() * 16;
        scale_lines_kernel<T><<<(unsigned)(want < most ? want : most), 256, 0, s>>>(C, p.lines, p.len, p.ldc, p.beta);
        count_launch();
        return cudaGetLastError();
    }
    if (p.lines >= (1u << 31) || p.len >= (1u << 31)) return cudaErrorNotSupported;
    // (One row has no pitch: any may be given, more than a tensor map takes too.)
    auto usable = [](const void* q, size_t ld, bool kcontig, size_t rows) { return kcontig && aligned16(q) && (ld % 16 == 0 || rows == 1); };
    const bool fixP = !usable(p.P, p.ldp, p.p_kcontig, p.lines), fixQ = !usable(p.Q, p.ldq, p.q_kcontig, p.len);
    const size_t kld = (p.K + 15) / 16 * 16;
    Operand a{p.P, p.K, p.lines, p.lines == 1 ? kld : p.ldp, 0}, b{p.Q, p.K, p.len, p.len == 1 ? kld : p.ldq, 0};
    unsigned char* ws = nullptr;
    cudaError_t e = cudaSuccess;
    if (fixP || fixQ) {
        const size_t pn = fixP ? kld * p.lines : 0, qn = fixQ ? kld * p.len : 0, at = (pn + 255) / 256 * 256;
        if ((e = ws_alloc(reinterpret_cast<void**>(&ws), at + qn, s)) != cudaSuccess) return e;
        PackJob jobs[2] = {};
        if (fixP) {
            jobs[0] = pack_job(ws, kld, p.P, p.ldp, p.lines, p.K, !p.p_kcontig);
            a.base = ws; a.ld = kld;
        }
        if (fixQ) {
            jobs[1] = pack_job(ws + at, kld, p.Q, p.ldq, p.len, p.K, !p.q_kcontig);
            b.base = ws + at; b.ld = kld;
        }
        if ((fixP && jobs[0].blocks == 0) || (fixQ && jobs[1].blocks == 0)) e = cudaErrorNotSupported;
        else e = launch_chained(pack_kernel, dim3(jobs[0].blocks + jobs[1].blocks), 256, s, jobs[0], jobs[1]);
        if (e == cudaSuccess) count_launch();
    }
    if (e == cudaSuccess) e = multiply<T>(a, b, p.s_lines, p.s_len, p.alpha, p.beta, C, p.ldc, s);
    if (e == cudaSuccess) {
        char name[64];
        std::snprintf(name, sizeof(name), "i8gemm_tcgen05<%s>", last_plan());
        set_last_variant(name);
    }
    if (ws) {
        const cudaError_t e2 = ws_free(ws, s);
        if (e == cudaSuccess) e = e2;
    }
    return e;
}

}  // namespace

cudaError_t i8gemm(const I8GemmProblem& p, cudaStream_t s)
{
    set_last_kernel("i8gemm_tcgen05");
    switch (p.type) {
        case clblasB200Float32: return i8gemm_typed<float>(p, s);
        case clblasB200Float16: return i8gemm_typed<__half>(p, s);
        default: return i8gemm_typed<__nv_bfloat16>(p, s);
    }
}

unsigned i8gemm_fault_flag() { return read_wait_timeout_flag(); }

}  // namespace cb200
