// Newton-Schulz orthogonalisation of matrices whose smaller side is at most 128 and whose larger is at most 1024 (2048 where there are at
// most 15: orthogonalize_small_applies), all steps in one kernel: a cluster of up to 8 CTAs holds a matrix on chip.  (The iteration, its roundings and its scales: orthogonalize.cu.)
//
// CTA r of a cluster keeps W columns of X (n <= 128 rows, padded to 128): hi in shared memory, as 64-column slabs of SWIZZLE_128B rows,
// lo in registers, always in the same fragments of the same threads.  One copy of hi serves both products: as
// a k-contiguous operand of the Gram product (k = columns) and as a v-contiguous one of the update (k = rows; the same bytes read MN-major).
// A step:
//   Gram     each CTA multiplies its columns; the partial sums (128 x 128 FP32) meet in distributed shared memory, where a rank sums a
//            slice of the columns in rank order, subtracts the shift and writes the FP16 slice into every CTA's A
//   square   A A by every CTA for itself (two slabs), P in place of A
//   update   P X on the CTA's own columns, hi back in place
// Two cluster barriers per step and no global memory between the first load and the result.  The chain of kernels takes about 6 us for
// each of a step's products whatever their size, three quarters of it launches, first loads and ends.
#include "orthogonalize.cuh"

#include <algorithm>

namespace cb200 {

namespace {

using namespace narrow;

constexpr int SMALL_N = 128, SMALL_W = 256, SMALL_CLUSTER = 8, SMALL_THREADS = 256;
constexpr int SLAB = SMALL_N * SLAB_BYTES;                     // 64 columns (or k) of 128 rows: 16 KB
constexpr int X_BYTES = SMALL_W / 64 * SLAB, A_BYTES = 2 * SLAB, PART_BYTES = SMALL_N * SMALL_N * 4;
constexpr int SMALL_SMEM = X_BYTES + A_BYTES + PART_BYTES + 1024 + 512;
constexpr int MAX_STEPS = 64;

template <typename T>
struct SmallParams {
    const T* G; size_t ldg, strideG;
    uint16_t* O; size_t ldo, strideO;                          // BF16
    float alpha, beta;
    unsigned n, m, W;                                          // W: columns per CTA, a multiple of 64
    u64 kappa_lo;                                              // bit k: step k puts kappa on lo
    int steps, align, align_g;                                 // align: of O's lines; align_g: of G's, 16, 4 or 2 bytes (16-bit types), 8 or 4 (FP32)
    bool flip;                                                 // X(u, v) at G[v * ldg + u] and O[v * ldo + u]
    float coeffs[3 * MAX_STEPS];
};

// Byte offset of element (row, col) in slabs of SWIZZLE_128B rows; col even: the pair lies in one word.
__device__ __forceinline__ int slab_at(int row, int col)
{
    return (col >> 6) * SLAB + row * SLAB_BYTES + ((((col & 63) >> 3) ^ (row & 7)) << 4) + (col & 7) * 2;
}

__device__ __forceinline__ void st_cluster1(uint32_t addr, double v) { asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory"); }
__device__ __forceinline__ void st_cluster1(uint32_t addr, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory"); }
__device__ __forceinline__ void st_cluster4(uint32_t addr, const uint32_t (&v)[4])
{
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
// Between writes (or, after a barrier, other threads' writes) to shared memory, here or in another CTA, and products that read them.
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async;" ::: "memory"); }

// A chunk of 32 rows x 32 columns of X0 (unscaled) as fragments, x[g][2 k + e]; zero outside.
template <typename T>
__device__ __forceinline__ void load_chunk(float (&x)[4][8], const SmallParams<T>& p, const T* G, unsigned u0, unsigned v0)
{
    const int lane = threadIdx.x & 31, q = lane & 3;
    if constexpr (sizeof(T) == 2) {
        Bits16<4> bits;
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int k = 0; k < 4; k++) bits.h[g][k] = 0;
        if (p.flip) {
            load_columns16<4>(bits, reinterpret_cast<const uint16_t*>(G), p.ldg, u0, v0, p.n, p.m, p.align_g);
            columns_to_fragments<4>(bits);
        } else {
            load_rows16<4>(bits, reinterpret_cast<const uint16_t*>(G), p.ldg, u0, v0, p.n, p.m, p.align_g);
            rows_to_fragments<4>(bits, v0, p.m, p.align_g);
        }
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const T* t = reinterpret_cast<const T*>(&bits.h[g][k]);
                x[g][2 * k] = to_f(t[0]);
                x[g][2 * k + 1] = to_f(t[1]);
            }
    } else {
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const unsigned u = u0 + 8 * g + lane / 4, v = v0 + 8 * k + 2 * q;
                float2 a = make_float2(0.f, 0.f);
                if (u < p.n && v < p.m) {
                    if (!p.flip && p.align_g == 8 && v + 2 <= p.m) {
                        a = *reinterpret_cast<const float2*>(G + (size_t)u * p.ldg + v);
                    } else {
                        a.x = p.flip ? G[(size_t)v * p.ldg + u] : G[(size_t)u * p.ldg + v];
                        if (v + 1 < p.m) a.y = p.flip ? G[(size_t)(v + 1) * p.ldg + u] : G[(size_t)u * p.ldg + v + 1];
                    }
                }
                x[g][2 * k] = a.x;
                x[g][2 * k + 1] = a.y;
            }
    }
}

template <typename T, int RANKS>
__global__ void __launch_bounds__(SMALL_THREADS, 1) orthogonalize_small_kernel(const __grid_constant__ SmallParams<T> p)
{
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* X = smem;
    unsigned char* A = smem + X_BYTES;
    // Partial sums: [RANKS sources][4 quarters][OWN groups of 8 columns][2 pairs of g][32 lanes], 16 bytes each.
    uint4* part = reinterpret_cast<uint4*>(smem + X_BYTES + A_BYTES);
    constexpr int OWN = 16 / RANKS;                            // groups that a rank sums
    uint64_t* bar = reinterpret_cast<uint64_t*>(smem + X_BYTES + A_BYTES + PART_BYTES);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + 1);
    double* from_rank = reinterpret_cast<double*>(bar + 2);    // [SMALL_CLUSTER], written by every rank
    double* from_warp = from_rank + SMALL_CLUSTER;             // [8]; both: 64 bits for the norm, FP32 for the sums of the steps

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, quarter = warp & 3, half = warp / 4, q = lane & 3;
    const uint32_t rank = cluster_ctarank();
    const unsigned z = blockIdx.x / RANKS, first = rank * p.W;  // first column of X here
    const int chunks = (int)p.W / 32, row0 = 32 * quarter + lane / 4;
    const T* G = p.G + z * p.strideG;

    if (threadIdx.x == 0) {
        mbar_init(bar, 1);
        mbar_fence_init();
    }
    if (warp == 0) tmem_alloc<1>(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();
    pdl_wait();

    // Sum over the CTA's threads in a fixed order, in two halves: before and after a __syncthreads().  It reaches every rank with
    // the next cluster barrier.
    auto gather_warp = [&](auto sum) {
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) reinterpret_cast<decltype(sum)*>(from_warp)[warp] = sum;
    };
    auto publish = [&](auto zero) {
        if (threadIdx.x < RANKS) {
            auto all = zero;
#pragma unroll
            for (int w = 0; w < 8; w++) all += reinterpret_cast<decltype(zero)*>(from_warp)[w];
            st_cluster1(map_shared(smem_u32(reinterpret_cast<decltype(zero)*>(from_rank) + rank), threadIdx.x), all);
        }
        __syncwarp();
    };
    auto gathered = [&](auto zero) {
        auto all = zero;
#pragma unroll
        for (int r = 0; r < RANKS; r++) all += reinterpret_cast<decltype(zero)*>(from_rank)[r];
        return all;
    };

    double sum = 0;
#pragma unroll 1
    for (int c = half; c < chunks; c += 2) {
        float x[4][8];
        load_chunk<T>(x, p, G, 32 * quarter, first + c * 32);
#pragma unroll
        for (int g = 0; g < 4; g++) sum += sum_of_squares(x[g]);
    }
    gather_warp(sum);
    cluster_sync();                                            // every CTA runs
    publish(0.0);
    cluster_sync();
    float f0, f1;
    double square;
    int e;                                                     // X is held times 2^e
    norm_factors(sqrt(gathered(0.0)), f0, f1, square, e);
    const float per_mean = 1.f / (SX * SX * (float)p.n), mean0 = (float)(square / p.n);

    constexpr int MINE = SMALL_W / 64;                         // chunks per warp at most
    uint32_t lo[MINE][4][4];
#pragma unroll
    for (int i = 0; i < MINE; i++) {
        const int c = half + 2 * i;
        if (c >= chunks) break;
        float x[4][8];
        load_chunk<T>(x, p, G, 32 * quarter, first + c * 32);
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float a = x[g][2 * k] * f0 * f1, b = x[g][2 * k + 1] * f0 * f1;
                const uint32_t h = pack(a, b);
                const float2 r = unpack(h);
                lo[i][g][k] = pack(a - r.x, b - r.y);
                *reinterpret_cast<uint32_t*>(X + slab_at(row0 + 8 * g, c * 32 + 8 * k + 2 * q)) = h;
            }
    }
    proxy_fence();
    __syncthreads();

    uint32_t phase = 0;
    bool ok = true;
    // One thread issues products and everybody waits for them.
    auto wait_products = [&] {
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar, phase));      // after one that ran out: no more, but all barriers
        phase ^= 1;
        tc_fence_after();
    };
#pragma unroll 1
    for (int step = 0; step < p.steps; step++) {
        const float a = p.coeffs[3 * step], b = p.coeffs[3 * step + 1], c = p.coeffs[3 * step + 2];
        // ---- Gram product of this CTA's columns ----
        if (threadIdx.x == 0) {
            tc_fence_after();
            constexpr uint32_t idesc = instr_desc<KIND_F16, 128, 1, false>();
            for (unsigned s = 0; s < p.W / 64; s++) {
                const uint64_t d = smem_desc<false>(smem_u32(X + s * SLAB));
                for (int ks = 0; ks < 4; ks++) umma<KIND_F16, 1>(tmem, d + 2 * ks, d + 2 * ks, idesc, s > 0 || ks > 0);
            }
            umma_commit<1>(bar);
        }
        __syncwarp();
        wait_products();
#pragma unroll
        for (int i = 0; i < 2; i++) {
            uint32_t lower[16], upper[16];
            const int c0 = half * 64 + i * 32;
            const uint32_t taddr = tmem + ((uint32_t)(32 * quarter) << 16) + c0;
            __syncwarp();
            tmem_ld_16x32(taddr, lower);
            tmem_ld_16x32(taddr + (16u << 16), upper);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int group = c0 / 8 + k;
                const uint32_t to = map_shared(smem_u32(part + ((int)rank * 4 + quarter) * OWN * 64 + (group % OWN) * 64 + lane), group / OWN);
                const uint32_t v[4] = {lower[4 * k], lower[4 * k + 1], lower[4 * k + 2], lower[4 * k + 3]};
                const uint32_t w[4] = {upper[4 * k], upper[4 * k + 1], upper[4 * k + 2], upper[4 * k + 3]};
                st_cluster4(to, v);
                st_cluster4(to + 512, w);
            }
        }
        __syncwarp();
        cluster_sync();
        // ---- this rank's slice of A = X X' - t I, into every CTA ----
        const bool last = step + 1 == p.steps;
        const float mean = step == 0 ? mean0 : gathered(0.f) * per_mean, t = shift(mean, e);
#pragma unroll
        for (int jj = 0; jj < (OWN + 1) / 2; jj++) {
            const int j = half + 2 * jj;
            if (j >= OWN) break;
            const uint4* w = part + (quarter * OWN + j) * 64 + lane;
            float v[8] = {};
#pragma unroll
            for (int r = 0; r < RANKS; r++) {
                const uint4 x = w[r * 4 * OWN * 64], y = w[r * 4 * OWN * 64 + 32];
                v[0] += __uint_as_float(x.x); v[1] += __uint_as_float(x.y); v[2] += __uint_as_float(x.z); v[3] += __uint_as_float(x.w);
                v[4] += __uint_as_float(y.x); v[5] += __uint_as_float(y.y); v[6] += __uint_as_float(y.z); v[7] += __uint_as_float(y.w);
            }
            const int col0 = ((int)rank * OWN + j) * 8;
            uint32_t h[4];
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const int row = row0 + 8 * g, off = row - col0 - 2 * q;
                float a0 = v[2 * g] * (SA / (SX * SX)), a1 = v[2 * g + 1] * (SA / (SX * SX));
                if (off == 0 && row < (int)p.n) a0 -= SA * t;
                if (off == 1 && row < (int)p.n) a1 -= SA * t;
                h[g] = pack(a0, a1);
            }
            quad_transpose(h);                                 // eight columns of row 8 q + lane / 4 of the quarter
            const uint32_t at = smem_u32(A + slab_at(32 * quarter + 8 * q + lane / 4, col0));
#pragma unroll
            for (int r = 0; r < RANKS; r++) st_cluster4(map_shared(at, r), h);
        }
        proxy_fence();
        __syncwarp();
        cluster_sync();
        // ---- P <- (b + 2 c t) A + c A^2 ----
        StepFactors by;
        if (c != 0.f) {
            if (threadIdx.x == 0) {
                proxy_fence();
                tc_fence_after();
                constexpr uint32_t idesc = instr_desc<KIND_F16, 128, 1, false>();
                for (int s = 0; s < 2; s++) {
                    const uint64_t d = smem_desc<false>(smem_u32(A + s * SLAB));
                    for (int ks = 0; ks < 4; ks++) umma<KIND_F16, 1>(tmem + 128, d + 2 * ks, d + 2 * ks, idesc, s > 0 || ks > 0);
                }
                umma_commit<1>(bar);
            }
            __syncwarp();
            by = step_factors(mean * (float)p.n, t, e, a, b, c, last, p.alpha / SX, (p.kappa_lo >> step) & 1);       // under the products
            wait_products();
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float x[4][4][2];
                const int c0 = half * 64 + i * 32;
                read_chunk<KIND_F16>(x, tmem + 128 + ((uint32_t)(32 * quarter) << 16) + c0);
#pragma unroll
                for (int g = 0; g < 4; g++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        uint32_t* w = reinterpret_cast<uint32_t*>(A + slab_at(row0 + 8 * g, c0 + 8 * k + 2 * q));
                        const float2 v = unpack(*w);
                        *w = pack(fmaf(by.b, v.x, by.f * x[g][k][0]), fmaf(by.b, v.y, by.f * x[g][k][1]));
                    }
            }
            tc_fence_before();
            proxy_fence();
            __syncthreads();
        }
        // ---- X <- (a + b t + c t^2) X + P X on this CTA's columns (A with factor b instead of P when c == 0) ----
        if (threadIdx.x == 0) {
            proxy_fence();
            tc_fence_after();
            const uint32_t idesc = (1u << 4) | (1u << 16) | ((p.W >> 3) << 17) | ((128u >> 4) << 24);
            for (int kb = 0; kb < 2; kb++) {
                const uint64_t dp = smem_desc<false>(smem_u32(A + kb * SLAB));
                // 64 columns x 64 rows of X, v-contiguous: the next 64 columns lie one slab further
                uint64_t dx = smem_desc<true>(smem_u32(X + kb * 64 * SLAB_BYTES));
                dx = (dx & ~((uint64_t)0x3fff << 16)) | (uint64_t)(SLAB >> 4) << 16;
                for (int ks = 0; ks < 4; ks++) umma<KIND_F16, 1>(tmem + 256, dp + 2 * ks, dx + ks * (16 * SLAB_BYTES >> 4), idesc, kb > 0 || ks > 0);
            }
            umma_commit<1>(bar);
        }
        __syncwarp();
        if (c == 0.f) by = step_factors(mean * (float)p.n, t, e, a, b, c, last, p.alpha / SX, (p.kappa_lo >> step) & 1);
        wait_products();
        e = by.next;
        float total = 0;
#pragma unroll
        for (int i = 0; i < MINE; i++) {
            const int ch = half + 2 * i;
            if (ch >= chunks) break;
            float x[4][4][2];
            read_chunk<KIND_F16>(x, tmem + 256 + ((uint32_t)(32 * quarter) << 16) + ch * 32);
            float sq = 0.f;
#pragma unroll
            for (int g = 0; g < 4; g++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint32_t* xs = reinterpret_cast<uint32_t*>(X + slab_at(row0 + 8 * g, ch * 32 + 8 * k + 2 * q));
                    const float2 h = unpack(*xs), l = unpack(lo[i][g][k]);
                    const float y0 = fmaf(by.w, h.x, fmaf(by.v, l.x, by.g * x[g][k][0])), y1 = fmaf(by.w, h.y, fmaf(by.v, l.y, by.g * x[g][k][1]));
                    x[g][k][0] = y0;
                    x[g][k][1] = y1;
                    if (!last) {
                        const uint32_t nh = pack(y0, y1);
                        const float2 r = unpack(nh);
                        lo[i][g][k] = pack(y0 - r.x, y1 - r.y);
                        *xs = nh;
                        sq = fmaf(y0, y0, fmaf(y1, y1, sq));  // zero outside the matrix
                    }
                }
            total += sq;
            if (last) {
                const unsigned u0 = 32 * quarter, v0 = first + ch * 32;
                uint16_t* o = p.O + z * p.strideO;
                Bits16<4> bits;
                if (p.beta != 0.f) {
                    if (p.flip) { load_columns16<4>(bits, o, p.ldo, u0, v0, p.n, p.m, p.align); columns_to_fragments<4>(bits); }
                    else        { load_rows16<4>(bits, o, p.ldo, u0, v0, p.n, p.m, p.align); rows_to_fragments<4>(bits, v0, p.m, p.align); }
#pragma unroll
                    for (int g = 0; g < 4; g++)
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const float2 old = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&bits.h[g][k]));
                            x[g][k][0] = fmaf(p.beta, old.x, x[g][k][0]);
                            x[g][k][1] = fmaf(p.beta, old.y, x[g][k][1]);
                        }
                }
#pragma unroll
                for (int g = 0; g < 4; g++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const __nv_bfloat162 v = __floats2bfloat162_rn(x[g][k][0], x[g][k][1]);
                        bits.h[g][k] = *reinterpret_cast<const uint32_t*>(&v);
                    }
                if (p.flip) store_columns16<4>(bits, o, p.ldo, u0, v0, p.n, p.m, p.align);
                else        store_rows16<4>(bits, o, p.ldo, u0, v0, p.n, p.m, p.align);
            }
        }
        if (!last) gather_warp(total);
        tc_fence_before();
        proxy_fence();
        __syncthreads();
        if (!last) publish(0.f);                                // read after the first cluster barrier of the next step
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync();                                            // no CTA leaves while another may still write to it
    tc_fence_after();
    if (warp == 0) tmem_free<1>(tmem, 512);
}

}  // namespace

namespace {

// Clusters of 1, 2, 4, 8 CTAs that run at once on 148 SMs, one CTA per SM (GPCs are not all of a size).
size_t clusters_at_once(unsigned ranks) { return ranks == 1 ? (size_t)sm_count() : ranks == 2 ? (size_t)sm_count() / 2 : ranks == 4 ? 33 : 15; }

// CTAs per matrix: no fewer than hold its columns, more (down to 64 columns each) while the whole batch stays one round.
unsigned small_ranks(size_t batch, size_t m)
{
    unsigned ranks = 1;
    while (ranks < SMALL_CLUSTER && (size_t)ranks * SMALL_W < m) ranks *= 2;
    while (ranks < SMALL_CLUSTER && (size_t)ranks * 64 < m && batch <= clusters_at_once(2 * ranks)) ranks *= 2;
    return ranks;
}

template <typename T, int RANKS>
cudaError_t launch_small(const SmallParams<T>& k, size_t batch, cudaStream_t s)
{
    auto kernel = orthogonalize_small_kernel<T, RANKS>;
    static DeviceOnce once;
    cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMALL_SMEM); });
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)batch * RANKS);
    cfg.blockDim = dim3(SMALL_THREADS);
    cfg.dynamicSmemBytes = SMALL_SMEM;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = RANKS;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, kernel, k);
    if (e == cudaSuccess) count_launch();
    return e;
}

}  // namespace

bool orthogonalize_small_applies(const OrthProblem& p)
{
    // Several rounds still win while 4 CTAs hold a matrix (256 matrices of 128 x 512: 256 us, the chain 353), and lose with 8 (64 of
    // 128 x 2048: 374 against 327).
    const size_t n = std::min(p.lines, p.len), m = std::max(p.lines, p.len);
    return n <= SMALL_N && (m <= (size_t)SMALL_W * 4 || (m <= (size_t)SMALL_W * SMALL_CLUSTER && p.batch <= clusters_at_once(SMALL_CLUSTER)));
}

template <typename T>
cudaError_t orthogonalize_small(const OrthProblem& p, cudaStream_t s)
{
    SmallParams<T> k = {};
    k.flip = p.lines > p.len;
    k.n = (unsigned)std::min(p.lines, p.len);
    k.m = (unsigned)std::max(p.lines, p.len);
    // As many CTAs as there are 64-column slabs, up to the cluster's limit and to one round of the whole batch.
    const unsigned ranks = small_ranks(p.batch, k.m);
    k.W = ((k.m + ranks - 1) / ranks + 63) / 64 * 64;
    k.G = static_cast<const T*>(p.G) + p.offG; k.ldg = p.ldg; k.strideG = p.strideG;
    k.O = static_cast<uint16_t*>(p.O) + p.offO; k.ldo = p.ldo; k.strideO = p.strideO;
    k.alpha = p.alpha; k.beta = p.beta; k.steps = p.steps;
    for (int i = 0; i < p.steps; i++) k.kappa_lo |= (u64)kappa_on_lo(k.n, p.coeffs, i, p.steps) << i;
    const size_t stride_g = p.batch > 1 ? p.strideG : 0;
    k.align_g = sizeof(T) == 2 ? line_alignment(k.G, p.ldg, stride_g)
                               : (reinterpret_cast<uintptr_t>(k.G) | p.ldg * 4 | stride_g * 4) % 8 == 0 ? 8 : 4;
    k.align = line_alignment(k.O, p.ldo, p.batch > 1 ? p.strideO : 0);
    for (int i = 0; i < p.steps; i++) {
        k.coeffs[3 * i] = p.coeffs ? p.coeffs[3 * i] : 3.4445f;
        k.coeffs[3 * i + 1] = p.coeffs ? p.coeffs[3 * i + 1] : -4.7750f;
        k.coeffs[3 * i + 2] = p.coeffs ? p.coeffs[3 * i + 2] : 2.0315f;
    }
    set_last_variant(ranks == 1 ? "orthogonalize_small<1>" : ranks == 2 ? "orthogonalize_small<2>" : ranks == 4 ? "orthogonalize_small<4>" : "orthogonalize_small<8>");
    switch (ranks) {
        case 1: return launch_small<T, 1>(k, p.batch, s);
        case 2: return launch_small<T, 2>(k, p.batch, s);
        case 4: return launch_small<T, 4>(k, p.batch, s);
        default: return launch_small<T, 8>(k, p.batch, s);
    }
}
template cudaError_t orthogonalize_small<float>(const OrthProblem&, cudaStream_t);
template cudaError_t orthogonalize_small<__half>(const OrthProblem&, cudaStream_t);
template cudaError_t orthogonalize_small<__nv_bfloat16>(const OrthProblem&, cudaStream_t);

unsigned orthogonalize_small_fault_flag() { return read_wait_timeout_flag(); }

}  // namespace cb200
