// Tensor-core tile engine of the narrow-type operators (8-bit products with scales, FP16 products of the Newton-Schulz
// orthogonalisation).  Both are  D[u, v] = sum_k P[u, k] * Q[v, k]  with P stored U x K and Q stored V x K, k contiguous (or, for Q, v contiguous:
// the MN-major form of the instruction); the epilogue is a functor.
//
// narrow_persistent_kernel: one CTA (or one pair of CTAs, tcgen05.mma.cta_group::2) per SM (pair of SMs) walks over output
// tiles.  10 warps: warp 0 loads slabs of 128 bytes along k with TMA into a ring, warp 1 owns tensor memory and issues the
// MMAs, warps 2-9 are the epilogue.  Two accumulators in tensor memory, so the epilogue of a tile runs under the products of the next.
//
// narrow_split_kernel: for products with fewer tiles than SMs.  The k range of a tile is cut over the CTAs of a cluster; the
// partial accumulators meet in distributed shared memory (each rank sums a slice of the columns, in rank order, so
// results do not depend on timing), then the same epilogue runs on the slices.  No workspace, no second launch.
//
// Every wait on an mbarrier is bounded (tma_pipeline.cuh).  A CTA whose wait ran out leaves its loops and still takes part in
// the cluster barriers, so its peers end too.
#pragma once

#include "common.h"
#include "tma_pipeline.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace cb200 {
namespace narrow {

enum Kind { KIND_F16 = 0, KIND_I8 = 1 };

constexpr int BM = 128;                       // rows of P per CTA = lanes of tensor memory
constexpr int SLAB_BYTES = 128;               // bytes along k per slab: one SWIZZLE_128B row
constexpr int EPI_WARPS = 8;
constexpr int THREADS = (2 + EPI_WARPS) * 32;
constexpr int STAGE_BUF = 32 * 32 * 4;        // per epilogue warp: 32 x 32 values on their way to coalesced stores

__host__ __device__ constexpr int slab_k(int kind) { return kind == KIND_I8 ? SLAB_BYTES : SLAB_BYTES / 2; }

// ---------------------------------------------------------------------------------------------------------------------
// PTX wrappers
// ---------------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t cluster_ctarank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_nctarank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
// All threads of all CTAs of the cluster; the warp must be converged.
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Address of `saddr` (this CTA's shared memory) in the shared memory of CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_shared(uint32_t saddr, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v)
{
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr)
{
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}

// 3-D tiled load (inner, row, batch).  CG == 2: the completion may be counted on the barrier of the pair's first CTA.
template <int CG>
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar)
{
    if (CG == 2)
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
            ::"r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
            ::"r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}

// Instruction descriptor: D = F32 / S32, A and B = F16 / signed 8-bit, M = BM * CG, N = BN; bit 16: Q is v-contiguous.
template <int KIND, int BN, int CG, bool QMN>
__host__ __device__ constexpr uint32_t instr_desc()
{
    return (KIND == KIND_I8 ? (2u << 4) | (1u << 7) | (1u << 10) : (1u << 4)) | (QMN ? 1u << 16 : 0u) |
           ((uint32_t)(BN >> 3) << 17) | ((uint32_t)((BM * CG) >> 4) << 24);
}

// Shared-memory matrix descriptor, SWIZZLE_128B.  k-contiguous: rows of 128 bytes, 8-row groups 1024 bytes apart.
// v-contiguous (MN-major): blocks of 64 v (128 bytes) x 64 k, each k one 128-byte row; groups of 8 k are 1024 bytes apart (stride
// offset), the next 64 v one block of 8192 bytes further (leading offset).
template <bool MN>
__device__ __forceinline__ uint64_t smem_desc(uint32_t saddr)
{
    uint64_t d = 0;
    d |= (uint64_t)((saddr >> 4) & 0x3fff);
    d |= (uint64_t)(MN ? (8192 >> 4) : 1) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

template <int KIND, int CG>
__device__ __forceinline__ void umma(uint32_t tmem_d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate)
{
#define CB200_UMMA(cg, kind)                                                                         \
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"                                         \
                 "tcgen05.mma.cta_group::" cg ".kind::" kind " [%0], %1, %2, %3, p;\n}\n"            \
                 ::"r"(tmem_d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory")
    if (KIND == KIND_I8) {
        if (CG == 2) CB200_UMMA("2", "i8"); else CB200_UMMA("1", "i8");
    } else {
        if (CG == 2) CB200_UMMA("2", "f16"); else CB200_UMMA("1", "f16");
    }
#undef CB200_UMMA
}

// Arrives on `bar` (and, for a pair, on the barrier at the same place in both CTAs) once the MMAs issued so far are done.
template <int CG>
__device__ __forceinline__ void umma_commit(uint64_t* bar)
{
    if (CG == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t cols)
{
    if (CG == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t cols)
{
    if (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
    else         asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 consecutive 32-bit columns of this thread's tensor-memory lane, waited for.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

template <int KIND>
__device__ __forceinline__ float acc_value(uint32_t v) { return KIND == KIND_I8 ? (float)(int)v : __uint_as_float(v); }

// ---------------------------------------------------------------------------------------------------------------------
// Problem description
// ---------------------------------------------------------------------------------------------------------------------

struct Shape {
    unsigned U, V, K, batch;
    unsigned tilesU, tilesV, tiles;           // tiles: per batch entry (of the lower triangle when tri)
    int tri;                                  // 1: U == V, square tiles, only tiles with tu >= tv; the functor mirrors them
};

// Tile number -> (tu, tv).  Full: groups of GROUP rows of tiles, column by column inside a group, so that the tiles in flight
// share operands in L2.  Triangle: row by row.
constexpr unsigned GROUP = 8;
__host__ __device__ inline void tile_coords(const Shape& s, unsigned t, unsigned& tu, unsigned& tv)
{
    if (s.tri) {
        unsigned r = (unsigned)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
        while (r * (r + 1) / 2 > t) r--;
        while ((r + 1) * (r + 2) / 2 <= t) r++;
        tu = r;
        tv = t - r * (r + 1) / 2;
        return;
    }
    const unsigned per_group = GROUP * s.tilesV, g = t / per_group, first = g * GROUP, left = s.tilesU - first;
    const unsigned rows = left < GROUP ? left : GROUP, r = t - g * per_group;
    tu = first + r % rows;
    tv = r / rows;
}

// ---------------------------------------------------------------------------------------------------------------------
// Epilogue of 32 rows (one per lane) x CH columns held as x[CH] per lane.
//   Epi::kMirror   also stores every value at (v, u) (symmetric results; tiles off the diagonal only)
//   epi.begin()    per thread and tile; returns the factor of this lane's row, applied to the accumulator
//   epi.column()   one value per lane, u contiguous over the lanes: transposed results and mirrored tiles
//   epi.segment()  up to 8 values with consecutive v of one row
//   epi.combine()  transposed results only: what the row contributes besides the accumulator, before column()
// ---------------------------------------------------------------------------------------------------------------------

template <class Epi, int CH>
__device__ __forceinline__ void epilogue_chunk(const Epi& epi, typename Epi::State& st, const Shape& s, float* buf, unsigned z, unsigned u0,
                                               unsigned v0, bool mirror, const float (&x)[CH])
{
    const int lane = threadIdx.x & 31;
    if (epi.transposed() || (Epi::kMirror && mirror)) {
        const unsigned u = u0 + lane;
        if (u < s.U) {
            float y[CH];
#pragma unroll
            for (int j = 0; j < CH; j++) y[j] = x[j];
            if (epi.transposed()) epi.template combine<CH>(st, z, u, v0, s.V, y);
#pragma unroll
            for (int j = 0; j < CH; j++)
                if (v0 + j < s.V) epi.column(st, z, u, v0 + j, y[j]);
        }
        if (epi.transposed()) return;
    }
    if (CH < 32) {                                        // narrow slices: each lane stores its own row
        const unsigned u = u0 + lane;
        if (u < s.U) {
#pragma unroll
            for (int j = 0; j < CH; j += 8) {
                constexpr int W = CH < 8 ? CH : 8;
                float y[8] = {};
#pragma unroll
                for (int i = 0; i < W; i++) y[i] = x[j + i];
                if (v0 + j < s.V) epi.segment(st, z, u, v0 + j, min((unsigned)W, s.V - v0 - j), y);
            }
        }
        return;
    }
    // 32 x 32 through shared memory: 16-byte pieces, piece c of row r at c ^ (r & 7), so that both the row-wise writes and the
    // reads (4 lanes per row, 8 values each) are free of bank conflicts.
    float4* b4 = reinterpret_cast<float4*>(buf);
    __syncwarp();
#pragma unroll
    for (int c = 0; c < CH / 4; c++) b4[lane * 8 + (c ^ (lane & 7))] = make_float4(x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]);
    __syncwarp();
    const unsigned v = v0 + (lane & 3) * 8;
#pragma unroll
    for (int it = 0; it < 4; it++) {
        const int r = it * 8 + lane / 4;
        const unsigned u = u0 + r;
        const float4 a = b4[r * 8 + ((2 * (lane & 3)) ^ (r & 7))], b = b4[r * 8 + ((2 * (lane & 3) + 1) ^ (r & 7))];
        float y[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        if (u < s.U && v < s.V) epi.segment(st, z, u, v, min(8u, s.V - v), y);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Loads and products shared by the two kernels
// ---------------------------------------------------------------------------------------------------------------------

// One slab: BM rows of P, BN / CG rows (or columns, QMN) of Q.
template <int KIND, int BN, int CG, bool QMN>
__device__ __forceinline__ void load_slab(unsigned char* sp, const CUtensorMap* mapP, const CUtensorMap* mapQ, int kt, int u0, int v0, int z, uint32_t bar)
{
    constexpr int BK = KIND == KIND_I8 ? SLAB_BYTES : SLAB_BYTES / 2;
    unsigned char* sq = sp + BM * SLAB_BYTES;
    tma_load_3d<CG>(sp, mapP, kt * BK, u0, z, bar);
    if (QMN) {
#pragma unroll
        for (int b = 0; b < BN / CG / 64; b++) tma_load_3d<CG>(sq + b * 8192, mapQ, v0 + b * 64, kt * BK, z, bar);
    } else {
        tma_load_3d<CG>(sq, mapQ, kt * BK, v0, z, bar);
    }
}

template <int KIND, int BN, int CG, bool QMN>
__device__ __forceinline__ void mma_slab(uint32_t sp, uint32_t tmem_d, bool first)
{
    const uint64_t pd = smem_desc<false>(sp), qd = smem_desc<QMN>(sp + BM * SLAB_BYTES);
    constexpr uint32_t idesc = instr_desc<KIND, BN, CG, QMN>();
#pragma unroll
    for (int ks = 0; ks < 4; ks++)            // 32 bytes along k per instruction; v-contiguous Q: 16 k = 16 rows of 128 bytes
        umma<KIND, CG>(tmem_d, pd + ks * (32 >> 4), qd + ks * (QMN ? (16 * 128) >> 4 : 32 >> 4), idesc, !(first && ks == 0));
}

template <int BN, int CG>
constexpr int stage_bytes() { return (BM + BN / CG) * SLAB_BYTES; }
template <int BN, int CG>
constexpr int persistent_stages()
{
    return (232448 - 1024 - 512 - EPI_WARPS * STAGE_BUF) / stage_bytes<BN, CG>();
}
template <int BN, int CG>
constexpr int persistent_smem() { return persistent_stages<BN, CG>() * stage_bytes<BN, CG>() + EPI_WARPS * STAGE_BUF + 1024 + 512; }

// ---------------------------------------------------------------------------------------------------------------------
// Persistent kernel
// ---------------------------------------------------------------------------------------------------------------------

template <int KIND, int BN, int CG, bool QMN, class Epi>
__global__ void __launch_bounds__(THREADS, 1)
narrow_persistent_kernel(const __grid_constant__ CUtensorMap mapP, const __grid_constant__ CUtensorMap mapQ, const Shape s, const Epi epi)
{
    constexpr int STAGES = persistent_stages<BN, CG>(), STAGE = stage_bytes<BN, CG>();
    constexpr uint32_t TMEM_COLS = 2 * BN < 32 ? 32 : 2 * BN;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* bufs = reinterpret_cast<float*>(smem + STAGES * STAGE);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE + EPI_WARPS * STAGE_BUF);
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;
    uint64_t* acc_empty = acc_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = CG == 2 ? cluster_ctarank() : 0;
    const unsigned group = blockIdx.x / CG, groups = gridDim.x / CG;
    const unsigned total = s.tiles * s.batch;
    const int nk = (int)((s.K + slab_k(KIND) - 1) / slab_k(KIND));

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], CG * EPI_WARPS);
        }
        mbar_fence_init();
        tma_prefetch_descriptor(&mapP);
        tma_prefetch_descriptor(&mapQ);
    }
    if (warp == 1) tmem_alloc<CG>(tmem_slot, TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();

    if (warp == 0) {
        if (lane == 0) {
            unsigned it = 0;
            bool ok = true;
            for (unsigned t = group; t < total && ok; t += groups) {
                unsigned tu, tv;
                const unsigned z = t / s.tiles;
                tile_coords(s, t - z * s.tiles, tu, tv);
                const int u0 = (int)(tu * BM * CG + rank * BM), v0 = (int)(tv * BN + rank * (BN / CG));
                for (int kt = 0; kt < nk; kt++, it++) {
                    const int slot = it % STAGES;
                    if (it >= STAGES && !mbar_wait(&empty[slot], ((it / STAGES) - 1) & 1)) { ok = false; break; }
                    // A pair's loads are all counted on the first CTA's barrier, which expects both halves.
                    uint32_t bar = smem_u32(&full[slot]);
                    if (CG == 2) bar = map_shared(bar, 0);
                    if (rank == 0) mbar_expect_tx(&full[slot], CG * STAGE);
                    load_slab<KIND, BN, CG, QMN>(smem + slot * STAGE, &mapP, &mapQ, kt, u0, v0, (int)z, bar);
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            unsigned it = 0, n = 0;
            bool ok = true;
            for (unsigned t = group; t < total && ok; t += groups, n++) {
                const unsigned a = n & 1;
                if (n >= 2 && !mbar_wait(&acc_empty[a], ((n >> 1) - 1) & 1)) break;
                tc_fence_after();
                for (int kt = 0; kt < nk; kt++, it++) {
                    const int slot = it % STAGES;
                    if (!mbar_wait(&full[slot], (it / STAGES) & 1)) { ok = false; break; }
                    tc_fence_after();
                    mma_slab<KIND, BN, CG, QMN>(smem_u32(smem + slot * STAGE), tmem + a * BN, kt == 0);
                    umma_commit<CG>(&empty[slot]);
                }
                umma_commit<CG>(&acc_full[a]);
            }
        }
    } else {
        const int ew = warp - 2, quarter = warp & 3, half = ew / 4;
        float* buf = bufs + ew * (STAGE_BUF / 4);
        unsigned n = 0;
        for (unsigned t = group; t < total; t += groups, n++) {
            unsigned tu, tv;
            const unsigned z = t / s.tiles;
            tile_coords(s, t - z * s.tiles, tu, tv);
            const unsigned a = n & 1;
            if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[a], (n >> 1) & 1))) break;
            tc_fence_after();
            const unsigned u0 = tu * BM * CG + rank * BM + quarter * 32;
            typename Epi::State st;
            const float factor = epi.begin(st, z, u0 + lane < s.U ? u0 + lane : s.U - 1);
            constexpr int CHUNKS = BN / 32 / 2;               // per half
#pragma unroll 1
            for (int c = 0; c < CHUNKS; c++) {
                const int col = (half * CHUNKS + c) * 32;
                uint32_t r[32];
                tmem_ld32(tmem + ((uint32_t)(32 * quarter) << 16) + a * BN + col, r);
                if (c == CHUNKS - 1) {                        // accumulator read: hand it back
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (CG == 2) mbar_arrive_cluster(map_shared(smem_u32(&acc_empty[a]), 0));
                        else mbar_arrive(&acc_empty[a]);
                    }
                }
                float x[32];
#pragma unroll
                for (int j = 0; j < 32; j++) x[j] = factor * acc_value<KIND>(r[j]);
                epilogue_chunk<Epi, 32>(epi, st, s, buf, z, u0, tv * BN + col, s.tri && tu != tv, x);
            }
            epi.end(st, z, t);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync();
    tc_fence_after();
    if (warp == 1) tmem_free<CG>(tmem, TMEM_COLS);
}

// ---------------------------------------------------------------------------------------------------------------------
// Split kernel: one tile per cluster, the slabs of k shared out over its CTAs
// ---------------------------------------------------------------------------------------------------------------------

// Two CTAs per SM for the narrow tiles (decoding: the loads of one run under the start and the end of the other), one for BN = 128.
template <int BN>
constexpr int split_stages() { return BN == 32 ? 5 : BN == 64 ? 4 : 6; }
template <int BN>
constexpr int split_smem() { return split_stages<BN>() * stage_bytes<BN, 1>() + 1024 + 256; }

template <int KIND, int BN, int S, bool QMN, class Epi>
__global__ void __launch_bounds__(THREADS)
narrow_split_kernel(const __grid_constant__ CUtensorMap mapP, const __grid_constant__ CUtensorMap mapQ, const Shape s, const Epi epi)
{
    constexpr int STAGES = split_stages<BN>(), STAGE = stage_bytes<BN, 1>();
    constexpr uint32_t TMEM_COLS = BN;
    constexpr int SL = BN / S;                                    // columns each rank sums and finishes
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    // The ring is free once the products of every CTA of the cluster are done: the partial sums and the store buffers use it again.
    uint32_t* part = reinterpret_cast<uint32_t*>(smem);                                // [S][SL][BM], written by all ranks
    float* bufs = reinterpret_cast<float*>(smem + BN * BM * 4);
    static_assert(BN * BM * 4 + EPI_WARPS * STAGE_BUF <= STAGES * STAGE, "the ring holds the partial sums and the store buffers");
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE);
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = S > 1 ? cluster_ctarank() : 0;
    const unsigned t = blockIdx.x / S, z = t / s.tiles;
    unsigned tu, tv;
    tile_coords(s, t - z * s.tiles, tu, tv);
    const int nk = (int)((s.K + slab_k(KIND) - 1) / slab_k(KIND));
    const int k0 = (int)((long long)nk * rank / S), k1 = (int)((long long)nk * (rank + 1) / S);   // the host keeps S <= nk

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        mbar_init(acc_full, 1);
        mbar_fence_init();
        tma_prefetch_descriptor(&mapP);
        tma_prefetch_descriptor(&mapQ);
    }
    if (warp == 1) tmem_alloc<1>(tmem_slot, TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();

    if (warp == 0) {
        if (lane == 0) {
            for (int i = 0; i < k1 - k0; i++) {
                const int slot = i % STAGES;
                if (i >= STAGES && !mbar_wait(&empty[slot], ((i / STAGES) - 1) & 1)) break;
                mbar_expect_tx(&full[slot], STAGE);
                load_slab<KIND, BN, 1, QMN>(smem + slot * STAGE, &mapP, &mapQ, k0 + i, (int)(tu * BM), (int)(tv * BN), (int)z, smem_u32(&full[slot]));
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            for (int i = 0; i < k1 - k0; i++) {
                const int slot = i % STAGES;
                if (!mbar_wait(&full[slot], (i / STAGES) & 1)) break;
                tc_fence_after();
                mma_slab<KIND, BN, 1, QMN>(smem_u32(smem + slot * STAGE), tmem, i == 0);
                umma_commit<1>(&empty[slot]);
            }
            umma_commit<1>(acc_full);
        }
    }
    const int ew = warp - 2, quarter = warp & 3, half = ew / 4;
    const unsigned u0 = tu * BM + quarter * 32;
    const bool mirror = s.tri && tu != tv;
    typename Epi::State st;
    float factor = 0.f;
    bool ok = true;
    if (warp >= 2) {
        factor = epi.begin(st, z, u0 + lane < s.U ? u0 + lane : s.U - 1);
        ok = __all_sync(0xffffffffu, mbar_wait(acc_full, 0));
        tc_fence_after();
    }
    __syncwarp();
    if (S > 1) cluster_sync();                                    // the products of all CTAs of the cluster are done
    if (warp >= 2) {
        if (ok) {
            constexpr int CHUNKS = BN / 32;
#pragma unroll 1
            for (int c = half; c < CHUNKS; c += 2) {
                uint32_t r[32];
                tmem_ld32(tmem + ((uint32_t)(32 * quarter) << 16) + c * 32, r);
                if (S == 1) {
                    float x[32];
#pragma unroll
                    for (int j = 0; j < 32; j++) x[j] = factor * acc_value<KIND>(r[j]);
                    epilogue_chunk<Epi, 32>(epi, st, s, bufs + ew * (STAGE_BUF / 4), z, u0, tv * BN + c * 32, mirror, x);
                } else {
#pragma unroll
                    for (int j = 0; j < 32; j++) {
                        const int col = c * 32 + j, owner = col / SL;
                        const uint32_t local = smem_u32(part + ((rank * SL + col % SL) * BM + quarter * 32 + lane));
                        st_cluster(map_shared(local, (uint32_t)owner), r[j]);
                    }
                }
            }
        }
    }
    if (S > 1) {
        __syncwarp();
        cluster_sync();
        if (warp >= 2 && ok) {
            // columns of this rank's slice, CH at a time; the two warps of a quarter take turns
            constexpr int CH = SL < 32 ? SL : 32;
#pragma unroll 1
            for (int c = half; c < SL / CH; c += 2) {
                float x[CH];
#pragma unroll
                for (int j = 0; j < CH; j++) {
                    const uint32_t* p = part + (c * CH + j) * BM + quarter * 32 + lane;
                    if (KIND == KIND_I8) {
                        int a = 0;
#pragma unroll
                        for (int q = 0; q < S; q++) a += (int)p[q * SL * BM];
                        x[j] = factor * (float)a;
                    } else {
                        float a = 0.f;
#pragma unroll
                        for (int q = 0; q < S; q++) a += __uint_as_float(p[q * SL * BM]);
                        x[j] = factor * a;
                    }
                }
                epilogue_chunk<Epi, CH>(epi, st, s, bufs + ew * (STAGE_BUF / 4), z, u0, tv * BN + rank * SL + c * CH, mirror, x);
            }
        }
    }
    if (warp >= 2 && ok) epi.end(st, z, t);
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_free<1>(tmem, TMEM_COLS);
}

// ---------------------------------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------------------------------

// 3-D map (inner, rows, batch) of 8- or 16-bit elements; boxes of 128 bytes x box_rows, SWIZZLE_128B, zeros out of bounds.
inline bool make_map(CUtensorMap* map, int kind, const void* base, size_t inner, size_t rows, size_t batch, size_t ld, size_t stride, unsigned box_rows)
{
    void* enc = get_tensor_map_encoder();
    if (!enc) return false;
    const size_t es = kind == KIND_I8 ? 1 : 2;
    cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)rows, (cuuint64_t)batch};
    cuuint64_t strides[2] = {(cuuint64_t)(ld * es), (cuuint64_t)((batch > 1 ? stride : ld * rows) * es)};
    cuuint32_t box[3] = {(cuuint32_t)slab_k(kind), box_rows, 1}, estr[3] = {1, 1, 1};
    return reinterpret_cast<TensorMapEncodeTiledFn>(enc)(
               map, kind == KIND_I8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims, strides, box,
               estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// An operand as the kernels read it: `rows` lines of `inner` contiguous elements per batch entry.
struct Operand {
    const void* base;
    size_t inner, rows, ld, stride;
};

inline void set_tiles(Shape& s, unsigned bu, unsigned bv)
{
    s.tilesU = (s.U + bu - 1) / bu;
    s.tilesV = (s.V + bv - 1) / bv;
    s.tiles = s.tri ? s.tilesU * (s.tilesU + 1) / 2 : s.tilesU * s.tilesV;
}

template <typename Kernel, typename Epi>
cudaError_t launch(Kernel kernel, unsigned grid, unsigned cluster, int smem, cudaStream_t st, const CUtensorMap& mp, const CUtensorMap& mq,
                   const Shape& s, const Epi& epi)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, mp, mq, s, epi);
    if (e == cudaSuccess) count_launch();
    return e;
}

template <int KIND, int BN, int CG, bool QMN, class Epi>
cudaError_t run_persistent(const Operand& p, const Operand& q, Shape s, const Epi& epi, cudaStream_t st)
{
    auto kernel = narrow_persistent_kernel<KIND, BN, CG, QMN, Epi>;
    constexpr int smem = persistent_smem<BN, CG>();
    static DeviceOnce once;
    cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    if (e != cudaSuccess) return e;
    CUtensorMap mp, mq;
    if (!make_map(&mp, KIND, p.base, p.inner, p.rows, s.batch, p.ld, p.stride, BM) ||
        !make_map(&mq, KIND, q.base, q.inner, q.rows, s.batch, q.ld, q.stride, QMN ? slab_k(KIND) : BN / CG))
        return cudaErrorNotSupported;
    set_tiles(s, BM * CG, BN);
    const unsigned slots = (unsigned)sm_count() / CG, work = s.tiles * s.batch;
    return launch(kernel, CG * (work < slots ? work : slots), CG, smem, st, mp, mq, s, epi);
}

template <int KIND, int BN, int S, bool QMN, class Epi>
cudaError_t run_split(const Operand& p, const Operand& q, Shape s, const Epi& epi, cudaStream_t st)
{
    auto kernel = narrow_split_kernel<KIND, BN, S, QMN, Epi>;
    constexpr int smem = split_smem<BN>();
    static DeviceOnce once;
    cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    if (e != cudaSuccess) return e;
    CUtensorMap mp, mq;
    if (!make_map(&mp, KIND, p.base, p.inner, p.rows, s.batch, p.ld, p.stride, BM) ||
        !make_map(&mq, KIND, q.base, q.inner, q.rows, s.batch, q.ld, q.stride, QMN ? slab_k(KIND) : BN))
        return cudaErrorNotSupported;
    set_tiles(s, BM, BN);
    return launch(kernel, s.tiles * s.batch * S, S, smem, st, mp, mq, s, epi);
}

// How a product of more than 64 columns runs.  Estimated clocks: rounds of tiles times (slabs x clocks per slab + what a tile costs besides).
//   pairs:  256 x 256 tiles on pairs of CTAs, 512 clocks per slab
//   single: 128 x 128 tiles, persistent, 300 clocks per slab (both operands are read from shared memory at its full rate)
//   split:  128 x 128 tiles, k over S CTAs of a cluster
struct Plan { bool pairs; unsigned split; };         // split == 0: persistent
inline Plan choose_plan(unsigned U, unsigned V, unsigned K, unsigned batch, int tri, int kind)
{
    const double sms = sm_count(), nk = (K + slab_k(kind) - 1) / slab_k(kind);
    auto tiles = [&](unsigned b) {
        const double tu = (U + b - 1) / b, tv = (V + b - 1) / b;
        return batch * (tri ? tu * (tu + 1) / 2 : tu * tv);
    };
    auto rounds = [](double work, double slots) { const double r = work / slots; return (double)(unsigned long long)r + (r > (double)(unsigned long long)r); };
    Plan best{true, 0};
    double least = rounds(tiles(256), (double)((int)sms / 2)) * (nk * 512 + 500) + 4000;
    const double t128 = tiles(128), single = rounds(t128, sms) * (nk * 300 + 500) + 3000;
    if (single < least) { least = single; best = {false, 0}; }
    for (unsigned s = 1; s <= 8 && s <= nk; s *= 2) {
        const double c = rounds(t128 * s, sms) * ((double)(((unsigned)nk + s - 1) / s) * 300 + 3000 + (s > 1 ? 1500 : 0));
        if (c < least) { least = c; best = {false, s}; }
    }
    return best;
}

template <int KIND, int BN, bool QMN, class Epi>
cudaError_t run_split_by(unsigned split, const Operand& p, const Operand& q, const Shape& s, const Epi& epi, cudaStream_t st)
{
    switch (split) {
        case 8: return run_split<KIND, BN, 8, QMN, Epi>(p, q, s, epi, st);
        case 4: return run_split<KIND, BN, 4, QMN, Epi>(p, q, s, epi, st);
        case 2: return run_split<KIND, BN, 2, QMN, Epi>(p, q, s, epi, st);
        default: return run_split<KIND, BN, 1, QMN, Epi>(p, q, s, epi, st);
    }
}

template <int KIND, bool QMN, class Epi>
cudaError_t run_planned(const Operand& p, const Operand& q, const Shape& s, const Epi& epi, cudaStream_t st)
{
    const Plan plan = choose_plan(s.U, s.V, s.K, s.batch, s.tri, KIND);
    if (plan.pairs) return run_persistent<KIND, 256, 2, QMN, Epi>(p, q, s, epi, st);
    if (plan.split == 0) return run_persistent<KIND, 128, 1, QMN, Epi>(p, q, s, epi, st);
    return run_split_by<KIND, 128, QMN, Epi>(plan.split, p, q, s, epi, st);
}

}  // namespace narrow
}  // namespace cb200
