// Tensor-core tile engine of the narrow-type operators (8-bit products with scales, FP16 products of the Newton-Schulz
// orthogonalisation).  Both are  D[u, v] = sum_k P[u, k] * Q[v, k]  with P stored U x K and Q stored V x K, k contiguous (or, for Q, v contiguous:
// the MN-major form of the instruction); the epilogue is a functor.
//
// narrow_persistent_kernel: pairs of CTAs (tcgen05.mma.cta_group::2, one CTA per SM) walk over output tiles of 256 rows.  10 warps: warp
// 0 loads slabs of 128 bytes along k with TMA into a ring, warp 1 owns tensor memory and issues the MMAs, warps 2-9 are the
// epilogue.  Two accumulators in tensor memory, so the epilogue of a tile runs under the products of the next.  Bound by what L2
// feeds the SMs (about 13 TB/s measured; a 256 x 256 tile moves 64 KB per slab) and, over seconds, by the power cap: 8-bit 8192^3
// 318 to 354 us alone, 397 to 412 us back to back (cuBLAS on the same GPU 377 and 439); FP16 gram product 4096 x 16384 182 to 205 us.
//
// narrow_split_kernel: for products with fewer tiles than SMs.  The k range of a tile is cut over the CTAs of a cluster; the
// partial accumulators meet in distributed shared memory (each rank sums a slice of the columns, in rank order, so
// results do not depend on timing), then the same epilogue runs on the slices.  No workspace, no second launch.  Bound by latency
// (launch 2 us, first load 0.7, barriers and exchange 2, epilogue 1) or, for few tokens, by reading the weights.
//
// Every wait on an mbarrier is bounded (tma_pipeline.cuh).  A CTA whose wait ran out leaves its loops and still takes part in
// the cluster barriers, so its peers end too.
#pragma once

#include "common.h"
#include "tma_pipeline.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

namespace cb200 {
namespace narrow {

enum Kind { KIND_F16 = 0, KIND_I8 = 1 };

constexpr int BM = 128;                       // rows of P per CTA = lanes of tensor memory
constexpr int SLAB_BYTES = 128;               // bytes along k per slab: one SWIZZLE_128B row
constexpr int EPI_WARPS = 8;
constexpr int THREADS = (2 + EPI_WARPS) * 32;

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
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync()
{
    cluster_arrive();
    cluster_wait();
}
// Address of `saddr` (this CTA's shared memory) in the shared memory of CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_shared(uint32_t saddr, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v, uint32_t w)
{
    asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(addr), "r"(v), "r"(w) : "memory");
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

// 16 rows x 32 columns of 32-bit accumulators as the fragments of 8 x 8 blocks: lane t holds, for column group k, row t / 4 columns
// 8 k + 2 (t % 4) + {0, 1} in v[4 k + {0, 1}] and row t / 4 + 8 of the same columns in v[4 k + {2, 3}].  The warp has to be converged.
__device__ __forceinline__ void tmem_ld_16x32(uint32_t taddr, uint32_t (&v)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

template <int KIND>
__device__ __forceinline__ float acc_value(uint32_t v) { return KIND == KIND_I8 ? (float)(int)v : __uint_as_float(v); }

// ---------------------------------------------------------------------------------------------------------------------
// Problem description
// ---------------------------------------------------------------------------------------------------------------------

struct Shape {
    unsigned U, V, K, batch;
    unsigned tilesU, tilesV, tiles;           // tiles: per batch entry (of the lower triangle when tri)
    int tri;                                  // 1: U == V, symmetric: square tiles, those that touch the lower triangle only
};

// What becomes of a chunk: its 128 x 128 block lies below the diagonal (stored at both places), on it, or above (in a 256 x 256 tile on
// the diagonal; not stored).
enum Part { PART_PLAIN = 0, PART_BELOW = 1, PART_ABOVE = -1 };
__device__ __forceinline__ int part_of(const Shape& s, unsigned u0, unsigned v0)
{
    if (!s.tri) return PART_PLAIN;
    const unsigned bu = u0 / 128, bv = v0 / 128;
    return bu > bv ? PART_BELOW : bu < bv ? PART_ABOVE : PART_PLAIN;
}

// Tile number -> (tu, tv).  Full: groups of GROUP rows of tiles, column by column inside a group, so that the tiles in flight
// share operands in L2.  Triangle: row by row.
constexpr unsigned GROUP = 8;
__host__ __device__ inline void tile_coords(const Shape& s, unsigned t, unsigned& tu, unsigned& tv)
{
    if (s.tri) {                              // row r has r + 1 tiles
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
// Epilogue.  A warp finishes chunks of 32 rows x 8 G columns, held as fragments x[g][k][e]: row 8 g + lane / 4, column
// 8 k + 2 (lane % 4) + e.  What a functor has:
//   kHeavy        reads as much as it writes (for choose_plan)
//   kTriangle     of symmetric products (Shape::tri)
//   begin()       per thread and tile; u0, v0: where the warp's first chunk begins (of all its tiles one warp has both 0)
//   Pre, fetch()  what a chunk needs besides the accumulators, requested one chunk ahead
//   chunk()       computes and stores (where: part_of()); requests the next chunk's (at column v_next, ~0u: none) as soon as its own is used
//   end()         per thread and tile
//
// Nothing goes through shared memory: its bandwidth is what the products and the loads that feed them use up (both sides
// together 128 bytes per clock), and an epilogue that staged its chunks there ran at a fifth of its speed beside them.
// Rows are put together by exchanges among the four lanes that share one (quad_transpose), columns by transposing 8 x 8 blocks
// (movmatrix); 16-bit results leave as 16 bytes a lane, 64 bytes a row.
// ---------------------------------------------------------------------------------------------------------------------

// r[k] of lane j of a quad becomes r[j] of lane k.
__device__ __forceinline__ void quad_transpose(uint32_t (&r)[4])
{
    const bool o1 = threadIdx.x & 1, o2 = threadIdx.x & 2;
    uint32_t a = __shfl_xor_sync(0xffffffffu, o1 ? r[0] : r[1], 1), b = __shfl_xor_sync(0xffffffffu, o1 ? r[2] : r[3], 1);
    if (o1) { r[0] = a; r[2] = b; } else { r[1] = a; r[3] = b; }
    a = __shfl_xor_sync(0xffffffffu, o2 ? r[0] : r[2], 2);
    b = __shfl_xor_sync(0xffffffffu, o2 ? r[1] : r[3], 2);
    if (o2) { r[0] = a; r[1] = b; } else { r[2] = a; r[3] = b; }
}
// Transposes an 8 x 8 block of 16-bit values held as fragments.
__device__ __forceinline__ uint32_t block_transpose(uint32_t v)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// 16-bit matrices (as raw bits): a lane's share of a chunk, by rows (16 bytes per 8 rows) or by fragments.
// `align`: bytes by which base and pitch are aligned, 16, 4 or 2; PADDED: 16, and a line may be read and written up to the next
// multiple of 8 elements.  Below 16, at the edge of a matrix that is not padded and for chunks narrower than 32 columns fragments are
// accessed directly, 4 or 2 bytes a lane.
constexpr int PADDED = 32;
template <int G>
struct Bits16 {
    uint32_t h[4][G];                                       // [g][k]: two values of row 8 g + lane / 4, columns 8 k + 2 (lane % 4)
};

template <int G>
__device__ __forceinline__ void load_rows16(Bits16<G>& f, const uint16_t* base, size_t ld, unsigned u0, unsigned v0, unsigned U, unsigned V, int align)
{
    const int lane = threadIdx.x & 31, q = lane & 3;
    const unsigned u = u0 + lane / 4;
    if (G == 4 && (align == PADDED || (align == 16 && v0 + 32 <= V))) {
        const uint16_t* p = base + (size_t)u * ld + v0 + 8 * q;
        if (v0 + 8 * q >= V) return;
#pragma unroll
        for (int g = 0; g < 4; g++, p += 8 * ld)
            if (u + 8 * g < U) *reinterpret_cast<uint4*>(f.h[g]) = *reinterpret_cast<const uint4*>(p);
    } else {
        const uint16_t* p = base + (size_t)u * ld + v0 + 2 * q;
#pragma unroll
        for (int g = 0; g < 4; g++, p += 8 * ld) {
            if (u + 8 * g >= U) continue;
#pragma unroll
            for (int k = 0; k < G; k++) {
                const unsigned v = v0 + 8 * k + 2 * q;
                if (align >= 4 && v + 2 <= V) f.h[g][k] = *reinterpret_cast<const uint32_t*>(p + 8 * k);
                else f.h[g][k] = (v < V ? p[8 * k] : 0u) | (v + 1 < V ? (uint32_t)p[8 * k + 1] << 16 : 0u);
            }
        }
    }
}
// What load_rows16 brought by rows, as fragments (all lanes of the warp).
template <int G>
__device__ __forceinline__ void rows_to_fragments(Bits16<G>& f, unsigned v0, unsigned V, int align)
{
    if constexpr (G == 4) {
        if (align == PADDED || (align == 16 && v0 + 32 <= V)) {
#pragma unroll
            for (int g = 0; g < 4; g++) quad_transpose(f.h[g]);
        }
    }
}
template <int G>
__device__ __forceinline__ void store_rows16(Bits16<G>& f, uint16_t* base, size_t ld, unsigned u0, unsigned v0, unsigned U, unsigned V, int align)
{
    const int lane = threadIdx.x & 31, q = lane & 3;
    const unsigned u = u0 + lane / 4;
    if constexpr (G == 4) {
        if (align == PADDED || (align == 16 && v0 + 32 <= V)) {
            uint16_t* p = base + (size_t)u * ld + v0 + 8 * q;
#pragma unroll
            for (int g = 0; g < 4; g++, p += 8 * ld) {
                quad_transpose(f.h[g]);
                if (u + 8 * g < U && v0 + 8 * q < V) *reinterpret_cast<uint4*>(p) = make_uint4(f.h[g][0], f.h[g][1], f.h[g][2], f.h[g][3]);
            }
            return;
        }
    }
    uint16_t* p = base + (size_t)u * ld + v0 + 2 * q;
#pragma unroll
    for (int g = 0; g < 4; g++, p += 8 * ld) {
        if (u + 8 * g >= U) continue;
#pragma unroll
        for (int k = 0; k < G; k++) {
            const unsigned v = v0 + 8 * k + 2 * q;
            if (align >= 4 && v + 2 <= V) *reinterpret_cast<uint32_t*>(p + 8 * k) = f.h[g][k];
            else {
                if (v < V) p[8 * k] = (uint16_t)f.h[g][k];
                if (v + 1 < V) p[8 * k + 1] = (uint16_t)(f.h[g][k] >> 16);
            }
        }
    }
}
// The chunk transposed: 8 G lines of 32 values.  Blocks are transposed here; the lines v run over k, and the 32 rows u along a line.
template <int G>
__device__ __forceinline__ void store_columns16(const Bits16<G>& f, uint16_t* base, size_t ld, unsigned u0, unsigned v0, unsigned U, unsigned V, int align)
{
    const int lane = threadIdx.x & 31, q = lane & 3;
    const unsigned v = v0 + lane / 4;
#pragma unroll
    for (int k = 0; k < G; k++) {
        uint32_t r[4];
#pragma unroll
        for (int g = 0; g < 4; g++) r[g] = block_transpose(f.h[g][k]);
        uint16_t* p = base + (size_t)(v + 8 * k) * ld + u0;
        if (align == PADDED || (align == 16 && u0 + 32 <= U)) {
            quad_transpose(r);
            if (v + 8 * k < V && u0 + 8 * q < U) *reinterpret_cast<uint4*>(p + 8 * q) = make_uint4(r[0], r[1], r[2], r[3]);
        } else if (v + 8 * k < V) {
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const unsigned u = u0 + 8 * g + 2 * q;
                if (align >= 4 && u + 2 <= U) *reinterpret_cast<uint32_t*>(p + 8 * g + 2 * q) = r[g];
                else {
                    if (u < U) p[8 * g + 2 * q] = (uint16_t)r[g];
                    if (u + 1 < U) p[8 * g + 2 * q + 1] = (uint16_t)(r[g] >> 16);
                }
            }
        }
    }
}
// The counterpart: reads what store_columns16 would overwrite, as fragments of blocks that are still transposed.
template <int G>
__device__ __forceinline__ void load_columns16(Bits16<G>& f, const uint16_t* base, size_t ld, unsigned u0, unsigned v0, unsigned U, unsigned V, int align)
{
    const int lane = threadIdx.x & 31, q = lane & 3;
    const unsigned v = v0 + lane / 4;
#pragma unroll
    for (int k = 0; k < G; k++) {
        const uint16_t* p = base + (size_t)(v + 8 * k) * ld + u0 + 2 * q;
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const unsigned u = u0 + 8 * g + 2 * q;
            if (v + 8 * k >= V) f.h[g][k] = 0;
            else if (align >= 4 && u + 2 <= U) f.h[g][k] = *reinterpret_cast<const uint32_t*>(p + 8 * g);
            else f.h[g][k] = (u < U ? p[8 * g] : 0u) | (u + 1 < U ? (uint32_t)p[8 * g + 1] << 16 : 0u);
        }
    }
}
template <int G>
__device__ __forceinline__ void columns_to_fragments(Bits16<G>& f)
{
#pragma unroll
    for (int g = 0; g < 4; g++)
#pragma unroll
        for (int k = 0; k < G; k++) f.h[g][k] = block_transpose(f.h[g][k]);
}

// Bytes by which lines of 16-bit elements are aligned.
inline int line_alignment(const void* base, size_t ld, size_t stride)
{
    const uintptr_t a = reinterpret_cast<uintptr_t>(base) | (uintptr_t)(ld * 2) | (uintptr_t)(stride * 2);
    return (a & 15) == 0 ? 16 : (a & 3) == 0 ? 4 : 2;
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

// 32 x 32 accumulators at a tensor-memory address (lane, column), as numbers.
template <int KIND>
__device__ __forceinline__ void read_chunk(float (&x)[4][4][2], uint32_t taddr)
{
    uint32_t a[16], b[16];
    __syncwarp();
    tmem_ld_16x32(taddr, a);
    tmem_ld_16x32(taddr + (16u << 16), b);
    tmem_ld_wait();
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            x[0][k][e] = acc_value<KIND>(a[4 * k + e]);
            x[1][k][e] = acc_value<KIND>(a[4 * k + 2 + e]);
            x[2][k][e] = acc_value<KIND>(b[4 * k + e]);
            x[3][k][e] = acc_value<KIND>(b[4 * k + 2 + e]);
        }
}

template <int BN, int CG>
constexpr int stage_bytes() { return (BM + BN / CG) * SLAB_BYTES; }
template <int BN>
constexpr int persistent_stages() { return (232448 - 1024 - 512) / stage_bytes<BN, 2>(); }
template <int BN>
constexpr int persistent_smem() { return persistent_stages<BN>() * stage_bytes<BN, 2>() + 1024 + 512; }

// ---------------------------------------------------------------------------------------------------------------------
// Persistent kernel
// ---------------------------------------------------------------------------------------------------------------------

template <int KIND, int BN, bool QMN, class Epi>
__global__ void __launch_bounds__(THREADS, 1)
narrow_persistent_kernel(const __grid_constant__ CUtensorMap mapP, const __grid_constant__ CUtensorMap mapQ, const Shape s, const Epi epi)
{
    constexpr int CG = 2, STAGES = persistent_stages<BN>(), STAGE = stage_bytes<BN, CG>();
    constexpr uint32_t TMEM_COLS = 2 * BN > 256 ? 512 : 256;          // two accumulators; a power of two
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE);
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;
    uint64_t* acc_empty = acc_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = cluster_ctarank();
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
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();
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
                    const uint32_t bar = map_shared(smem_u32(&full[slot]), 0);
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
        const int quarter = warp & 3, half = (warp - 2) / 4;
        unsigned n = 0;
        for (unsigned t = group; t < total; t += groups, n++) {
            unsigned tu, tv;
            const unsigned z = t / s.tiles;
            tile_coords(s, t - z * s.tiles, tu, tv);
            const unsigned a = n & 1;
            const unsigned u0 = tu * BM * CG + rank * BM + quarter * 32;
            constexpr int CHUNKS = BN / 32 / 2;               // per half
            const unsigned v0 = tv * BN + half * CHUNKS * 32;
            typename Epi::State st;
            epi.begin(st, s, z, u0, v0);
            typename Epi::template Pre<4> pre;
            epi.fetch(pre, s, z, u0, v0);
            if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[a], (n >> 1) & 1))) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < CHUNKS; c++) {
                float x[4][4][2];
                read_chunk<KIND>(x, tmem + ((uint32_t)(32 * quarter) << 16) + a * BN + (half * CHUNKS + c) * 32);
                if (c == CHUNKS - 1) {                        // accumulator read: hand it back
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(map_shared(smem_u32(&acc_empty[a]), 0));
                }
                epi.chunk(st, pre, s, z, u0, v0 + c * 32, c + 1 < CHUNKS ? v0 + (c + 1) * 32 : ~0u, part_of(s, u0, v0 + c * 32), x);
            }
            epi.end(st, z, t);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    if (warp == 1) tmem_free<CG>(tmem, TMEM_COLS);
}

// ---------------------------------------------------------------------------------------------------------------------
// Split kernel: one tile per cluster, the slabs of k shared out over its CTAs
// ---------------------------------------------------------------------------------------------------------------------

// Two CTAs per SM for the narrow tiles (decoding: the loads of one run under the start and the end of the other), one for BN = 128.
// The partial sums have a place of their own beside the ring, so that a CTA may receive them while its products still run.
template <int BN, int S>
constexpr int split_part() { return S == 1 ? 0 : BN * BM * 4 * (S > BN / 8 ? S * 8 / BN : 1); }
template <int BN, int S>
constexpr int split_stages() { return BN == 128 ? (S == 1 ? 6 : 4) : ((232448 - 2048) / 2 - 1280 - split_part<BN, S>()) / stage_bytes<BN, 1>(); }
template <int BN, int S>
constexpr int split_smem() { return split_stages<BN, S>() * stage_bytes<BN, 1>() + split_part<BN, S>() + 1024 + 256; }

template <int KIND, int BN, int S, bool QMN, class Epi>
__global__ void __launch_bounds__(THREADS)
narrow_split_kernel(const __grid_constant__ CUtensorMap mapP, const __grid_constant__ CUtensorMap mapQ, const Shape s, const Epi epi)
{
    constexpr int STAGES = split_stages<BN, S>(), STAGE = stage_bytes<BN, 1>();
    constexpr uint32_t TMEM_COLS = BN;
    // Column groups of 8 that a rank sums and finishes; with S > BN / 8 the last ranks have none.
    constexpr int GROUPS = BN / 8, OWNERS = S < GROUPS ? S : GROUPS, OWN = GROUPS / OWNERS;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    // Partial sums as fragments: [S ranks][4 quarters][OWN groups][4 g][32 lanes] pairs.
    uint2* part = reinterpret_cast<uint2*>(smem + STAGES * STAGE);
    static_assert(S == 1 || S * OWN * 8 * BM * 4 == split_part<BN, S>(), "size of the partial sums");
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE + split_part<BN, S>());
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
    __syncwarp();
    if (S > 1) cluster_arrive();                                  // waited for before this CTA writes to the others: by then they run
    if (warp == 1) tmem_alloc<1>(tmem_slot, TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();
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
    const int quarter = warp & 3, half = (warp - 2) / 4;
    const unsigned u0 = tu * BM + quarter * 32;
    const int where = part_of(s, u0, tv * BN);
    typename Epi::State st;
    // The columns this warp finishes: chunks of G groups, every second one (the two warps of a quarter take turns).
    constexpr int G = OWN < 4 ? OWN : 4;
    const unsigned v_own = tv * BN + rank * (OWN * 8) + half * (G * 8);
    const bool finishes = warp >= 2 && rank < OWNERS && half < OWN / G;
    typename Epi::template Pre<G> pre;
    bool ok = true;
    if (warp >= 2) {
        epi.begin(st, s, z, u0, v_own);
        if (finishes) epi.fetch(pre, s, z, u0, v_own);
        ok = __all_sync(0xffffffffu, mbar_wait(acc_full, 0));
        tc_fence_after();
    }
    __syncwarp();
    if (S > 1) cluster_wait();
    if (warp >= 2 && ok) {
#pragma unroll 1
        for (int c = half; c < BN / 32; c += 2) {
            const uint32_t taddr = tmem + ((uint32_t)(32 * quarter) << 16) + c * 32;
            if constexpr (S == 1) {
                float x[4][4][2];
                read_chunk<KIND>(x, taddr);
                epi.chunk(st, pre, s, z, u0, tv * BN + c * 32, c + 2 < BN / 32 ? tv * BN + (c + 2) * 32 : ~0u, where, x);
            } else {
                uint32_t a[16], b[16];
                __syncwarp();
                tmem_ld_16x32(taddr, a);
                tmem_ld_16x32(taddr + (16u << 16), b);
                tmem_ld_wait();
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int group = c * 4 + k;
                    const uint32_t to = map_shared(smem_u32(part + (((rank * 4 + quarter) * OWN + group % OWN) * 4) * 32 + lane), group / OWN);
                    st_cluster(to, a[4 * k], a[4 * k + 1]);
                    st_cluster(to + 256, a[4 * k + 2], a[4 * k + 3]);
                    st_cluster(to + 512, b[4 * k], b[4 * k + 1]);
                    st_cluster(to + 768, b[4 * k + 2], b[4 * k + 3]);
                }
            }
        }
    }
    if (S > 1) {
        __syncwarp();
        cluster_sync();
        if (finishes && ok) {
#pragma unroll 1
            for (int c = half; c < OWN / G; c += 2) {
                const unsigned v0 = tv * BN + rank * (OWN * 8) + c * (G * 8);
                float x[4][G][2];
#pragma unroll
                for (int k = 0; k < G; k++)
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        const uint2* p = part + ((quarter * OWN + c * G + k) * 4 + g) * 32 + lane;
                        if (KIND == KIND_I8) {
                            int i0 = 0, i1 = 0;
#pragma unroll
                            for (int q = 0; q < S; q++) { const uint2 w = p[q * 4 * OWN * 4 * 32]; i0 += (int)w.x; i1 += (int)w.y; }
                            x[g][k][0] = (float)i0; x[g][k][1] = (float)i1;
                        } else {
                            float f0 = 0.f, f1 = 0.f;
#pragma unroll
                            for (int q = 0; q < S; q++) { const uint2 w = p[q * 4 * OWN * 4 * 32]; f0 += __uint_as_float(w.x); f1 += __uint_as_float(w.y); }
                            x[g][k][0] = f0; x[g][k][1] = f1;
                        }
                    }
                epi.chunk(st, pre, s, z, u0, v0, c + 2 < OWN / G ? v0 + 2 * G * 8 : ~0u, where, x);
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
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    // The kernel may start (barriers, tensor memory, descriptors) while the one before it on the stream drains, and waits for it in
    // pdl_wait(); it lets its own successor do so from its start on.  One 256 x 1024 orthogonalisation, 17 launches: 170 -> 113 us; 48 x
    // 8192 x 8192 products in a row: 17.3 -> 16.1 us each.
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, mp, mq, s, epi);
    if (e == cudaSuccess) count_launch();
    return e;
}

// Name of the plan of the calling thread's last product (for clblasB200LastGemmVariant).
inline const char*& last_plan()
{
    static thread_local const char* name = "";
    return name;
}
constexpr const char* plan_name(int bn, int split)        // split 0: pairs
{
    if (split == 0) return bn == 256 ? "pairs256" : bn == 192 ? "pairs192" : "pairs128";
    if (bn == 32) return split == 1 ? "split32x1" : split == 2 ? "split32x2" : split == 4 ? "split32x4" : "split32x8";
    if (bn == 64) return split == 1 ? "split64x1" : split == 2 ? "split64x2" : split == 4 ? "split64x4" : "split64x8";
    return split == 1 ? "split128x1" : split == 2 ? "split128x2" : "split128x4";
}

template <int KIND, int BN, bool QMN, class Epi>
cudaError_t run_persistent(const Operand& p, const Operand& q, Shape s, const Epi& epi, cudaStream_t st)
{
    constexpr int CG = 2;
    auto kernel = narrow_persistent_kernel<KIND, BN, QMN, Epi>;
    constexpr int smem = persistent_smem<BN>();
    static DeviceOnce once;
    cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    if (e != cudaSuccess) return e;
    CUtensorMap mp, mq;
    if (!make_map(&mp, KIND, p.base, p.inner, p.rows, s.batch, p.ld, p.stride, BM) ||
        !make_map(&mq, KIND, q.base, q.inner, q.rows, s.batch, q.ld, q.stride, QMN ? slab_k(KIND) : BN / CG))
        return cudaErrorNotSupported;
    set_tiles(s, BM * CG, BN);
    last_plan() = plan_name(BN, 0);
    const unsigned slots = (unsigned)sm_count() / CG, work = s.tiles * s.batch;
    return launch(kernel, CG * (work < slots ? work : slots), CG, smem, st, mp, mq, s, epi);
}

template <int KIND, int BN, int S, bool QMN, class Epi>
cudaError_t run_split(const Operand& p, const Operand& q, Shape s, const Epi& epi, cudaStream_t st)
{
    auto kernel = narrow_split_kernel<KIND, BN, S, QMN, Epi>;
    constexpr int smem = split_smem<BN, S>();
    static DeviceOnce once;
    cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    if (e != cudaSuccess) return e;
    CUtensorMap mp, mq;
    if (!make_map(&mp, KIND, p.base, p.inner, p.rows, s.batch, p.ld, p.stride, BM) ||
        !make_map(&mq, KIND, q.base, q.inner, q.rows, s.batch, q.ld, q.stride, QMN ? slab_k(KIND) : BN))
        return cudaErrorNotSupported;
    set_tiles(s, BM, BN);
    last_plan() = plan_name(BN, S);
    return launch(kernel, s.tiles * s.batch * S, S, smem, st, mp, mq, s, epi);
}

// How a product of more than 64 columns runs:
//   pairs:  256 x pairs tiles (256, 192 or 128 wide) on pairs of CTAs, persistent; 192 for 8-bit operands only (v-contiguous ones
//           come in blocks of 64 per CTA, triangles in blocks of 128)
//   split:  128 x 128 tiles, one per cluster of `split` CTAs, which share k and the epilogue's columns
// The plan with the shortest estimate is taken.  The estimates, in us, are fitted to all plans measured on twelve FP16 shapes from
// 100 x 130 to 2048 x 8192; on thirteen 8-bit shapes from 160 x 4096 x 4096 to 8192 x 1024 x 8192 the plan taken was within 6 % of
// the best:
//   a launch and its end                 3, persistent 5
//   a slab of k, 128 x 128 tiles         0.30                            1 round of 136 tiles, 128 slabs: 46.7
//   a slab of k, 256 x 256               0.30 for a lone tile, 0.37 with all SMs at it, 0.36 to 0.45 in later rounds, when
//                                        the epilogues (0.45: `heavy` ones, that read as much as they write) share L2 with the loads
//   a slab of k, 256 x 128               0.30, later 0.37
//   an epilogue                          128 x 128: 5.0, 4.6, 4.2 with 1, 2, 4 CTAs at it (heavy: 6.3, 5.6, 4.5); 256 x 256: 5.0
//                                        (8.5); 256 x 128: 5.0 (7.0) a round, 0.7 of it in the first
// A round of a persistent kernel takes the longer of its slabs and the epilogue before; clusters of 4 fill 128 SMs, clusters of 8 (never the
// best here) fewer.
struct Plan { unsigned pairs, split; };               // one of the two is 0
inline Plan choose_plan(unsigned U, unsigned V, unsigned K, unsigned batch, int tri, int kind, bool heavy)
{
    const unsigned nk = (K + slab_k(kind) - 1) / slab_k(kind);
    const double sms = sm_count();
    auto tiles = [&](unsigned bu, unsigned bv) {
        const double tu = (U + bu - 1) / bu, tv = (V + bv - 1) / bv;
        return batch * (tri ? tu * (tu + 1) / 2 : tu * tv);
    };
    Plan best{};
    double least = 1e30;
    auto consider = [&](Plan plan, double us) { if (us < least) { least = us; best = plan; } };
    const double pairs = std::floor(sms / 2), t256 = tiles(256, 256), t128 = tiles(128, 128), e256 = heavy ? 8.5 : 5.0, e128 = heavy ? 7.0 : 5.0;
    consider({256, 0}, 5 + nk * (0.30 + 0.07 * std::fmin(1.0, t256 / pairs)) + e256 + (std::ceil(t256 / pairs) - 1) * std::fmax(nk * (heavy ? 0.45 : 0.36), e256));
    // (For triangles never the shortest: up to one round, 74 tiles, 128 x 128 tiles take 0.5 less, beyond it 256 x 256 ones half the rounds.)
    if (!tri) consider({128, 0}, 5 + nk * 0.30 + 0.7 * e128 + (std::ceil(tiles(256, 128) / pairs) - 1) * std::fmax(nk * 0.37, e128));
    if (kind == KIND_I8)
        consider({192, 0}, 5 + nk * 0.33 + 0.75 * e256 + 0.5 + (std::ceil(tiles(256, 192) / pairs) - 1) * std::fmax(nk * (heavy ? 0.40 : 0.33), 0.75 * e256 + 0.5));
    const double finish[3] = {heavy ? 6.3 : 5.0, heavy ? 5.6 : 4.6, heavy ? 4.5 : 4.2};
    for (unsigned i = 0, s = 1; i < 3 && s <= nk; i++, s *= 2)
        consider({0, s}, 3 + std::ceil(t128 * s / (s == 4 ? sms - 20 : sms)) * ((nk + s - 1) / s * 0.30 + finish[i]));
    return best;
}

template <int KIND, int BN, bool QMN, class Epi>
cudaError_t run_split_by(unsigned split, const Operand& p, const Operand& q, const Shape& s, const Epi& epi, cudaStream_t st)
{
    if constexpr (BN < 128)
        if (split == 8) return run_split<KIND, BN, 8, QMN, Epi>(p, q, s, epi, st);
    switch (split) {
        case 4: return run_split<KIND, BN, 4, QMN, Epi>(p, q, s, epi, st);
        case 2: return run_split<KIND, BN, 2, QMN, Epi>(p, q, s, epi, st);
        default: return run_split<KIND, BN, 1, QMN, Epi>(p, q, s, epi, st);
    }
}

template <int KIND, bool QMN, class Epi>
cudaError_t run_planned(const Operand& p, const Operand& q, const Shape& s, const Epi& epi, cudaStream_t st)
{
    const Plan plan = choose_plan(s.U, s.V, s.K, s.batch, s.tri, KIND, Epi::kHeavy);
    if (plan.pairs == 256) return run_persistent<KIND, 256, QMN, Epi>(p, q, s, epi, st);
    if constexpr (!Epi::kTriangle)
        if (plan.pairs == 128) return run_persistent<KIND, 128, QMN, Epi>(p, q, s, epi, st);
    if constexpr (KIND == KIND_I8)
        if (plan.pairs == 192) return run_persistent<KIND, 192, QMN, Epi>(p, q, s, epi, st);
    return run_split_by<KIND, 128, QMN, Epi>(plan.split, p, q, s, epi, st);
}

}  // namespace narrow
}  // namespace cb200
