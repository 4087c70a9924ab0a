// The tile engine of the dense operators: C = A B^T over row tiles, on the 5th-generation tensor cores.
//
// A CTA pair (two SMs, `cta_group::2`) computes 256 x N of C, each CTA loading and owning 128 of the 256 rows of A and
// half of the N rows of B, so every operand byte a CTA stages feeds 256 columns; problems of at most 128 rows take one
// CTA (`cta_group::1`, 128 x N).  One warp issues tiled TMA loads into a ring of stages (one 128-byte swizzle span of K
// each), one lane issues the tcgen05.mma instructions, the accumulator sits in tensor memory twice (2 x N columns) so the
// epilogue of a tile overlaps the next one, and the epilogue warps read it with tcgen05.ld.  Grids are persistent: one CTA
// or pair per SM (pair of SMs), tiles dealt out in an order that lets the tiles in flight share operands in L2.
//
// Operands: f16 or bf16, K-major (rows of K values) or MN-major (rows of M or N values, for products that contract over
// the rows of a stored matrix), or e4m3 with one power-of-two scale byte per 128 values of K: `kind::mxf8f6f4.block_scale`
// multiplies the scales inside the tensor core, so scaled products cost no epilogue work and no extra accumulators.
//
// No load is multicast; every tensor map covers this GPU's own memory.  Every wait is bounded: a wait that runs out raises
// the error word, the CTA waits (bounded) for its copies and instructions in flight, frees its tensor memory and returns.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>

#include "apoe_common.cuh"

namespace apoe {

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                  const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
int encode_fn(EncodeTiledFn *out);   // the driver's tensor-map encoder (apoe_exact.cu)

namespace tile {

enum : int { kF16 = 0, kBf16 = 1, kE4m3 = 2 };   // operand kinds

constexpr uint32_t kWaitLimit = 1u << 22;
constexpr int kEpiWarps = 8;                      // two per quarter of the tensor-memory lanes, each half of the columns
constexpr int kThreads = (kEpiWarps + 4) * 32;    // + TMA producer, MMA issuer, two scale writers (e4m3 only)

// One shape of the engine.  N: columns of a tile; CG: CTAs of a group; AMN / BMN: operand stored with M (N) contiguous.
template <int KIND_, int CG_, int N_, bool AMN_ = false, bool BMN_ = false>
struct Shape {
    static constexpr int KIND = KIND_, CG = CG_, N = N_;
    static constexpr bool AMN = AMN_, BMN = BMN_, SCALED = KIND_ == kE4m3;
    static constexpr int M = 128 * CG;
    static constexpr int K = SCALED ? 128 : 64;            // values of K in a stage: one 128-byte span
    static constexpr int BR = N / CG;                      // rows of B a CTA loads
    static constexpr uint32_t A_BYTES = 128 * 128, B_BYTES = BR * 128;
    static constexpr uint32_t SFA_BYTES = SCALED ? 512 : 0, SFB_BYTES = SCALED ? 1024 : 0;   // 128 and 256 scale words
    static constexpr uint32_t LOAD_BYTES = A_BYTES + B_BYTES;
    static constexpr uint32_t STAGE_BYTES = (LOAD_BYTES + SFA_BYTES + SFB_BYTES + 1023) / 1024 * 1024;
    static constexpr uint32_t EPI_BYTES = kEpiWarps * 4096;
    // as many stages as fit beside the epilogue's staging; e4m3: also one set of scale columns in tensor memory per stage
    static constexpr int FIT = (int)((232448 - 1024 - 512 - EPI_BYTES) / STAGE_BYTES);
    static constexpr int SF_COLS = SCALED ? 12 : 0;        // 4 (128 rows of A) + 8 (up to 256 rows of B)
    static constexpr int SF_FIT = SCALED ? (512 - 2 * N) / 12 : 16;
    static constexpr int STAGES = FIT < SF_FIT ? (FIT < 8 ? FIT : 8) : (SF_FIT < 8 ? SF_FIT : 8);
    static constexpr uint32_t SMEM = STAGES * STAGE_BYTES + EPI_BYTES + 1024;
    static_assert(STAGES >= 3, "too few stages");
    static_assert(2 * N + STAGES * SF_COLS <= 512, "tensor memory");
    static_assert(BR % 8 == 0 && (!BMN || BR % 64 == 0), "rows of B per CTA");
    static_assert(!SCALED || (!AMN && !BMN), "8-bit operands are K-major");
    static_assert(N % 32 == 0 && N <= 256, "columns");
    // kind::f16: D fp32 (bit 4), A / B type (bits 7, 10), MN-major flags (15, 16), N >> 3 (17), M >> 4 (24);
    // kind::mxf8f6f4: e4m3 types are 0, scale type ue8m0 (bit 23), scale byte 0 of each word (bits 4, 29)
    static constexpr uint32_t IDESC = SCALED ? ((1u << 23) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24))
                                             : ((1u << 4) | ((uint32_t)KIND << 7) | ((uint32_t)KIND << 10) | ((AMN ? 1u : 0u) << 15) |
                                                ((BMN ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24));
};

// The tiles of one product and their order.  Groups of `group_m` row tiles walk the column tiles together, so the tiles in
// flight share both operands in L2.  `splits` cuts K: split s contracts its share of the K blocks into a result of its own.
struct Grid {
    uint32_t tiles_m, tiles_n, splits, group_m, kblocks, total;
};
__device__ __forceinline__ void locate(const Grid &g, uint32_t id, uint32_t &mi, uint32_t &ni, uint32_t &si) {
    const uint32_t per = g.tiles_m * g.tiles_n;
    si = id / per;
    id -= si * per;
    const uint32_t span = g.group_m * g.tiles_n, grp = id / span, r = id - grp * span;
    const uint32_t rows = min(g.group_m, g.tiles_m - grp * g.group_m);
    ni = r / rows;
    mi = grp * g.group_m + (r - ni * rows);
}

// ---- instructions ----------------------------------------------------------------------------------------------------
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t leader_addr(const void *p) {   // shared::cluster address of the same object in CTA 0 of the cluster
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
    return a;
}
__device__ __forceinline__ void arrive_cluster(uint32_t addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// waits with cluster-scope acquire: the arrivals may come from the pair's other CTA
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, uint32_t *err, uint32_t code, uint32_t limit = kWaitLimit) {
    for (uint32_t i = 0; i < limit; ++i) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\t"
                     "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
                     "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
        if (ok) return true;
    }
    if (err) atomicExch(err, code);
    return false;
}
template <int CG>
__device__ __forceinline__ void load_2d(void *dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    if (CG == 2)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
template <int CG>
__device__ __forceinline__ void commit(uint64_t *bar) {   // arrives on the barrier of every CTA of the group
    if (CG == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    if (CG == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
template <int CG>
__device__ __forceinline__ void mma_mx8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t acc) {
    if (CG == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(sfa), "r"(sfb) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(sfa), "r"(sfb) : "memory");
}
// 32 lanes x 16 bytes of shared memory to 4 columns of tensor memory, repeated in each quarter of the lanes
template <int CG>
__device__ __forceinline__ void copy_scales(uint32_t dst, uint64_t desc) {
    if (CG == 2) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(dst), "l"(desc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(dst), "l"(desc) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t (&r)[32], uint32_t addr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// ---- shared-memory descriptors (version 1) -----------------------------------------------------------------------------
// K-major, 128-byte swizzle: 8-row groups 1024 bytes apart; a K step of 32 bytes moves the start address
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// MN-major, 128-byte swizzle: slabs of 64 M (N) values x 64 K rows of 128 bytes, 8192 bytes apart (bits 16-29); groups of 8
// K rows 1024 bytes apart (bits 32-45); a K step of 16 rows moves the start address by 2048 bytes
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(8192 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// scale words: no swizzle, 8-row groups of 16-byte rows 128 bytes apart
__device__ __forceinline__ uint64_t desc_sf(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(128 >> 4) << 32) | (1ull << 46);
}

// Scale bytes of the operands (e4m3): [rows][ld], one per 128 values of K.
struct Scales {
    const uint8_t *a, *b;
    size_t lda, ldb;
    uint32_t m, n;
};

// ---- the kernel --------------------------------------------------------------------------------------------------------
// Epi: a type with `Args`, `Epi(const Args &, uint8_t *staging, int warp_row, int lane)`, `begin(m0, n0, split)`,
// `chunk(uint32_t (&r)[32], col)` for 32 columns of the lane's row, `end()`.  Every lane of a warp makes the same calls.
template <class S, class Epi>
__global__ void __launch_bounds__(kThreads, 1) tile_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                           const Grid grid, const Scales scales, const typename Epi::Args epi_args, uint32_t *err) {
    extern __shared__ __align__(1024) uint8_t tile_smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(tile_smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full_bar[S::STAGES], empty_bar[S::STAGES], tfull_bar[2], tempty_bar[2], drain_bar;
    __shared__ uint32_t tmem_base_s;
    constexpr int CG = S::CG;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0u;
    const uint32_t group = blockIdx.x / CG, groups = gridDim.x / CG;

    if (tid == 0) {
        // full: the leader's expect + (e4m3) one arrival per CTA whose scale words are written
        for (int s = 0; s < S::STAGES; ++s) { mbar_init(&full_bar[s], S::SCALED ? 1 + CG : 1); mbar_init(&empty_bar[s], 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(&tfull_bar[s], 1); mbar_init(&tempty_bar[s], kEpiWarps * CG); }
        mbar_init(&drain_bar, 1);
        mbar_fence_init();
    }
    if (warp == kEpiWarps + 1) {
        if (CG == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync();
    fence_after();
    const uint32_t tmem = tmem_base_s;

    if (warp == kEpiWarps) {
        // ---------------- TMA producer (every CTA loads its own rows; the pair's leader counts the bytes of both) -------
        if (lane == 0) {
            uint32_t g = 0;
            bool ok = true;
            for (uint32_t t = group; t < grid.total && ok; t += groups) {
                uint32_t mi, ni, si;
                locate(grid, t, mi, ni, si);
                const int m0 = (int)(mi * S::M + rank * 128), n0 = (int)(ni * S::N + rank * S::BR);
                const uint32_t k0 = (uint32_t)((uint64_t)grid.kblocks * si / grid.splits), k1 = (uint32_t)((uint64_t)grid.kblocks * (si + 1) / grid.splits);
                for (uint32_t kb = k0; kb < k1; ++kb, ++g) {
                    const uint32_t s = g % S::STAGES;
                    ok = wait(&empty_bar[s], ((g / S::STAGES) & 1u) ^ 1u, err, 30u);
                    if (!ok) break;
                    uint8_t *st = smem + (size_t)s * S::STAGE_BYTES;
                    if (rank == 0) mbar_arrive_expect_tx(&full_bar[s], S::LOAD_BYTES * CG);
                    const uint32_t bar = CG == 2 ? leader_addr(&full_bar[s]) : smem_u32(&full_bar[s]);
                    const int k = (int)(kb * S::K);
                    if (S::AMN) {
                        load_2d<CG>(st, &map_a, m0, k, bar);
                        load_2d<CG>(st + 8192, &map_a, m0 + 64, k, bar);
                    } else load_2d<CG>(st, &map_a, k, m0, bar);
                    if (S::BMN) {
#pragma unroll
                        for (int j = 0; j < S::BR / 64; ++j) load_2d<CG>(st + S::A_BYTES + j * 8192, &map_b, n0 + j * 64, k, bar);
                    } else load_2d<CG>(st + S::A_BYTES, &map_b, k, n0, bar);
                }
            }
            if (!ok && rank == 0)   // copies still on their way (both CTAs') complete on these barriers
                for (uint32_t j = g > S::STAGES ? g - S::STAGES : 0; j < g; ++j) wait(&full_bar[j % S::STAGES], (j / S::STAGES) & 1u, nullptr, 0u, 1u << 12);
        }
        __syncwarp();
    } else if (warp == kEpiWarps + 1) {
        // ---------------- MMA issue (one lane of the leader) ------------------------------------------------------------
        if (lane == 0 && rank == 0) {
            uint32_t g = 0, it = 0;
            bool ok = true;
            for (uint32_t t = group; t < grid.total && ok; t += groups, ++it) {
                uint32_t mi, ni, si;
                locate(grid, t, mi, ni, si);
                const uint32_t k0 = (uint32_t)((uint64_t)grid.kblocks * si / grid.splits), k1 = (uint32_t)((uint64_t)grid.kblocks * (si + 1) / grid.splits);
                const uint32_t acc = it & 1u, d = tmem + acc * S::N;
                ok = wait(&tempty_bar[acc], ((it >> 1) & 1u) ^ 1u, err, 31u);
                if (!ok) break;
                fence_after();
                for (uint32_t kb = k0; kb < k1; ++kb, ++g) {
                    const uint32_t s = g % S::STAGES;
                    ok = wait(&full_bar[s], (g / S::STAGES) & 1u, err, 32u);
                    if (!ok) break;
                    fence_after();
                    const uint32_t a = smem_u32(smem + (size_t)s * S::STAGE_BYTES), b = a + S::A_BYTES;
                    const uint32_t sfa = tmem + 2 * S::N + s * S::SF_COLS, sfb = sfa + 4;
                    if (S::SCALED) {
                        // the stage's own scale columns: the products that read them last have completed (their commit freed the stage)
                        copy_scales<CG>(sfa, desc_sf(b + S::B_BYTES));
                        copy_scales<CG>(sfb, desc_sf(b + S::B_BYTES + 512));
                        copy_scales<CG>(sfb + 4, desc_sf(b + S::B_BYTES + 1024));
                    }
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        const uint64_t da = S::AMN ? desc_mn(a + kk * 2048) : desc_k(a + kk * 32);
                        const uint64_t db = S::BMN ? desc_mn(b + kk * 2048) : desc_k(b + kk * 32);
                        const uint32_t add = (kb != k0 || kk != 0) ? 1u : 0u;
                        if (S::SCALED) mma_mx8<CG>(d, da, db, S::IDESC, sfa, sfb, add);
                        else mma_f16<CG>(d, da, db, S::IDESC, add);
                    }
                    commit<CG>(&empty_bar[s]);
                }
                if (ok) commit<CG>(&tfull_bar[acc]);
            }
            if (!ok) {   // instructions in flight finish before the tensor memory is given back
                commit<CG>(&drain_bar);
                wait(&drain_bar, 0u, nullptr, 0u, 1u << 14);
            }
        }
        __syncwarp();
    } else if (warp >= kEpiWarps + 2) {
        // ---------------- scale writers (e4m3): the two warps take the K blocks in turn -----------------------------------
        if (S::SCALED) {
            uint32_t g = 0;
            bool ok = true;
            for (uint32_t t = group; t < grid.total && ok; t += groups) {
                uint32_t mi, ni, si;
                locate(grid, t, mi, ni, si);
                const uint32_t m0 = mi * S::M + rank * 128, n0 = ni * S::N;
                const uint32_t k0 = (uint32_t)((uint64_t)grid.kblocks * si / grid.splits), k1 = (uint32_t)((uint64_t)grid.kblocks * (si + 1) / grid.splits);
                for (uint32_t kb = k0; kb < k1 && ok; ++kb, ++g) {
                    if ((g & 1u) != (uint32_t)(warp & 1)) continue;
                    const uint32_t s = g % S::STAGES;
                    // lane i of the 32 lanes keeps rows i, i + 32, i + 64, i + 96 in its 16 bytes; rows past the end: 2^0
                    uint32_t w[12];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t row = m0 + j * 32 + lane;
                        w[j] = row < scales.m ? scales.a[(size_t)row * scales.lda + kb] : 127u;
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const uint32_t row = n0 + j * 32 + lane;
                        w[4 + j] = j * 32 < S::N && row < scales.n ? scales.b[(size_t)row * scales.ldb + kb] : 127u;
                    }
                    ok = wait(&empty_bar[s], ((g / S::STAGES) & 1u) ^ 1u, err, 33u);
                    ok = __all_sync(0xFFFFFFFFu, ok);
                    if (!ok) break;
                    uint4 *dst = reinterpret_cast<uint4 *>(smem + (size_t)s * S::STAGE_BYTES + S::LOAD_BYTES);
                    dst[lane] = make_uint4(w[0], w[1], w[2], w[3]);
                    dst[32 + lane] = make_uint4(w[4], w[5], w[6], w[7]);
                    dst[64 + lane] = make_uint4(w[8], w[9], w[10], w[11]);
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) {
                        if (CG == 2) arrive_cluster(leader_addr(&full_bar[s]));
                        else mbar_arrive(&full_bar[s]);
                    }
                }
            }
        }
    } else {
        // ---------------- epilogue: warp w reads the lanes 32 (w mod 4) .. of the accumulator, warps 0-3 the first half of
        // the columns, 4-7 the second ------------------------------------------------------------------------------------
        const int quarter = warp & 3, half = warp >> 2;
        constexpr int CHUNKS = S::N / 32, FIRST = (CHUNKS + 1) / 2;
        Epi epi(epi_args, smem + (size_t)S::STAGES * S::STAGE_BYTES + warp * 4096, lane);
        uint32_t it = 0;
        bool ok = true;
        for (uint32_t t = group; t < grid.total && ok; t += groups, ++it) {
            uint32_t mi, ni, si;
            locate(grid, t, mi, ni, si);
            const uint32_t acc = it & 1u;
            epi.begin(mi * S::M + rank * 128 + quarter * 32, ni * S::N, si, ni * 2 + half);
            ok = wait(&tfull_bar[acc], (it >> 1) & 1u, err, 34u);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            fence_after();
            const uint32_t src = tmem + ((uint32_t)(32 * quarter) << 16) + acc * S::N;
            const int c1 = half ? CHUNKS : FIRST;
            uint32_t r[32];
            for (int c = half ? FIRST : 0; c < c1; ++c) {
                tmem_ld32(r, src + c * 32);
                tmem_wait_ld();
                if (c == c1 - 1) {          // the last read of this warp: the accumulator can be written again
                    fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (CG == 2) arrive_cluster(leader_addr(&tempty_bar[acc]));
                        else mbar_arrive(&tempty_bar[acc]);
                    }
                }
                epi.chunk(r, ni * S::N + c * 32);
            }
            epi.end();
        }
    }
    fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync();
    if (warp == kEpiWarps + 1) {
        fence_after();
        if (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

}  // namespace tile
}  // namespace apoe
