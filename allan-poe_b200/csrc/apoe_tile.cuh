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

#include <type_traits>

#include "apoe_common.cuh"

namespace apoe {

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                  const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
int encode_fn(EncodeTiledFn *out);   // the driver's tensor-map encoder (apoe_exact.cu)

namespace tile {

enum : int { kF16 = 0, kBf16 = 1, kE4m3 = 2 };   // operand kinds

constexpr uint32_t kWaitLimit = 1u << 20;         // polls of a few microseconds: seconds, where milliseconds are long
constexpr uint32_t kWarp = 0xFFFFFFFFu;
constexpr int kEpiWarps = 8;                      // two per quarter of the tensor-memory lanes, each half of the columns
constexpr int kThreads = (kEpiWarps + 4) * 32;    // + TMA producer, MMA issuer, two scale writers (e4m3 only)

// One shape of the engine.  N: most columns of a tile (a launch may use fewer: Grid::tile_n); CG: CTAs of a group; AMN / BMN:
// operand stored with M (N) contiguous.
template <int KIND_, int CG_, int N_, bool AMN_ = false, bool BMN_ = false>
struct Shape {
    static constexpr int KIND = KIND_, CG = CG_, N = N_;
    static constexpr bool AMN = AMN_, BMN = BMN_, SCALED = KIND_ == kE4m3;
    static constexpr int M = 128 * CG;
    static constexpr int K = SCALED ? 128 : 64;            // values of K in a stage: one 128-byte span
    static constexpr int BR = N / CG;                      // rows of B a CTA has room for
    static constexpr uint32_t A_BYTES = 128 * 128, B_BYTES = BR * 128;
    static constexpr uint32_t STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr uint32_t EPI_BYTES = kEpiWarps * 4096;
    // scale words (e4m3): four K blocks at a time, 128 rows of A and up to 256 of B, in a ring of their own; each slot has its
    // 12 columns of tensor memory
    static constexpr int SF_SLOTS = SCALED ? 4 : 0;
    static constexpr uint32_t SF_BYTES = SCALED ? 1536 : 0;
    static constexpr uint32_t SF_ROOM = SF_SLOTS * SF_BYTES;
    static constexpr int FIT = (int)((232448 - 1024 - 1024 - EPI_BYTES - SF_ROOM) / STAGE_BYTES);   // alignment, barriers, staging
    static constexpr int STAGES = FIT < 8 ? FIT : 8;
    static constexpr uint32_t SMEM = STAGES * STAGE_BYTES + SF_ROOM + EPI_BYTES + 1024;
    static_assert(STAGES >= 3, "too few stages");
    static_assert(2 * N + SF_SLOTS * 12 <= 512, "tensor memory");
    static_assert(BR % 8 == 0 && (!BMN || BR % 64 == 0), "rows of B per CTA");
    static_assert(!SCALED || (!AMN && !BMN), "8-bit operands are K-major");
    static_assert(N % 32 == 0 && N <= 256, "columns");
    static_assert(!SCALED || 4 + N / 32 <= 12, "scale words");
    // kind::f16: D fp32 (bit 4), A / B type (bits 7, 10), MN-major flags (15, 16), N >> 3 (17: added), M >> 4 (24);
    // kind::mxf8f6f4: e4m3 types are 0, scale type ue8m0 (bit 23), the byte of the scale words to use (bits 4 and 29: added)
    static constexpr uint32_t IDESC = SCALED ? ((1u << 23) | ((uint32_t)(M >> 4) << 24))
                                             : ((1u << 4) | ((uint32_t)KIND << 7) | ((uint32_t)KIND << 10) | ((AMN ? 1u : 0u) << 15) |
                                                ((BMN ? 1u : 0u) << 16) | ((uint32_t)(M >> 4) << 24));
};

// The tiles of one product and their order.  Groups of `group_m` row tiles walk the column tiles together, so the tiles in
// flight share both operands in L2.  K may be cut: split s contracts K blocks s * kper .. into a result of its own.
struct Grid {
    uint32_t tiles_m, tiles_n, group_m, kblocks, kper, total;   // kper: K blocks of a split (the last one may have fewer)
    uint32_t tile_n;                                            // columns of a tile: a multiple of 32, at most the shape's N
    uint32_t a_rows;                                            // rows of A a load brings (K-major): 128, fewer where there are fewer
    uint32_t early;                                             // the operands are complete before the kernel's predecessor has ended
};
__device__ __forceinline__ void locate(const Grid &g, uint32_t id, uint32_t &mi, uint32_t &ni, uint32_t &si) {
    const uint32_t per = g.tiles_m * g.tiles_n;
    si = g.kper < g.kblocks ? id / per : 0u;
    id -= si * per;
    const uint32_t span = g.group_m * g.tiles_n, grp = id / span, r = id - grp * span;
    const uint32_t rows = min(g.group_m, g.tiles_m - grp * g.group_m);
    ni = r / rows;
    mi = grp * g.group_m + (r - ni * rows);
}

// Programmatic launch: wait until the kernels before this one have ended and their writes are visible / let the next kernel of
// the stream start, as far as SMs are free.  Every kernel of the dense operators waits first and then lets the next one
// start: so all that came before a kernel's predecessor is complete when the kernel starts, and it may read that (the
// operators' inputs, once a kernel of the same call has run) before its own wait.  It writes nothing before.
// Loads are plain ones, never non-coherent (ld.global.nc, __restrict__ on what is read): those are promised memory that nothing
// writes while the kernel runs, and the predecessor of a kernel that has started early may still be writing what the
// kernel reads after its wait (the scale bytes of rows quantised just before, the factor of the gradients).
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

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
// Arrival on a barrier of the pair's leader.  With cluster-scope release: orders this thread's ordinary writes (the scale words)
// for the other CTA.  Without: for arrivals that only say "read"; a release at cluster scope would first wait for the
// epilogue's global stores, about a microsecond per tile.
__device__ __forceinline__ void arrive_cluster_release(uint32_t addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// Bounded waits; the second form sees what the pair's other CTA wrote before its releasing arrival.
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, uint32_t *err, uint32_t code, uint32_t limit = kWaitLimit) {
    for (uint32_t i = 0; i < limit; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    if (err) atomicExch(err, code);
    return false;
}
__device__ __forceinline__ bool wait_warp(uint64_t *bar, uint32_t parity, uint32_t *err, uint32_t code) {   // one answer for the warp
    return __all_sync(kWarp, wait(bar, parity, err, code));
}
__device__ __forceinline__ bool ask(uint64_t *bar, uint32_t parity) {      // without waiting
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool ask_cluster(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool wait_cluster(uint64_t *bar, uint32_t parity, uint32_t *err, uint32_t code) {
    for (uint32_t i = 0; i < kWaitLimit; ++i) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\t"
                     "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
                     "selp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
        if (ok) return true;
    }
    atomicExch(err, code);
    return false;
}
__device__ __forceinline__ bool elect_one() {   // true in one lane of the (whole) warp
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
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

// One 64-byte wide box of shared memory to a matrix of a stack of them, plain or added to what is there (f32, in L2).
__device__ __forceinline__ void store_3d(const CUtensorMap *map, const void *src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];"
                 ::"l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(src)) : "memory");
}
__device__ __forceinline__ void add_3d(const CUtensorMap *map, const void *src, int x, int y, int z) {
    asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.bulk_group [%0, {%1, %2, %3}], [%4];"
                 ::"l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(src)) : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void store_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(LEFT) : "memory"); }

// ---- shared-memory descriptors (version 1) -----------------------------------------------------------------------------
// K-major, 128-byte swizzle: 8-row groups 1024 bytes apart; a K step of 32 bytes moves the start address
__host__ __device__ constexpr uint64_t desc_k(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// MN-major, 128-byte swizzle: slabs of 64 M (N) values x 64 K rows of 128 bytes, 8192 bytes apart (bits 16-29); groups of 8
// K rows 1024 bytes apart (bits 32-45); a K step of 16 rows moves the start address by 2048 bytes
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(8192 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_of(uint32_t hi, uint32_t lo) { return (uint64_t)hi << 32 | lo; }
// scale words: no swizzle, 8-row groups of 16-byte rows 128 bytes apart
__device__ __forceinline__ uint64_t desc_sf(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(128 >> 4) << 32) | (1ull << 46);
}

// Scale bytes of the operands (e4m3): [rows][ld], one per 128 values of K.
struct Scales {
    const uint8_t *a, *b, *a_end, *b_end;
    size_t lda, ldb;
    uint32_t m, n;
    uint32_t words;            // both: rows on 4-byte boundaries
};

// A warp's 4 KB of shared memory for results on their way out: two boxes of 2 KB, used in turn.
struct Staging {
    uint8_t *base;
    uint32_t boxes;            // boxes written so far
};

// ---- the kernel --------------------------------------------------------------------------------------------------------
// Epi: a type with `Args`, `Epi(const Args &, Staging &, const CUtensorMap *out, int lane)`, `ahead(first row)` as early as
// possible (what a row needs from global memory is on its way while the tile before is worked on), `begin(first row, first
// column, split, part)`, `chunk(uint32_t (&r)[32], col)` for 32 columns of the lane's row, `end()` after a tile, `finish()`
// after the last.  Every lane of a warp makes the same calls.
// Epi2 other than NoSecond: a second product of the same shape but for an MN-major A, with operands, grid and results of its
// own, whose tiles follow the first one's (the two products of a gradient share one launch and fill each other's rounds).
// Tiles of a product are dealt out in turn; the groups that get one tile of the first product less than the others get
// `lead` tiles of the second before the turns begin, so all end together although the tiles differ in cost.
struct NoSecond {
    struct Args {};
    __device__ __forceinline__ NoSecond(const Args &, Staging &, const CUtensorMap *, int) {}
    __device__ __forceinline__ void ahead(uint32_t) {}
    __device__ __forceinline__ void begin(uint32_t, uint32_t, uint32_t, uint32_t) {}
    __device__ __forceinline__ void chunk(uint32_t (&)[32], uint32_t) {}
    __device__ __forceinline__ void end() {}
    __device__ __forceinline__ void finish() {}
};
template <class Epi2>
struct Second {
    CUtensorMap map_a, map_b, map_out;
    Grid grid;
    uint32_t lead;
    typename Epi2::Args epi;
};
template <> struct Second<NoSecond> { NoSecond::Args epi; };
template <class S, class Epi, class Epi2>
__global__ void __launch_bounds__(kThreads, 1) tile_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                           const __grid_constant__ CUtensorMap map_out, const Grid grid, const Scales scales, const typename Epi::Args epi_args,
                                                           const __grid_constant__ Second<Epi2> second, uint32_t *err) {
    extern __shared__ __align__(1024) uint8_t tile_smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(tile_smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full_bar[S::STAGES], empty_bar[S::STAGES], tfull_bar[2], tempty_bar[2], drain_bar;
    __shared__ uint64_t sfull_bar[S::SCALED ? S::SF_SLOTS : 1], sempty_bar[S::SCALED ? S::SF_SLOTS : 1];
    __shared__ uint32_t tmem_base_s;
    constexpr int CG = S::CG;
    constexpr bool DUAL = !std::is_same<Epi2, NoSecond>::value;
    static_assert(!DUAL || (!S::SCALED && !S::AMN), "second products");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0u;
    const uint32_t group = blockIdx.x / CG, groups = gridDim.x / CG;
    // this group's tiles, in order: `first(tile)` for the first product, `then(tile)` for the second, while `ok`
    auto walk = [&](const bool &ok, auto first, auto then) {
        for (uint32_t t = group; t < grid.total && ok; t += groups) first(t);
        if constexpr (DUAL) {
            const uint32_t rest = grid.total % groups, light = groups - rest, before = second.lead * light;
            uint32_t i = 0, t = group;
            if (group >= rest) t = second.lead ? group - rest : before + group;
            else t = before + group;
            while (t < second.grid.total && ok) {
                then(t);
                ++i;
                if (group >= rest && i < second.lead) t += light;
                else if (group >= rest && i == second.lead) t = before + group;
                else t += groups;
            }
        }
    };

    if (tid == 0) {
        for (int s = 0; s < S::STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
        for (int s = 0; s < S::SF_SLOTS; ++s) { mbar_init(&sfull_bar[s], CG); mbar_init(&sempty_bar[s], 1); }   // an arrival per CTA
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
    if (!grid.early || warp < kEpiWarps) pdl_wait();
    if (tid == 0) pdl_launch();

    if (warp == kEpiWarps) {
        // ---------------- TMA producer (every CTA loads its own rows; the pair's leader counts the bytes of both) -----------
        // As in the MMA warp, all lanes walk the loop and one elected lane issues: with the loop inside a one-lane branch the
        // products were issued at 215 cycles each (e4m3, 112 needed) and 170 (f16, 128 needed).
        uint32_t s = 0, phase = 0, issued = 0;
        bool ok = true, free = true;
        auto load = [&](const CUtensorMap &ma, const CUtensorMap &mb, const Grid &gr, uint32_t t, auto amn) {
            constexpr bool AMN = decltype(amn)::value;
            const uint32_t br = gr.tile_n / CG, bytes = ((AMN ? S::A_BYTES : gr.a_rows * 128) + (S::BMN ? (br + 63) / 64 * 8192 : br * 128)) * CG;
            uint32_t mi, ni, si;
            locate(gr, t, mi, ni, si);
            const int m0 = (int)(mi * S::M + rank * 128), n0 = (int)(ni * gr.tile_n + rank * br);
            const uint32_t k0 = si * gr.kper, k1 = min(k0 + gr.kper, gr.kblocks);
            for (uint32_t kb = k0; kb < k1; ++kb) {
                if (!free) {
                    ok = wait_warp(&empty_bar[s], phase ^ 1u, err, 30u);
                    if (!ok) break;
                }
                uint8_t *st = smem + s * S::STAGE_BYTES;
                uint64_t *full = &full_bar[s];
                const uint32_t bar = CG == 2 ? leader_addr(full) : smem_u32(full);
                const int k = (int)(kb * S::K);
                ++issued;
                if (++s == S::STAGES) { s = 0; phase ^= 1u; }
                const bool asked = ask(&empty_bar[s], phase ^ 1u);   // the next stage's, while this one's loads are issued
                if (elect_one()) {
                    if (rank == 0) mbar_arrive_expect_tx(full, bytes);
                    if (AMN) {
                        load_2d<CG>(st, &ma, m0, k, bar);
                        load_2d<CG>(st + 8192, &ma, m0 + 64, k, bar);
                    } else load_2d<CG>(st, &ma, k, m0, bar);
                    if (S::BMN)
                        for (uint32_t j = 0; j * 64 < br; ++j) load_2d<CG>(st + S::A_BYTES + j * 8192, &mb, n0 + (int)j * 64, k, bar);
                    else load_2d<CG>(st + S::A_BYTES, &mb, k, n0, bar);
                }
                free = __all_sync(kWarp, asked);                     // one answer for the warp
            }
        };
        walk(ok, [&](uint32_t t) { load(map_a, map_b, grid, t, std::integral_constant<bool, S::AMN>{}); },
             [&](uint32_t t) { if constexpr (DUAL) load(second.map_a, second.map_b, second.grid, t, std::true_type{}); });
        if (!ok && rank == 0)   // copies still on their way (both CTAs') complete on these barriers
            for (uint32_t j = issued > S::STAGES ? issued - S::STAGES : 0; j < issued; ++j)
                wait(&full_bar[j % S::STAGES], (j / S::STAGES) & 1u, nullptr, 0u, 1u << 12);
    } else if (warp == kEpiWarps + 1) {
        // ---------------- MMA issue (the leader; the warp walks the loop together and one elected lane issues) -----------
        if (rank == 0) {
            // A wait on a barrier that is ready costs about 145 cycles from issue to use, the products of a K block 256 to 512:
            // the next stage's barrier is asked while this one's products are issued, and only the low words of the
            // descriptors change.
            constexpr uint32_t A_STEP = 2, B_STEP = S::BMN ? 128 : 2;             // a K step, in the address field's 16 bytes
            constexpr uint32_t DESC_HI = (uint32_t)(desc_k(0) >> 32);             // the same for all kinds
            constexpr uint32_t LBO_K = 1u << 16, LBO_MN = (8192u >> 4) << 16;
            const uint32_t base = (smem_u32(smem) & 0x3FFFFu) >> 4;
            uint32_t s = 0, phase = 0, it = 0, sg = 0, sf = 0;
            bool ok = true, ready = false, sready = false;
            auto multiply = [&](const Grid &gr, uint32_t t, auto amn) {
                constexpr bool AMN = decltype(amn)::value;
                constexpr uint32_t FLAG = AMN && !S::AMN ? 1u << 15 : 0u;
                const uint32_t si = gr.kper < gr.kblocks ? t / (gr.tiles_m * gr.tiles_n) : 0u;
                const uint32_t k0 = si * gr.kper, k1 = min(k0 + gr.kper, gr.kblocks);
                const uint32_t acc = it & 1u, d = tmem + acc * S::N;
                uint32_t idesc = S::IDESC | ((gr.tile_n >> 3) << 17) | FLAG, add = 0;
                ok = wait_warp(&tempty_bar[acc], ((it >> 1) & 1u) ^ 1u, err, 31u);
                if (!ok) return;
                fence_after();
                for (uint32_t kb = k0; kb < k1; ++kb) {
                    if (!ready) {
                        ok = wait_warp(&full_bar[s], phase, err, 32u);
                        if (!ok) break;
                    }
                    const uint32_t slot = sg % (S::SCALED ? S::SF_SLOTS : 1);
                    const bool fresh = S::SCALED && kb % 4 == 0, last = kb + 1 == k1;
                    if (fresh) {
                        // the slot's own scale columns: the products that read them last have completed (their commit freed it)
                        if (!sready) {
                            ok = __all_sync(kWarp, wait_cluster(&sfull_bar[slot], (sg / (S::SCALED ? S::SF_SLOTS : 1)) & 1u, err, 35u));
                            if (!ok) break;
                        }
                        sf = tmem + 2 * S::N + slot * 12;
                    }
                    fence_after();
                    const uint32_t here = s, a = base + s * (S::STAGE_BYTES >> 4), b = a + (S::A_BYTES >> 4);
                    if (++s == S::STAGES) { s = 0; phase ^= 1u; }
                    bool sasked = false;
                    const bool asked = ask(&full_bar[s], phase);   // the next stage's (after the last one: of the next tile)
                    if (S::SCALED && (kb % 4 == 3 || last)) {
                        ++sg;
                        sasked = ask_cluster(&sfull_bar[sg % (S::SCALED ? S::SF_SLOTS : 1)], (sg / (S::SCALED ? S::SF_SLOTS : 1)) & 1u);
                    }
                    if (elect_one()) {
                        if (fresh) {
                            const uint32_t w = smem_u32(smem) + S::STAGES * S::STAGE_BYTES + slot * S::SF_BYTES;
                            copy_scales<CG>(sf, desc_sf(w));
                            copy_scales<CG>(sf + 4, desc_sf(w + 512));
                            if (S::N > 128) copy_scales<CG>(sf + 8, desc_sf(w + 1024));
                        }
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            const uint64_t da = desc_of(DESC_HI, (a + kk * (AMN ? 128 : A_STEP)) | (AMN ? LBO_MN : LBO_K));
                            const uint64_t db = desc_of(DESC_HI, (b + kk * B_STEP) | (S::BMN ? LBO_MN : LBO_K));
                            if (S::SCALED) mma_mx8<CG>(d, da, db, idesc | ((kb & 3u) << 4) | ((kb & 3u) << 29), sf, sf + 4, add | kk);
                            else mma_f16<CG>(d, da, db, idesc, add | kk);
                        }
                        commit<CG>(&empty_bar[here]);
                        if (S::SCALED && (kb % 4 == 3 || last)) commit<CG>(&sempty_bar[slot]);
                        if (last) commit<CG>(&tfull_bar[acc]);
                    }
                    add = 1;
                    ready = __all_sync(kWarp, asked);          // one answer for the warp
                    if (S::SCALED && (kb % 4 == 3 || last)) sready = __all_sync(kWarp, sasked);
                }
            };
            walk(ok, [&](uint32_t t) { multiply(grid, t, std::integral_constant<bool, S::AMN>{}); ++it; },
                 [&](uint32_t t) { if constexpr (DUAL) { multiply(second.grid, t, std::true_type{}); ++it; } });
            if (!ok) {   // instructions in flight finish before the tensor memory is given back
                if (elect_one()) commit<CG>(&drain_bar);
                wait(&drain_bar, 0u, nullptr, 0u, 1u << 14);
            }
        }
        __syncwarp();
    } else if (warp >= kEpiWarps + 2) {
        // ---------------- scale writers (e4m3): the two warps take groups of four K blocks in turn ------------------------
        // A word of the tensor core's scale layout holds four bytes of a row and every product names the one it uses: the words
        // are the rows' own bytes of four blocks of 128, copied once per 16 products.  The next group's words are on their way
        // while the current one waits for its slot.
        if constexpr (S::SCALED) {
            constexpr int ROWS = 4 + S::N / 32;
            const uint32_t per_tile = (grid.kblocks + 3) / 4;        // scaled products are never split
            uint32_t t = group, grp = (uint32_t)(warp & 1), sg = grp;   // this warp's next group; its number over all tiles
            auto settle = [&]() { while (t < grid.total && grp >= per_tile) { grp -= per_tile; t += groups; } };
            // The four bytes of a row may start anywhere: the two words around them (none past the last byte) are loaded and
            // shifted when they are used.  Nothing waits inside, so all rows' loads are under way together.  Rows past the
            // end read some other row's bytes: their values are zero, their results are not stored.
            uint32_t lo[ROWS], hi[ROWS], places = 0;
            auto fetch = [&]() {
                uint32_t mi, ni, si;
                locate(grid, t, mi, ni, si);
                const uint32_t m0 = mi * S::M + rank * 128, n0 = ni * grid.tile_n, kb = grp * 4;
                places = 0;
#pragma unroll
                for (int j = 0; j < ROWS; ++j) {
                    const bool of_a = j < 4;
                    const uint32_t row = min(of_a ? m0 + j * 32 + lane : n0 + (j - 4) * 32 + lane, (of_a ? scales.m : scales.n) - 1);
                    const uintptr_t p = (uintptr_t)(of_a ? scales.a + (size_t)row * scales.lda : scales.b + (size_t)row * scales.ldb) + kb;
                    const uintptr_t last = ((uintptr_t)(of_a ? scales.a_end : scales.b_end) - 1) & ~uintptr_t(3), q = p & ~uintptr_t(3);
                    places |= ((uint32_t)p & 3u) << (2 * j);
                    lo[j] = *reinterpret_cast<const uint32_t *>(q);
                    hi[j] = scales.words ? 0u : *reinterpret_cast<const uint32_t *>(q < last ? q + 4 : last);
                }
            };
            settle();
            if (t < grid.total) fetch();
            bool ok = true;
            while (t < grid.total) {
                uint32_t w[12];
#pragma unroll
                for (int j = 0; j < 12; ++j) w[j] = j < ROWS ? __funnelshift_r(lo[j < ROWS ? j : 0], hi[j < ROWS ? j : 0], 8 * (places >> (2 * j) & 3u)) : 0u;
                grp += 2;
                settle();
                if (t < grid.total) fetch();
                const uint32_t slot = sg % S::SF_SLOTS;
                ok = wait_warp(&sempty_bar[slot], ((sg / S::SF_SLOTS) & 1u) ^ 1u, err, 33u);
                if (!ok) break;
                // lane l of the 32 keeps rows l, l + 32, l + 64, l + 96 in its 16 bytes
                uint4 *dst = reinterpret_cast<uint4 *>(smem + S::STAGES * S::STAGE_BYTES + slot * S::SF_BYTES);
                dst[lane] = make_uint4(w[0], w[1], w[2], w[3]);
                dst[32 + lane] = make_uint4(w[4], w[5], w[6], w[7]);
                if (S::N > 128) dst[64 + lane] = make_uint4(w[8], w[9], w[10], w[11]);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) {
                    if (CG == 2) arrive_cluster_release(leader_addr(&sfull_bar[slot]));
                    else mbar_arrive(&sfull_bar[slot]);
                }
                sg += 2;
            }
        }
    } else {
        // ---------------- epilogue: warp w reads the lanes 32 (w mod 4) .. of the accumulator, warps 0-3 the first half of
        // the columns, 4-7 the second ------------------------------------------------------------------------------------
        const int quarter = warp & 3, half = warp >> 2;
        Staging staging{smem + S::STAGES * S::STAGE_BYTES + S::SF_ROOM + warp * 4096, 0u};
        Epi epi(epi_args, staging, &map_out, lane);
        const CUtensorMap *out2 = nullptr;
        if constexpr (DUAL) out2 = &second.map_out;
        Epi2 epi2(second.epi, staging, out2, lane);
        uint32_t it = 0;
        bool ok = true;
        uint32_t mi = 0, ni = 0, si = 0;          // place of the next tile
        auto look_ahead = [&](uint32_t t) {
            if (t >= grid.total) return;
            locate(grid, t, mi, ni, si);
            epi.ahead(mi * S::M + rank * 128 + quarter * 32);
        };
        auto finish_tile = [&](const Grid &gr, auto &e, auto &&then) {
            const int chunks = (int)gr.tile_n / 32, c0 = half ? (chunks + 1) / 2 : 0, c1 = half ? chunks : (chunks + 1) / 2;
            const uint32_t acc = it & 1u, col = ni * gr.tile_n;
            e.begin(mi * S::M + rank * 128 + quarter * 32, col, si, ni * 2 + half);
            then();
            ok = wait_warp(&tfull_bar[acc], (it >> 1) & 1u, err, 34u);
            if (!ok) return;
            fence_after();
            const uint32_t src = tmem + ((uint32_t)(32 * quarter) << 16) + acc * S::N;
            auto release = [&]() {          // the last read of this warp is done: the accumulator can be written again
                fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (CG == 2) arrive_cluster(leader_addr(&tempty_bar[acc]));
                    else mbar_arrive(&tempty_bar[acc]);
                }
            };
            uint32_t r0[32], r1[32];        // one chunk is worked on while the next one is read
            if (c0 < c1) {
                tmem_ld32(r0, src + c0 * 32);
                tmem_wait_ld();
            }
            if (c1 - c0 <= 1) release();
            for (int c = c0; c < c1; c += 2) {
                if (c + 1 < c1) tmem_ld32(r1, src + (c + 1) * 32);
                e.chunk(r0, col + c * 32);
                if (c + 1 < c1) {
                    tmem_wait_ld();
                    if (c + 2 < c1) tmem_ld32(r0, src + (c + 2) * 32);
                    else release();
                    e.chunk(r1, col + (c + 1) * 32);
                    if (c + 2 < c1) {
                        tmem_wait_ld();
                        if (c + 3 >= c1) release();
                    }
                }
            }
            e.end();
        };
        look_ahead(group);
        walk(ok, [&](uint32_t t) { finish_tile(grid, epi, [&] { look_ahead(t + groups); }); ++it; },
             [&](uint32_t t) {
                 if constexpr (DUAL) { locate(second.grid, t, mi, ni, si); finish_tile(second.grid, epi2, [] {}); ++it; }
             });
        epi.finish();
        epi2.finish();
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
