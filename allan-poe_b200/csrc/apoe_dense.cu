// Operators over dense query and document vectors: 8-bit rows with a power-of-two scale for each block of 128 values, the
// scores of such rows against each other, and the softmax loss of queries over all documents with its gradients.
//
//   quantize    q = e4m3(x 2^-e), e the smallest exponent (>= -126) with max |x| of the block <= 448 * 2^e
//   scores      S = alpha * sum over blocks of 2^(ea + eb) <qa, qb>
//   loss        l[t][v] = scale <x_t, w_v>;  lse_t = log sum_v exp l[t][v];  loss_t = lse_t - l[t][target_t]
//   gradients   G[t][v] = grad_t (exp(l[t][v] - lse_t) - [v = target_t]);  dX = scale G W;  dW = scale G^T X
//
// The products run on the tile engine (apoe_tile.cuh).  Neither the scores' scaled operands nor the logits of the loss are
// ever held whole: the loss keeps a running maximum and sum per row and column tile, the gradients recompute the logits of
// one piece of the documents at a time.
//
// Measured on the device: quantize 200 000 x 1024 f32 151 us (6.8 TB/s, bound by memory); scores 8192 x 65 536 x 1024 to bf16
// 473-491 us (2.2 PFLOP/s; 2.6 without the epilogue; 569 us per call back to back, under the power cap); loss 8192 x 100 003 x 1024
// bf16 1.00-1.03 ms (1.65 PFLOP/s, the tensor pipe 95 % active); loss and gradients 4096 x 50 021 x 1024 bf16 1.10-1.13 ms
// (1.5 PFLOP/s with the logits made twice; 89 to 95 %).  Beside these the join of a row takes 3 to 7 us, the prepared copy and
// the last rounding 3 to 7 us each.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>

#include "apoe_tile.cuh"

namespace apoe {

using tile::Grid;
using tile::Scales;

constexpr uint32_t kNoTarget = 0xFFFFFFFFu;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;       // maximum of nothing: below every logit, and differences to it are not NaN
constexpr uint32_t kAll = 0xFFFFFFFFu;

__device__ uint32_t dense_error_word;   // raised by a kernel whose bounded wait ran out; read by ap_dense_check_status

struct DeviceScope {   // calls leave the caller's current device as it was
    int prev = -1;
    ~DeviceScope() { if (prev >= 0) cudaSetDevice(prev); }
    int enter(int device) {
        AP_CUDA(cudaGetDevice(&prev));
        if (prev == device) { prev = -1; return AP_OK; }
        const cudaError_t e = cudaSetDevice(device);
        if (e != cudaSuccess) { prev = -1; return fail(AP_ERR_CUDA, "cudaSetDevice(%d) failed: %s", device, cudaGetErrorString(e)); }
        return AP_OK;
    }
};

template <class T> struct Half16;
template <> struct Half16<__half> {
    static constexpr int kind = tile::kF16;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_half2(lo, hi); }
    static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<__half2 *>(&v)); }
    static __device__ __forceinline__ __half cast(float v) { return __float2half_rn(v); }
};
template <> struct Half16<__nv_bfloat16> {
    static constexpr int kind = tile::kBf16;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&p);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162 *>(&v)); }
    static __device__ __forceinline__ __nv_bfloat16 cast(float v) { return __float2bfloat16_rn(v); }
};

// ---------------------------------------------------------------------------------------------------------------------
// 8-bit rows
// ---------------------------------------------------------------------------------------------------------------------
// Exponent of a block from its largest magnitude a = 1.f * 2^E: the smallest e with a <= 448 * 2^e = 1.75 * 2^(e + 8), kept
// at or above -126 so that 2^-e is a normal float (blocks below 448 * 2^-126 then use fewer of the 8 bits).  Exact: read
// from the bits.  An infinity counts as 2^128: its quantised value times its scale overflows back to infinity.
__device__ __forceinline__ int block_exponent(float a) {
    const uint32_t b = __float_as_uint(a);
    return max((int)(b >> 23) - 127 - ((b & 0x7FFFFFu) <= 0x600000u ? 8 : 7), -126);
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {   // nearest even; beyond 448: 448; NaN stays NaN
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
template <class T> __device__ __forceinline__ float load_as_float(const T *p);
template <> __device__ __forceinline__ float load_as_float<float>(const float *p) { return *p; }
template <> __device__ __forceinline__ float load_as_float<__half>(const __half *p) { return __half2float(*p); }
template <> __device__ __forceinline__ float load_as_float<__nv_bfloat16>(const __nv_bfloat16 *p) { return __bfloat162float(*p); }

struct QuantArgs {
    const void *src;
    uint8_t *q, *scale;
    size_t lds, ldq, ldsc;     // row strides: elements of src, bytes of q and scale
    uint32_t items;            // rows x blocks, below 2^31
    uint32_t dim, blocks;
    uint32_t magic, shift;     // item / blocks = umulhi(item, magic) >> shift, for items below 2^31
};

// One pass, bound by memory where the arithmetic of rows stays small.  A lane holds 16 bytes of a block: the 32 lanes of a warp
// one block of f32, two blocks of f16 or bf16; shuffles give each block's maximum.  A warp has four such loads in flight, of
// neighbouring blocks; one round per warp (a persistent grid with the next round's loads ahead of the current one's work was
// slower: 217 to 281 us instead of 149 for 200 000 x 1024 f32, by its registers).
//   kFlat: whole blocks, rows back to back on both sides: the matrix is one row of blocks (6.9 TB/s at 200 000 x 1024 f32)
//   kUnits: rows of whole 16-byte units on 16-byte boundaries;  kAny: the rest, value by value where it has to be
enum : int { kFlat, kUnits, kAny };
constexpr int kQuantUnroll = 4;
template <class T, int MODE>
__global__ void __launch_bounds__(256) quantize_kernel(const QuantArgs a) {
    constexpr int V = 16 / (int)sizeof(T), LANES = 128 / V, PER = 32 / LANES;   // values of a lane, lanes and blocks of a load
    constexpr uint32_t STEP = kQuantUnroll * PER;
    const uint32_t lane = threadIdx.x & 31, sub = lane / LANES, c0 = (lane % LANES) * V;
    const uint32_t warp = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    tile::pdl_wait();
    tile::pdl_launch();
    const uint32_t it0 = warp * STEP + sub;
    uint32_t row[kQuantUnroll], c[kQuantUnroll];      // first value of the lane: row, and place in it (kFlat: block, 0)
    uint4 raw[kQuantUnroll];
    auto live = [&](int u) { return it0 + u * PER < a.items; };
#pragma unroll
    for (int u = 0; u < kQuantUnroll; ++u) {
        const uint32_t it = it0 + u * PER;
        row[u] = MODE == kFlat || a.blocks == 1 ? it : __umulhi(it, a.magic) >> a.shift;
        c[u] = (MODE == kFlat ? 0u : (it - row[u] * a.blocks) * 128) + c0;
        raw[u] = make_uint4(0u, 0u, 0u, 0u);
        if (!live(u) || (MODE != kFlat && c[u] >= a.dim)) continue;
        const T *p = static_cast<const T *>(a.src) + (size_t)row[u] * (MODE == kFlat ? 128 : a.lds) + c[u];
        if (MODE != kAny) raw[u] = __ldcs(reinterpret_cast<const uint4 *>(p));
        else {
            uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (c[u] + i < a.dim) {
                    if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(p[i]);
                    else w[i / 2] |= (uint32_t)*reinterpret_cast<const uint16_t *>(p + i) << (16 * (i & 1));
                }
            raw[u] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    uint8_t mine = 0, *at = nullptr;
#pragma unroll
    for (int u = 0; u < kQuantUnroll; ++u) {
        float v[V];
        const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(w[i]);
            else { const float2 f = Half16<T>::unpack(w[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
        }
        float m = 0.0f;                                  // a NaN is never taken: fmaxf returns the other one
#pragma unroll
        for (int i = 0; i < V; ++i) m = fmaxf(m, fabsf(v[i]));
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kAll, m, o));
        const int e = block_exponent(m);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
        if (!live(u)) continue;
        if (lane % LANES == (uint32_t)u) {
            mine = (uint8_t)(e + 127);
            at = a.scale + (MODE == kFlat ? row[u] : (size_t)row[u] * a.ldsc + c[u] / 128);
        }
        if (MODE != kFlat && c[u] >= a.dim) continue;
        uint32_t p[V / 4];
#pragma unroll
        for (int i = 0; i < V / 4; ++i)
            p[i] = e4m3x2(v[4 * i] * down, v[4 * i + 1] * down) | (e4m3x2(v[4 * i + 2] * down, v[4 * i + 3] * down) << 16);
        uint8_t *o = a.q + (size_t)row[u] * (MODE == kFlat ? 128 : a.ldq) + c[u];
        if (MODE != kAny) {
            if constexpr (V == 4) *reinterpret_cast<uint32_t *>(o) = p[0];
            else *reinterpret_cast<uint2 *>(o) = make_uint2(p[0], p[1]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) if (c[u] + i < a.dim) o[i] = (uint8_t)(p[i / 4] >> (8 * (i & 3)));
        }
    }
    if (at) *at = mine;      // the scale bytes of the warp's blocks in one store
}

// ---------------------------------------------------------------------------------------------------------------------
// epilogues of the tile engine
// ---------------------------------------------------------------------------------------------------------------------
// Stores a tile through the warp's 4 KB of shared memory, in boxes of 32 rows x 64 bytes (16-byte units exchanged as the
// 64-byte TMA swizzle does, so writing them has no bank conflicts).  Two boxes are in flight: one leaves by TMA while the next
// is written; the tensor map cuts off rows that lie outside, but columns only by 16 bytes.  So the last columns of a row that
// ends inside a box, and all of an output whose rows do not start on 16-byte boundaries, are written element by element.
template <class T>
struct StoreEpi {
    struct Args {
        T *out;                      // results of the splits: stack of m x n matrices, only the first one without `tma`
        size_t ld;                   // elements
        uint32_t m, n;
        float alpha;
        const float *alpha_dev;      // another factor, read on the device (may be null)
        uint32_t add;                // f32 with `tma` only: add to what is there
        uint32_t tma;
        uint32_t padded;             // what follows a row up to the next 16 bytes may be overwritten
    };
    static constexpr int UNITS = (int)sizeof(T) / 2;       // boxes of 32 columns
    static constexpr int COLS = 32 / UNITS;                // columns of a box
    const Args &a;
    tile::Staging &st;
    const CUtensorMap *map;
    int lane;
    float alpha;
    uint32_t row0 = 0, split = 0;
    __device__ __forceinline__ StoreEpi(const Args &args, tile::Staging &staging, const CUtensorMap *out, int lane_) : a(args), st(staging), map(out), lane(lane_) {
        alpha = a.alpha_dev ? a.alpha * *a.alpha_dev : a.alpha;
    }
    __device__ __forceinline__ void ahead(uint32_t) {}
    __device__ __forceinline__ void begin(uint32_t r0, uint32_t, uint32_t s, uint32_t) { row0 = r0; split = s; }
    __device__ __forceinline__ void end() {}
    // shared memory is given up when the copies have read it; that they are written is part of the kernel's end
    __device__ __forceinline__ void finish() { if (lane == 0) tile::store_wait_read<0>(); }
    __device__ __forceinline__ void chunk(uint32_t (&r)[32], uint32_t col) {
#pragma unroll
        for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * alpha);
        put(r, col);
    }
    __device__ __forceinline__ void put(const uint32_t (&r)[32], uint32_t col) {
        if (row0 >= a.m) return;                           // uniform over the warp, as all conditions but the lane's own
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const uint32_t c = col + u * COLS;
            if (c >= a.n) return;
            uint8_t *box = st.base + (st.boxes & 1) * 2048;
            if (st.boxes >= 2) {                              // the box written two rounds ago has left
                if (lane == 0) tile::store_wait_read<1>();
                __syncwarp();
            }
            ++st.boxes;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t p[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (sizeof(T) == 4) p[i] = r[16 * u + 4 * j + i];
                    else p[i] = Half16<T>::pack(__uint_as_float(r[8 * j + 2 * i]), __uint_as_float(r[8 * j + 2 * i + 1]));
                }
                *reinterpret_cast<uint4 *>(box + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = make_uint4(p[0], p[1], p[2], p[3]);
            }
            if (a.tma && (a.padded || c + COLS <= a.n)) {
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) {
                    if (sizeof(T) == 4 && a.add) tile::add_3d(map, box, (int)c, (int)row0, (int)split);
                    else tile::store_3d(map, box, (int)c, (int)row0, (int)split);
                    tile::store_commit();
                }
            } else {
                __syncwarp();
                const uint32_t rows = min(32u, a.m - row0);
                constexpr int PER = 16 / (int)sizeof(T), RPI = 32 / COLS;      // values of a unit, rows a pass covers
                const int k = lane % COLS;
                T *o = a.out + (size_t)row0 * a.ld + c + k;
                const bool in = c + k < a.n;
#pragma unroll 8
                for (int i = 0; i < 32 / RPI; ++i) {
                    const uint32_t row = i * RPI + lane / COLS;
                    const T v = *reinterpret_cast<const T *>(box + row * 64 + (((k / PER) ^ ((row >> 1) & 3)) << 4) + (k % PER) * sizeof(T));
                    if (in && row < rows) o[(size_t)row * a.ld] = v;
                }
                if (lane == 0) tile::store_commit();       // an empty group: the wait above counts one group per box
                __syncwarp();
            }
        }
    }
};

__device__ __forceinline__ float exp2_fast(float x) {   // 2^x, 2 ulp; results below 2^-126 become 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {   // a NaN is never taken
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// two fp32 operations in one instruction
struct Pair { uint64_t v; };
__device__ __forceinline__ Pair pair(float lo, float hi) { Pair p; asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(lo), "f"(hi)); return p; }
__device__ __forceinline__ float2 split(Pair p) { float2 f; asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p.v)); return f; }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) { Pair d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return d; }
__device__ __forceinline__ Pair add2(Pair a, Pair b) { Pair d; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v)); return d; }
__device__ __forceinline__ Pair mul2(Pair a, Pair b) { Pair d; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v)); return d; }

// Running maximum and sum of a row over the columns of a tile, the target's column left out: the target's own logit is computed
// apart and more exactly, because the loss is a difference against it.  The maximum m is one of the products s themselves
// (of -s for a negative scale), the sum one of 2^((s - m) |c|), c = scale * log2 e: a difference of products near each other is
// exact, while a maximum of l = c s would be rounded, by more than an exponential can bear where logits are beyond 2^31.
struct LseEpi {
    static __device__ __forceinline__ float weight(float c) { return fmaxf(fabsf(c), 1.4e-45f); }   // 0: minus infinity has to stay that
    struct Args {
        float2 *part;            // [rows][parts]: maximum and sum
        const uint32_t *target;
        uint32_t parts, m, n, col0;   // col0: document of this piece's first column
        float c;                 // scale * log2 e
    };
    const Args &a;
    int lane;
    uint32_t row = 0, part = 0, tgt = 0, next = kNoTarget;
    float top = 0.f, sum = 0.f;
    __device__ __forceinline__ LseEpi(const Args &args, tile::Staging &, const CUtensorMap *, int lane_) : a(args), lane(lane_) {}
    __device__ __forceinline__ void ahead(uint32_t r0) { next = r0 + lane < a.m ? a.target[r0 + lane] : kNoTarget; }
    __device__ __forceinline__ void begin(uint32_t r0, uint32_t, uint32_t, uint32_t p) {
        row = r0 + lane; part = p;
        tgt = next - a.col0;              // a target of another piece is none of this one's columns, and kNoTarget none at all
        top = kLowest; sum = 0.f;
    }
    __device__ __forceinline__ void chunk(uint32_t (&r)[32], uint32_t col) {
        if (a.c < 0.f)
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] ^= 0x80000000u;
        const uint32_t at = tgt - col, cols = a.n > col ? a.n - col : 0u;
        if (__any_sync(kAll, at < 32u) || cols < 32u) {
#pragma unroll
            for (int j = 0; j < 32; ++j) if (at == (uint32_t)j || (uint32_t)j >= cols) r[j] = 0xFF800000u;
        }
        // several chains for the maximum and the sum: one would make the warp wait for its own last result 32 times over
        float m4[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) m4[j] = __uint_as_float(r[j]);
#pragma unroll
        for (int j = 4; j < 28; j += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k) m4[k] = max3(m4[k], __uint_as_float(r[j + k]), __uint_as_float(r[j + 4 + k]));
        const float m1 = max3(m4[0], __uint_as_float(r[28]), __uint_as_float(r[29])), m2 = max3(m4[1], __uint_as_float(r[30]), __uint_as_float(r[31]));
        const float c = weight(a.c), m = fmaxf(top, fmaxf(max3(m1, m2, m4[2]), m4[3]));
        const Pair cc = pair(c, c), mm = pair(-m, -m);
        Pair s[4] = {pair(0.f, 0.f), pair(0.f, 0.f), pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
            const float2 x = split(mul2(add2(pair(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), mm), cc));
            s[(j >> 1) & 3] = add2(s[(j >> 1) & 3], pair(exp2_fast(x.x), exp2_fast(x.y)));
        }
        const float2 f = split(add2(add2(s[0], s[1]), add2(s[2], s[3])));
        sum = sum * exp2_fast((top - m) * c) + (f.x + f.y);
        top = m;
    }
    __device__ __forceinline__ void finish() {}
    __device__ __forceinline__ void end() { if (row < a.m) a.part[(size_t)row * a.parts + part] = make_float2(top, sum); }
};

// One piece of G, times a power of two that brings its largest value to 2^14 (f16 keeps small ones normal); a rounding
// to 16 bits per element, the operands of the two products that follow.
template <class T>
struct GradEpi {
    struct Args {
        typename StoreEpi<T>::Args out;
        const uint32_t *target;
        const float *loss, *lse, *grad;
        const float *factor;     // the power of two
        uint32_t col0, docs;
        float c;
        float base, base_rest;   // what lse is taken times: log2 e as c has it, as the sum of two floats
    };
    const Args &a;
    StoreEpi<T> store;
    uint32_t tgt = 0, next = kNoTarget;
    float lse2 = 0.f, g = 0.f, at_target = 0.f, grad = 0.f, lse = 0.f, loss = 0.f, factor;
    __device__ __forceinline__ GradEpi(const Args &args, tile::Staging &staging, const CUtensorMap *out, int lane) : a(args), store(args.out, staging, out, lane) {
        factor = *a.factor;
    }
    __device__ __forceinline__ void ahead(uint32_t r0) {
        const uint32_t row = min(r0 + store.lane, a.out.m - 1);      // past the last row: nothing is stored
        next = a.target[row];
        grad = a.grad[row]; lse = a.lse[row]; loss = a.loss[row];
    }
    __device__ __forceinline__ void begin(uint32_t r0, uint32_t n0, uint32_t s, uint32_t p) {
        store.begin(r0, n0, s, p);
        const bool has = next < a.docs;
        tgt = has ? next - a.col0 : kNoTarget;
        g = has ? grad * factor : 0.f;
        at_target = has ? g * expm1f(-loss) : 0.f;                  // -(1 - p) of the target, exact where p is near 1
        // p = 2^(c s - base lse), base = c / scale: with c a rounding of scale * log2 e, lse has to be taken times the same rounding,
        // or the whole row is off by 2^-24 of its logits (an f16 step at 8000).  What lse2 loses as a float goes into the row's
        // factor (in 64 bits this cost 3 % of 2000 x 20 000 x 128).
        lse2 = has ? lse * a.base : 0.f;
        const float lost = fmaf(lse, a.base, -lse2) + lse * a.base_rest;
        if (fabsf(lost) < 64.f) g *= exp2_fast(-lost);              // more only where lse itself is off by as much; nor infinite, nor NaN
    }
    __device__ __forceinline__ void end() {}
    __device__ __forceinline__ void finish() { store.finish(); }
    __device__ __forceinline__ void chunk(uint32_t (&r)[32], uint32_t col) {
        const bool live = g != 0.f;      // rows without a target may hold anything, NaN included: their G is zero
        const Pair cc = pair(a.c, a.c), ll = pair(-lse2, -lse2), gg = pair(g, g);
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
            const float2 x = split(fma2(pair(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), cc, ll));
            const float2 y = split(mul2(gg, pair(exp2_fast(x.x), exp2_fast(x.y))));
            r[j] = live ? __float_as_uint(y.x) : 0u;
            r[j + 1] = live ? __float_as_uint(y.y) : 0u;
        }
        const uint32_t at = tgt - col;
        if (__any_sync(kAll, at < 32u)) {
#pragma unroll
            for (int j = 0; j < 32; ++j) if (at == (uint32_t)j) r[j] = __float_as_uint(at_target);
        }
        store.put(r, col);
    }
};

// ---------------------------------------------------------------------------------------------------------------------
// loss: joining the tiles, preparing and finishing the gradients
// ---------------------------------------------------------------------------------------------------------------------
struct JoinArgs {
    const float2 *part;
    float2 *carry;               // [rows] running maximum and sum over the pieces before this one
    const void *x, *w;
    size_t ldx, ldw;
    const uint32_t *target;
    float *loss, *lse;
    uint32_t rows, docs, dim, parts, first, last;
    float scale, c;              // c: what the tiles took the products times
};
// One warp per row.  With z = log(sum of the others) - (target's logit): loss = log(1 + e^z), which keeps its digits where the
// row is nearly certain (z << 0) and where it is hopeless; lse = target's logit + loss.
template <class T>
__global__ void __launch_bounds__(256) loss_join_kernel(const JoinArgs a) {
    const uint32_t row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const uint32_t t = a.last && row < a.rows ? a.target[row] : kNoTarget;
    double dot = 0.0;                    // the target's logit, from inputs that are complete: while the tiles are still at work
    if (t < a.docs) {
        // products of 16-bit values are exact; eight of them are summed in fp32, the sums in 64 bits
        const T *x = static_cast<const T *>(a.x) + (size_t)row * a.ldx, *w = static_cast<const T *>(a.w) + (size_t)t * a.ldw;
        uint32_t i = lane * 8;
        for (; i + 8 <= a.dim; i += 256) {
            const uint4 u = *reinterpret_cast<const uint4 *>(x + i), v = *reinterpret_cast<const uint4 *>(w + i);
            const uint32_t us[4] = {u.x, u.y, u.z, u.w}, vs[4] = {v.x, v.y, v.z, v.w};
            float d0 = 0.f, d1 = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 fu = Half16<T>::unpack(us[k]), fv = Half16<T>::unpack(vs[k]);
                d0 = fmaf(fu.x, fv.x, d0); d1 = fmaf(fu.y, fv.y, d1);
            }
            dot += (double)(d0 + d1);
        }
        for (uint32_t k = i; k < min(i + 8, a.dim); ++k) dot += (double)(load_as_float(x + k) * load_as_float(w + k));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(kAll, dot, o);
    }
    tile::pdl_wait();
    tile::pdl_launch();
    if (row >= a.rows) return;
    float top = kLowest, sum = 0.f;
    const float c = LseEpi::weight(a.c);
    const auto join = [&](float t2, float s2) {
        const float m = fmaxf(top, t2);
        sum = sum * exp2f((top - m) * c) + s2 * exp2f((t2 - m) * c);
        top = m;
    };
    const float2 *p = a.part + (size_t)row * a.parts;
    for (uint32_t i = lane; i < a.parts; i += 32) {
        const float2 e = p[i];
        join(e.x, e.y);
    }
    if (lane == 0 && !a.first) {
        const float2 e = a.carry[row];
        join(e.x, e.y);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float t2 = __shfl_xor_sync(kAll, top, o), s2 = __shfl_xor_sync(kAll, sum, o);
        join(t2, s2);
    }
    if (!a.last) { if (lane == 0) a.carry[row] = make_float2(top, sum); return; }
    float loss = 0.f, lse = 0.f;
    if (t < a.docs) {
        // c is a rounding of scale * log2 e, but the sum holds differences only
        const double at = (double)a.scale * dot;
        const float z = (float)(fabs((double)a.scale) * (double)top + log2((double)sum) * 0.6931471805599453 - at);   // one document: minus infinity, loss 0
        loss = z > 0.f ? z + log1pf(expf(-z)) : log1pf(expf(z));  // a NaN stays one
        lse = (float)(at + (double)loss);
    } else if (t != kNoTarget) loss = lse = __int_as_float(0x7FFFFFFF);
    if (lane == 0) { a.loss[row] = loss; a.lse[row] = lse; }
}

struct PrepArgs {
    const void *x;
    void *xc;
    size_t ldx, ldxc;
    const uint32_t *target;
    const float *grad, *loss;
    float *factor;               // [0] the power of two, [1] scale / that
    uint32_t rows, docs, dim;
    float scale;
};
// A copy of the query rows with those that have no target set to zero (0 times whatever a padding row holds would not be 0
// inside a product); block 0 also finds the factor of G from the largest of its values in the rows that count.
template <class T>
__global__ void __launch_bounds__(256) grad_prep_kernel(const PrepArgs a) {
    tile::pdl_wait();
    tile::pdl_launch();
    if (blockIdx.x == 0) {
        // No |G| of a row exceeds that of its target, |grad| (1 - p): where a whole batch is nearly certain, so is the factor
        __shared__ float s[2][8];
        float top = 0.f, g = 0.f;
        for (uint32_t i = threadIdx.x; i < a.rows; i += 256)
            if (a.target[i] < a.docs) {
                const float x = fabsf(a.grad[i]);
                g = fmaxf(g, x);
                top = fmaxf(top, x * -expm1f(-a.loss[i]));
            }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) { top = fmaxf(top, __shfl_xor_sync(kAll, top, o)); g = fmaxf(g, __shfl_xor_sync(kAll, g, o)); }
        if ((threadIdx.x & 31) == 0) { s[0][threadIdx.x >> 5] = top; s[1][threadIdx.x >> 5] = g; }
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int i = 1; i < 8; ++i) { top = fmaxf(top, s[0][i]); g = fmaxf(g, s[1][i]); }
            int e = 0, eg = 0;                                     // top <= 2^e, g <= 2^eg
            if (top > 0.f && top < INFINITY) frexpf(top, &e);
            if (g > 0.f && g < INFINITY) frexpf(g, &eg);
            const int k = max(min(min(14 - e, 126), 120 - eg), -126);   // grad times the factor stays finite
            a.factor[0] = ldexpf(1.f, k);
            a.factor[1] = ldexpf(a.scale, -k);
        }
        return;
    }
    const uint32_t lane = threadIdx.x & 31;
    for (uint32_t row = (blockIdx.x - 1) * 8 + (threadIdx.x >> 5); row < a.rows; row += (gridDim.x - 1) * 8) {
        const bool live = a.target[row] < a.docs;
        const T *x = static_cast<const T *>(a.x) + (size_t)row * a.ldx;
        T *o = static_cast<T *>(a.xc) + (size_t)row * a.ldxc;
        for (uint32_t i = lane * 8; i < a.dim; i += 256) {
            if (i + 8 <= a.dim) *reinterpret_cast<uint4 *>(o + i) = live ? *reinterpret_cast<const uint4 *>(x + i) : make_uint4(0u, 0u, 0u, 0u);
            else for (uint32_t k = i; k < a.dim; ++k) o[k] = live ? x[k] : Half16<T>::cast(0.f);
        }
    }
}

struct FinishArgs {
    const float *part;           // [splits][rows][ldp]
    const float *factor;
    void *dx;
    size_t ldp, ldd;
    uint32_t rows, dim, splits;
};
// dX from the partial sums of the splits (added in a fixed order), rounded once
template <class T>
__global__ void __launch_bounds__(256) grad_finish_kernel(const FinishArgs a) {
    tile::pdl_wait();
    tile::pdl_launch();
    const float f = a.factor[1];
    const uint32_t quads = (a.dim + 3) / 4;
    const uint64_t total = (uint64_t)a.rows * quads;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
        const uint32_t row = (uint32_t)(i / quads), c = (uint32_t)(i - (uint64_t)row * quads) * 4;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint32_t k = 0; k < a.splits; ++k) {
            const float4 v = __ldcs(reinterpret_cast<const float4 *>(a.part + ((size_t)k * a.rows + row) * a.ldp + c));
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        T *o = static_cast<T *>(a.dx) + (size_t)row * a.ldd + c;
        if (c + 4 <= a.dim)
            *reinterpret_cast<uint2 *>(o) = make_uint2(Half16<T>::pack(s.x * f, s.y * f), Half16<T>::pack(s.z * f, s.w * f));
        else {
            const float v[4] = {s.x * f, s.y * f, s.z * f, s.w * f};
            for (uint32_t k = 0; c + k < a.dim; ++k) o[k] = Half16<T>::cast(v[k]);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------------
// rows x cols values, rows `ld` values apart; box = one 128-byte span of columns x box_rows rows, 128-byte swizzle.  Reads
// beyond the extents give zeros.
static int make_map_2d(CUtensorMap *map, int kind, const void *base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows) {
    EncodeTiledFn fn;
    AP_TRY(encode_fn(&fn));
    const uint32_t size = kind == tile::kE4m3 ? 1 : 2;
    const CUtensorMapDataType t = kind == tile::kE4m3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                : kind == tile::kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const cuuint64_t dims[2] = {cols, rows};
    const cuuint64_t strides[1] = {ld * size};
    const cuuint32_t box[2] = {128 / size, box_rows};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(map, t, 2, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(AP_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
    return AP_OK;
}
// a stack of m x n results, written in boxes of 32 rows x 64 bytes
static int make_map_out(CUtensorMap *map, CUtensorMapDataType t, uint32_t size, void *base, uint64_t stack, uint64_t m, uint64_t n, uint64_t ld) {
    EncodeTiledFn fn;
    AP_TRY(encode_fn(&fn));
    const cuuint64_t dims[3] = {n, m, stack};
    const cuuint64_t strides[2] = {ld * size, m * ld * size};
    const cuuint32_t box[3] = {64 / size, 32, 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = fn(map, t, 3, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                          CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(AP_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
    return AP_OK;
}
template <class T> struct MapType;
template <> struct MapType<float> { static constexpr CUtensorMapDataType v = CU_TENSOR_MAP_DATA_TYPE_FLOAT32; };
template <> struct MapType<__half> { static constexpr CUtensorMapDataType v = CU_TENSOR_MAP_DATA_TYPE_FLOAT16; };
template <> struct MapType<__nv_bfloat16> { static constexpr CUtensorMapDataType v = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16; };
template <class T>
static int out_map(CUtensorMap *map, const typename StoreEpi<T>::Args &a, uint32_t stack) {
    return a.tma ? make_map_out(map, MapType<T>::v, sizeof(T), a.out, stack, a.m, a.n, a.ld) : AP_OK;
}
template <class T> static int out_map_of(CUtensorMap *map, const typename StoreEpi<T>::Args &a, uint32_t stack, const StoreEpi<T> *) { return out_map<T>(map, a, stack); }
template <class T> static int out_map_of(CUtensorMap *map, const typename GradEpi<T>::Args &a, uint32_t, const GradEpi<T> *) { return out_map<T>(map, a.out, 1); }
static int out_map_of(CUtensorMap *, const LseEpi::Args &, uint32_t, const LseEpi *) { return AP_OK; }

struct Operand {   // a stored matrix: rows x cols, row stride in values
    const void *base;
    uint64_t rows, cols, ld;
};
static uint32_t ceil_div(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

// A kernel of 256 threads, started while the one before it ends (every kernel here waits for that before it reads or writes)
template <class Args>
static int launch(void (*kernel)(Args), uint32_t grid, const Args &args, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    AP_CUDA(cudaLaunchKernelEx(&cfg, kernel, args));
    return AP_OK;
}

// What a tile costs, in K blocks of a full 16-bit tile (0.39 us on a pair of SMs): its K blocks, whose cost falls more slowly
// than their columns, and 1.5 for its ends; a short K leaves the epilogue (2 us for 256 columns) to wait for.  Measured on
// pairs at K = 4096, us per K block: 16 bits 0.26 / 0.29 / 0.35 / 0.39 at 64 / 128 / 224 / 256 columns, 8 bits 0.34 / 0.36 / 0.40
// at 64 / 128 / 224.  One CTA per tile (few rows) waits for its columns from memory: 8 bits 0.36 / 0.48 / 0.64 / 0.72 at 32 / 128 /
// 192 / 224 columns, 16 bits 0.50 / 0.65 / 0.82 at 128 / 192 / 256.
static double tile_cost(int cg, uint32_t tile_n, uint32_t kblocks, bool scaled = false) {
    const double block = cg == 1 ? std::max((tile_n + 75) / 160.0, scaled ? 0.92 : 0.66)
                                 : scaled ? (tile_n + 900) / 1100.0 : std::max((tile_n + 192) / 448.0, 0.66);
    return std::max(kblocks * block + 1.5, 5.0 * tile_n / 256.0 + 1.0);
}
// Columns of a tile: as many as the shape allows, unless narrower tiles fill the rounds of the persistent grid better
// (1000 x 10007 x 1024: 160 tiles of 256 x 256 on 74 pairs take three rounds, 212 of 256 x 192 three shorter ones).
static uint32_t pick_n(uint32_t most, uint32_t least, int cg, uint32_t m, uint32_t n, uint32_t kblocks, int sms, bool scaled = false) {
    const uint32_t groups = (uint32_t)std::max(1, sms / cg), tiles_m = ceil_div(m, 128 * (uint32_t)cg);
    uint32_t best = most;
    double best_cost = 1e300;
    for (uint32_t w = most; w >= least; w -= 32) {
        const double cost = (double)(((uint64_t)tiles_m * ceil_div(n, w) + groups - 1) / groups) * tile_cost(cg, w, kblocks, scaled);
        if (cost < best_cost * 0.985) { best_cost = cost; best = w; }
    }
    return best;
}

// One product C[m][n] = sum over k of A B^T on one shape: its tensor maps and tiles, K cut into at most `splits` parts.
// K-major operands are stored rows x K, MN-major ones K x rows.
struct Product {
    CUtensorMap a, b, out;
    Grid grid;
};
template <class S, bool AMN, class Epi>
static int make_product(Product *p, const Operand &a, const Operand &b, uint32_t m, uint32_t n, uint32_t k, uint32_t splits, uint32_t tile_n,
                        const typename Epi::Args &epi) {
    // few rows: the rest of the 128 is not loaded (as zeros); what the products make of it is in rows that are not stored
    p->grid.a_rows = S::CG == 1 && !AMN ? std::min<uint32_t>(128, ceil_div(m, 8) * 8) : 128;
    AP_TRY(make_map_2d(&p->a, S::KIND, a.base, a.rows, a.cols, a.ld, AMN ? 64 : p->grid.a_rows));
    AP_TRY(make_map_2d(&p->b, S::KIND, b.base, b.rows, b.cols, b.ld, S::BMN ? 64 : tile_n / S::CG));
    Grid &g = p->grid;
    g.tiles_m = ceil_div(m, S::M);
    g.tile_n = tile_n;
    g.tiles_n = ceil_div(n, tile_n);
    g.kblocks = ceil_div(k, S::K);
    g.kper = ceil_div(g.kblocks, splits);
    const uint32_t parts = ceil_div(g.kblocks, g.kper);
    g.total = g.tiles_m * g.tiles_n * parts;
    AP_TRY(out_map_of(&p->out, epi, parts, static_cast<const Epi *>(nullptr)));
    // row tiles that walk the columns together: all of them while their operand stays in L2 (32 MB of it), else 8
    const uint64_t row_bytes = (uint64_t)S::M * k * (S::SCALED ? 1 : 2);
    g.group_m = std::min<uint32_t>(g.tiles_m, (uint32_t)std::max<uint64_t>(8, (32ull << 20) / row_bytes));
    return AP_OK;
}
template <class S, class Epi, class Epi2>
static int tile_launch(const Product &p, uint32_t total, const Scales &sc, const typename Epi::Args &epi, const tile::Second<Epi2> &second, int sms,
                       uint32_t *err, cudaStream_t st) {
    static std::atomic<uint64_t> allowed{0};    // devices on which this kernel's shared-memory size has been set
    int device = 0;
    AP_CUDA(cudaGetDevice(&device));
    if (device >= 64 || !(allowed.load(std::memory_order_acquire) >> device & 1)) {
        AP_CUDA(cudaFuncSetAttribute(tile::tile_kernel<S, Epi, Epi2>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM));
        if (device < 64) allowed.fetch_or(1ull << device, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(std::min<uint32_t>(total, std::max(1u, (uint32_t)sms / S::CG)) * S::CG);
    cfg.blockDim = dim3(tile::kThreads);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = S::CG; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    AP_CUDA(cudaLaunchKernelEx(&cfg, tile::tile_kernel<S, Epi, Epi2>, p.a, p.b, p.out, p.grid, sc, epi, second, err));
    return AP_OK;
}
template <class S, class Epi>
static int run_product(const Operand &a, const Operand &b, uint32_t m, uint32_t n, uint32_t k, uint32_t tile_n, const Scales &sc,
                       const typename Epi::Args &epi, int sms, uint32_t *err, cudaStream_t st, bool early = false) {
    Product p = {};
    AP_TRY((make_product<S, S::AMN, Epi>(&p, a, b, m, n, k, 1, tile_n, epi)));
    p.grid.early = early;
    return tile_launch<S, Epi, tile::NoSecond>(p, p.grid.total, sc, epi, tile::Second<tile::NoSecond>{}, sms, err, st);
}

// SM count and address of the error word, looked up once per device
static int device_facts(int device, int *sms, uint32_t **err) {
    struct Facts { std::atomic<uint32_t *> err{nullptr}; int sms = 0; };
    static Facts facts[64];
    static std::mutex mu;
    if (device < 0 || device >= 64) return fail(AP_ERR_ARG, "device %d", device);
    Facts &f = facts[device];
    if (!f.err.load(std::memory_order_acquire)) {
        std::lock_guard<std::mutex> lock(mu);
        AP_CUDA(cudaDeviceGetAttribute(&f.sms, cudaDevAttrMultiProcessorCount, device));
        void *p = nullptr;
        AP_CUDA(cudaGetSymbolAddress(&p, dense_error_word));
        f.err.store(static_cast<uint32_t *>(p), std::memory_order_release);
    }
    *sms = f.sms;
    *err = f.err.load(std::memory_order_acquire);
    return AP_OK;
}
static bool aligned(const void *p, uint64_t stride_bytes, uint64_t to) { return (uintptr_t)p % to == 0 && stride_bytes % to == 0; }
static bool words(const void *a, const void *b = nullptr, const void *c = nullptr, const void *d = nullptr) {   // all on 4-byte boundaries
    return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d) & 3) == 0;
}
static int elem_size(uint32_t type) { return type == AP_TYPE_F32 ? 4 : (type == AP_TYPE_F16 || type == AP_TYPE_BF16) ? 2 : 0; }

// ---- loss: how the work is cut ------------------------------------------------------------------------------------------
constexpr uint32_t kTileN = 256;
static size_t round256(size_t b) { return (b + 255) & ~size_t(255); }

struct ForwardPlan { uint32_t piece, parts; size_t part_bytes, bytes; };
// Narrow tiles only where few documents leave SMs without work: the partial results of a row grow with their number.  Tiles down to
// 32 columns instead of 128: 128 x 4096 x 1024 9.2 us instead of 10.2, 128 x 10 000 10.7 instead of 11.0; within 3 % of each
// other from 256 rows on, the same from 20 000 documents on.
static uint32_t least_n(uint32_t docs) { return docs <= 16384 ? 32 : 128; }
// The tiles' maxima and sums, 8 bytes per row and half a tile, by pieces of the documents: at most 64 MB, or 512 bytes a row where
// that is more (from 131 072 rows on).  A piece has at least 8192 documents (with pieces of 1024, 2^20 x 4096 x 128 took 3.16 ms
// instead of 2.46), and where that many in narrow tiles would need more, its tiles are wider: the row tiles alone fill the SMs.
static ForwardPlan forward_plan(uint32_t rows, uint32_t docs) {
    ForwardPlan p;
    const uint64_t fit = (64ull << 20) / ((uint64_t)rows * 16);         // tiles of a row in 64 MB
    uint32_t least = least_n(docs);
    while (least < kTileN && fit * least < std::min<uint64_t>(docs, 32 * kTileN)) least *= 2;
    p.piece = (uint32_t)std::min<uint64_t>((uint64_t)ceil_div(docs, kTileN) * kTileN, std::max<uint64_t>(fit * least, 32 * kTileN));
    p.parts = 2 * ceil_div(std::min(p.piece, docs), least);
    p.part_bytes = round256((size_t)rows * p.parts * 8);
    p.bytes = p.part_bytes + round256((size_t)rows * 8);
    return p;
}

// The two products of a piece's gradients share a launch: the parts of dX (K = the piece's documents, cut into `splits`), then
// the tiles of dW (K = the rows).  The groups of SMs that get a part of dX less get `lead` tiles of dW more.
struct Cut { uint32_t splits, n; };        // parts of dX's K; columns of a tile
struct Deal { uint32_t lead; double cost; };
static Deal deal(uint32_t groups, uint32_t tx, uint32_t tw, double cx, double cw) {
    const uint32_t each = tx / groups, rest = tx % groups, light = groups - rest;
    const uint32_t lead = rest ? std::min<uint32_t>((uint32_t)(cx / cw + 0.5), tw / light) : 0, left = tw - lead * light;
    const auto turns = [&](uint32_t g) { return left > g ? (left - g - 1) / groups + 1 : 0; };
    const double heavy = rest ? (each + 1) * cx + turns(0) * cw : 0.0, lighter = each * cx + (lead + turns(rest)) * cw;
    return {lead, std::max(heavy, lighter)};
}
static Deal deal_of(uint32_t rows, uint32_t docs, uint32_t dim, const Cut &c, int sms) {
    const uint32_t cg = rows <= 128 ? 1 : 2, groups = std::max(1u, (uint32_t)sms / cg), cols = ceil_div(dim, c.n), kx = ceil_div(docs, 64);
    const uint32_t tx = ceil_div(rows, 128 * cg) * cols * c.splits, tw = ceil_div(docs, 128 * cg) * cols;
    return deal(std::min(groups, tx + tw), tx, tw, tile_cost((int)cg, c.n, ceil_div(kx, c.splits)), tile_cost((int)cg, c.n, ceil_div(rows, 64)));
}
static Cut pick_cut(uint32_t rows, uint32_t docs, uint32_t dim, uint32_t most_splits, int sms) {
    // the narrowest tiles that still cover dim in as few columns of tiles as the widest do
    const uint32_t wide = ceil_div(dim, 256), kx = ceil_div(docs, 64);
    Cut best{1, std::max(32u, ceil_div(ceil_div(dim, wide), 32) * 32)};
    double best_cost = 1e300;
    for (uint32_t s = 1; s <= most_splits && (s == 1 || kx / s >= 8); ++s) {
        if (ceil_div(kx, ceil_div(kx, s)) != s) continue;
        const Cut c{s, best.n};
        // a part is a matrix of fp32 sums that is written and read once more: its time at 6.5 TB/s, in units of 0.39 us
        const double cost = deal_of(rows, docs, dim, c, sms).cost + (s > 1 ? 2.0 + s * (double)rows * dim * 6.0 / 6.5e12 / 0.39e-6 : 0.0);
        if (cost < best_cost * 0.98) { best_cost = cost; best.splits = s; }
    }
    return best;
}

struct BackwardPlan { uint32_t piece, splits; bool direct; size_t ldx, ldg, ldp, x_off, g_off, p_off, bytes; };
static BackwardPlan backward_plan(uint32_t rows, uint32_t docs, uint32_t dim, int sms) {
    BackwardPlan p;
    // documents per piece: G of at most 512 MB, or 4096 bytes a row where that is more: at least 2048 documents, 4 GB at 2^20
    // rows.  Every piece adds to the sums of dX once more; both gradients with 32 / 128 / 512 MB: 4096 x 50 021 x 1024 0.95 / 0.87 /
    // 0.81 ms, 4096 x 50 021 x 128 450 / 351 / 314 us, 2000 x 20 000 x 128 87 / 72 / 72 us.
    const uint64_t most = std::max<uint64_t>(8, (512ull << 20) / ((uint64_t)rows * 2) / kTileN);
    p.piece = (uint32_t)std::min<uint64_t>(most, ceil_div(docs, kTileN)) * kTileN;
    p.splits = pick_cut(rows, std::min(p.piece, docs), dim, 32, sms).splits;
    p.direct = p.splits == 1 && p.piece >= docs;     // one part of one piece: dX needs no sums of its own
    p.ldx = (dim + 7) / 8 * 8;
    p.ldg = p.piece;
    p.ldp = (dim + 3) / 4 * 4;
    p.x_off = 256;
    p.g_off = p.x_off + round256((size_t)rows * p.ldx * 2);
    p.p_off = p.g_off + round256((size_t)rows * p.ldg * 2);
    p.bytes = p.p_off + (p.direct ? 0 : round256((size_t)p.splits * rows * p.ldp * 4));
    return p;
}

struct LossCall {
    uint32_t rows, docs, dim;
    const void *x, *w;
    uint64_t ldx, ldw;
    const uint32_t *target;
    float scale;
    int sms;
    uint32_t *err;
    cudaStream_t st;
};

template <class T, int CG>
static int forward_run(const LossCall &c, const ForwardPlan &p, uint8_t *ws, float *loss, float *lse) {
    using S = tile::Shape<Half16<T>::kind, CG, kTileN>;
    float2 *part = reinterpret_cast<float2 *>(ws), *carry = reinterpret_cast<float2 *>(ws + p.part_bytes);
    const Operand x{c.x, c.rows, c.dim, c.ldx};
    for (uint32_t v0 = 0; v0 < c.docs; v0 += p.piece) {
        const uint32_t n = std::min(p.piece, c.docs - v0);
        const Operand w{static_cast<const T *>(c.w) + (size_t)v0 * c.ldw, n, c.dim, c.ldw};
        const uint32_t least = std::max(least_n(c.docs), ceil_div(ceil_div(n, p.parts / 2), 32) * 32);     // as many tiles as there is room for
        const uint32_t tn = pick_n(kTileN, least, CG, c.rows, n, ceil_div(c.dim, 64), c.sms);
        LseEpi::Args ea{part, c.target, 2 * ceil_div(n, tn), c.rows, n, v0, c.scale * kLog2e};
        AP_TRY((run_product<S, LseEpi>(x, w, c.rows, n, c.dim, tn, Scales{}, ea, c.sms, c.err, c.st)));
        JoinArgs ja{part, carry, c.x, c.w, c.ldx, c.ldw, c.target, loss, lse, c.rows, c.docs, c.dim, ea.parts, v0 == 0 ? 1u : 0u,
                    v0 + n == c.docs ? 1u : 0u, c.scale, ea.c};
        AP_TRY(launch(loss_join_kernel<T>, ceil_div(c.rows, 8), ja, c.st));
    }
    return AP_OK;
}

// dX (stored by E: sums of parts, or the gradient itself) and dW of one piece in one launch
template <class S, class E, class T>
static int gradients_launch(const LossCall &c, const Cut &cut, const Operand &x, const Operand &w, const Operand &g, uint32_t n,
                            const typename E::Args &xa, const typename StoreEpi<T>::Args &wa) {
    Product px = {}, pw = {};
    AP_TRY((make_product<S, false, E>(&px, g, w, c.rows, c.dim, n, cut.splits, cut.n, xa)));
    AP_TRY((make_product<S, true, StoreEpi<T>>(&pw, g, x, n, c.dim, c.rows, 1, cut.n, wa)));
    const tile::Second<StoreEpi<T>> second{pw.a, pw.b, pw.out, pw.grid, deal_of(c.rows, n, c.dim, cut, c.sms).lead, wa};
    return tile_launch<S, E, StoreEpi<T>>(px, px.grid.total + pw.grid.total, Scales{}, xa, second, c.sms, c.err, c.st);
}

template <class T, int CG>
static int backward_run(const LossCall &c, const BackwardPlan &p, uint8_t *ws, const float *loss, const float *lse, const float *grad, void *dx,
                        uint64_t lddx, void *dw, uint64_t lddw) {
    constexpr int KIND = Half16<T>::kind;
    using SG = tile::Shape<KIND, CG, kTileN>;                       // G: rows x documents, over dim
    using SX = tile::Shape<KIND, CG, kTileN, false, true>;          // dX: rows x dim, over documents (dW: A MN-major as well)
    float *factor = reinterpret_cast<float *>(ws);
    T *xc = reinterpret_cast<T *>(ws + p.x_off), *g = reinterpret_cast<T *>(ws + p.g_off);
    float *part = reinterpret_cast<float *>(ws + p.p_off);
    PrepArgs pa{c.x, xc, c.ldx, p.ldx, c.target, grad, loss, factor, c.rows, c.docs, c.dim, c.scale};
    AP_TRY(launch(grad_prep_kernel<T>, 1 + std::min<uint32_t>(ceil_div(c.rows, 8), 4 * (uint32_t)c.sms), pa, c.st));
    const Operand x{xc, c.rows, c.dim, p.ldx}, given{c.x, c.rows, c.dim, c.ldx};
    for (uint32_t v0 = 0; v0 < c.docs; v0 += p.piece) {
        const uint32_t n = std::min(p.piece, c.docs - v0);
        const Operand w{static_cast<const T *>(c.w) + (size_t)v0 * c.ldw, n, c.dim, c.ldw};
        const Operand go{g, c.rows, n, p.ldg};
        typename GradEpi<T>::Args ga{};
        ga.out.out = g; ga.out.ld = p.ldg; ga.out.m = c.rows; ga.out.n = n; ga.out.alpha = 1.f; ga.out.tma = 1; ga.out.padded = 1;
        ga.target = c.target; ga.loss = loss; ga.lse = lse; ga.grad = grad; ga.factor = factor; ga.col0 = v0; ga.docs = c.docs; ga.c = c.scale * kLog2e;
        const double base = std::isnormal(ga.c) ? (double)ga.c / (double)c.scale : 1.4426950408889634;   // no scale: c s is 0 in any case
        ga.base = (float)base; ga.base_rest = (float)(base - (double)ga.base);
        const uint32_t tn = pick_n(kTileN, 32, CG, c.rows, n, ceil_div(c.dim, 64), c.sms);
        // from the rows as they were given: the logits are under way while the rows are prepared, the epilogue waits
        AP_TRY((run_product<SG, GradEpi<T>>(given, w, c.rows, n, c.dim, tn, Scales{}, ga, c.sms, c.err, c.st, true)));
        typename StoreEpi<T>::Args wa{};
        wa.out = static_cast<T *>(dw) + (size_t)v0 * lddw; wa.ld = lddw; wa.m = n; wa.n = c.dim; wa.alpha = 1.f; wa.alpha_dev = factor + 1;
        wa.tma = aligned(wa.out, lddw * 2, 16);
        Cut cut = pick_cut(c.rows, n, c.dim, p.splits, c.sms);
        if (v0 == 0) cut.splits = p.splits;                         // the first piece writes every part, the others add to some
        if (p.direct) {
            typename StoreEpi<T>::Args xa{};
            xa.out = static_cast<T *>(dx); xa.ld = lddx; xa.m = c.rows; xa.n = c.dim; xa.alpha = 1.f; xa.alpha_dev = factor + 1;
            xa.tma = aligned(dx, lddx * 2, 16);
            return gradients_launch<SX, StoreEpi<T>, T>(c, cut, x, w, go, n, xa, wa);
        }
        typename StoreEpi<float>::Args xa{};
        xa.out = part; xa.ld = p.ldp; xa.m = c.rows; xa.n = c.dim; xa.alpha = 1.f; xa.add = v0 != 0; xa.tma = 1; xa.padded = 1;
        AP_TRY((gradients_launch<SX, StoreEpi<float>, T>(c, cut, x, w, go, n, xa, wa)));
    }
    FinishArgs fa{part, factor, dx, p.ldp, lddx, c.rows, c.dim, p.splits};
    const uint64_t quads = (uint64_t)c.rows * ((c.dim + 3) / 4);
    return launch(grad_finish_kernel<T>, (uint32_t)std::min<uint64_t>((quads + 255) / 256, 8ull * c.sms), fa, c.st);
}

// ---- scores: the shapes ---------------------------------------------------------------------------------------------------
template <class T, int CG, int N>
static int scores_run(const ap_scaled_rows &a, const ap_scaled_rows &b, uint32_t dim, float alpha, T *out, uint64_t ldo, int sms, uint32_t *err,
                      cudaStream_t st) {
    using S = tile::Shape<tile::kE4m3, CG, N>;
    const Operand oa{a.q, a.rows, dim, a.ldq}, ob{b.q, b.rows, dim, b.ldq};
    typename StoreEpi<T>::Args ea{};
    ea.out = out; ea.ld = ldo; ea.m = a.rows; ea.n = b.rows; ea.alpha = alpha; ea.tma = aligned(out, ldo * sizeof(T), 16);
    const uint32_t blocks = ceil_div(dim, 128);
    const Scales sc{a.scale, b.scale, a.scale + (a.rows - 1) * a.ld_scale + blocks, b.scale + (b.rows - 1) * b.ld_scale + blocks, a.ld_scale, b.ld_scale, a.rows, b.rows,
                    aligned(a.scale, a.ld_scale, 4) && aligned(b.scale, b.ld_scale, 4)};
    return run_product<S, StoreEpi<T>>(oa, ob, a.rows, b.rows, dim, pick_n(N, 32, CG, a.rows, b.rows, ceil_div(dim, 128), sms, true), sc, ea, sms, err, st);
}
template <class T>
static int scores_pick(const ap_scaled_rows &a, const ap_scaled_rows &b, uint32_t dim, float alpha, void *out, uint64_t ldo, int sms, uint32_t *err,
                       cudaStream_t st) {
    T *o = static_cast<T *>(out);
    return a.rows > 128 ? scores_run<T, 2, 224>(a, b, dim, alpha, o, ldo, sms, err, st) : scores_run<T, 1, 224>(a, b, dim, alpha, o, ldo, sms, err, st);
}

static int check_loss(const char *what, uint32_t rows, uint32_t docs, uint32_t dim, uint32_t type, const void *x, uint64_t ldx, const void *w, uint64_t ldw,
                      const uint32_t *target, float scale) {
    if (!x || !w || !target) return fail(AP_ERR_ARG, "%s: null argument", what);
    if (type != AP_TYPE_F16 && type != AP_TYPE_BF16) return fail(AP_ERR_ARG, "%s: type %u: the vectors are f16 or bf16", what, type);
    if (rows == 0 || docs == 0 || dim == 0) return fail(AP_ERR_ARG, "%s: %u queries, %u documents, %u values: none may be 0", what, rows, docs, dim);
    if (rows > (1u << 20) || docs > (1u << 30) || dim > (1u << 16))
        return fail(AP_ERR_LIMIT, "%s: up to 2^20 queries, 2^30 documents, 2^16 values", what);
    if (ldx < dim || ldw < dim) return fail(AP_ERR_ARG, "%s: a row stride is shorter than a row", what);
    if (!aligned(x, ldx * 2, 16) || !aligned(w, ldw * 2, 16)) return fail(AP_ERR_ARG, "%s: rows start on 16-byte boundaries (base and stride)", what);
    if (!std::isfinite(scale)) return fail(AP_ERR_ARG, "%s: the scale is not finite", what);
    return AP_OK;
}

}  // namespace apoe

using namespace apoe;

namespace apoe {
// Takes the error word: read and cleared in one step, so an error that another stream raises at the same moment is either in
// what is taken or still there for the next check.
__global__ void dense_take_error_kernel(uint32_t *taken) { *taken = atomicExch(&dense_error_word, 0u); }
}  // namespace apoe

extern "C" int ap_dense_check_status(int device, void *stream) {
    DeviceScope scope;
    AP_TRY(scope.enter(device));
    cudaStream_t st = (cudaStream_t)stream;
    uint32_t *taken = nullptr, ew = 0;
    AP_CUDA(cudaMallocAsync(&taken, sizeof(uint32_t), st));      // of this check alone: several may run at once
    dense_take_error_kernel<<<1, 1, 0, st>>>(taken);
    cudaError_t asked = cudaGetLastError();
    if (asked == cudaSuccess) asked = cudaMemcpyAsync(&ew, taken, sizeof(uint32_t), cudaMemcpyDeviceToHost, st);
    const cudaError_t freed = cudaFreeAsync(taken, st);
    AP_CUDA(asked);
    AP_CUDA(freed);
    AP_CUDA(cudaStreamSynchronize(st));
    return ew ? fail(AP_ERR_DEVICE, "a dense operator raised error word %u (a bounded wait ran out)", ew) : AP_OK;
}

namespace apoe {
__global__ void dense_wait_probe_kernel(uint32_t polls, uint32_t *err) {
    __shared__ uint64_t bar;
    mbar_init(&bar, 1);
    mbar_fence_init();
    tile::wait(&bar, 0u, err, 39u, polls);        // nothing arrives: the wait runs out, the kernel ends
}
}  // namespace apoe

extern "C" int ap_debug_dense_wait_timeout(int device, uint32_t polls, void *stream) {
    if (polls > 4096) return fail(AP_ERR_ARG, "at most 4096 polls");
    DeviceScope scope;
    AP_TRY(scope.enter(device));
    int sms;
    uint32_t *err;
    AP_TRY(device_facts(device, &sms, &err));
    dense_wait_probe_kernel<<<1, 1, 0, (cudaStream_t)stream>>>(polls, err);
    AP_CUDA(cudaGetLastError());
    return AP_OK;
}

extern "C" int ap_quantize_rows_device(int device, uint32_t rows, uint32_t dim, uint32_t type, const void *src, uint64_t ld, uint8_t *q, uint64_t ldq,
                                       uint8_t *scale, uint64_t ld_scale, void *stream) {
    const int size = elem_size(type);
    if (!size) return fail(AP_ERR_ARG, "quantize: type %u", type);
    if (dim == 0) return fail(AP_ERR_ARG, "quantize: rows of 0 values");
    if (rows == 0) return AP_OK;
    if (!src || !q || !scale) return fail(AP_ERR_ARG, "quantize: null argument");
    const uint32_t blocks = ceil_div(dim, 128);
    if (ld < dim || ldq < dim || ld_scale < blocks) return fail(AP_ERR_ARG, "quantize: a row stride is shorter than a row");
    if ((uint64_t)rows * blocks >= (1ull << 31)) return fail(AP_ERR_LIMIT, "quantize: %u rows of %u blocks in one call", rows, blocks);
    if ((uintptr_t)src % (uint32_t)size) return fail(AP_ERR_ARG, "quantize: the source is not aligned to its type");
    DeviceScope scope;
    AP_TRY(scope.enter(device));
    int sms;
    uint32_t *err;
    AP_TRY(device_facts(device, &sms, &err));
    QuantArgs a{src, q, scale, ld, ldq, ld_scale, rows * blocks, dim, blocks, 0, 0};
    if (blocks > 1) {                  // with s = ceil(log2 blocks): magic = ceil(2^(31 + s) / blocks) < 2^32, exact for items below 2^31
        uint32_t s = 1;
        while ((1u << s) < blocks) ++s;
        a.magic = (uint32_t)(((1ull << (31 + s)) + blocks - 1) / blocks);
        a.shift = s - 1;
    }
    const bool units = aligned(src, ld * size, 16) && aligned(q, ldq, 16 / size) && dim % (16 / size) == 0;
    const bool flat = units && dim % 128 == 0 && ld == dim && ldq == dim && ld_scale == blocks;
    const uint32_t step = kQuantUnroll * 8 * (size == 4 ? 1 : 2), grid = (a.items - 1) / step + 1;
    cudaStream_t st = (cudaStream_t)stream;
    if (type == AP_TYPE_F32) return launch(flat ? quantize_kernel<float, kFlat> : units ? quantize_kernel<float, kUnits> : quantize_kernel<float, kAny>, grid, a, st);
    if (type == AP_TYPE_F16) return launch(flat ? quantize_kernel<__half, kFlat> : units ? quantize_kernel<__half, kUnits> : quantize_kernel<__half, kAny>, grid, a, st);
    return launch(flat ? quantize_kernel<__nv_bfloat16, kFlat> : units ? quantize_kernel<__nv_bfloat16, kUnits> : quantize_kernel<__nv_bfloat16, kAny>, grid, a, st);
}

extern "C" int ap_scaled_scores_device(int device, uint32_t dim, const ap_scaled_rows *a, const ap_scaled_rows *b, float alpha, uint32_t out_type, void *out,
                                       uint64_t ldo, void *stream) {
    if (!a || !b) return fail(AP_ERR_ARG, "scores: null argument");
    const int size = elem_size(out_type);
    if (!size) return fail(AP_ERR_ARG, "scores: output type %u", out_type);
    if (dim == 0) return fail(AP_ERR_ARG, "scores: rows of 0 values");
    if (a->rows == 0 || b->rows == 0) return AP_OK;
    if (!a->q || !a->scale || !b->q || !b->scale || !out) return fail(AP_ERR_ARG, "scores: null argument");
    if (a->rows > (1u << 30) || b->rows > (1u << 30) || dim > (1u << 20)) return fail(AP_ERR_LIMIT, "scores: up to 2^30 rows of 2^20 values");
    const uint32_t blocks = ceil_div(dim, 128);
    if (a->ldq < dim || b->ldq < dim || a->ld_scale < blocks || b->ld_scale < blocks || ldo < b->rows)
        return fail(AP_ERR_ARG, "scores: a row stride is shorter than a row");
    if (!aligned(a->q, a->ldq, 16) || !aligned(b->q, b->ldq, 16)) return fail(AP_ERR_ARG, "scores: 8-bit rows start on 16-byte boundaries (base and stride)");
    if ((uintptr_t)out % (uint32_t)size) return fail(AP_ERR_ARG, "scores: the output is not aligned to its type");
    if ((uint64_t)ceil_div(a->rows, 128) * ceil_div(b->rows, 32) >= (1ull << 31)) return fail(AP_ERR_LIMIT, "scores: %u x %u scores in one call", a->rows, b->rows);
    DeviceScope scope;
    AP_TRY(scope.enter(device));
    int sms;
    uint32_t *err;
    AP_TRY(device_facts(device, &sms, &err));
    cudaStream_t st = (cudaStream_t)stream;
    if (out_type == AP_TYPE_F32) return scores_pick<float>(*a, *b, dim, alpha, out, ldo, sms, err, st);
    if (out_type == AP_TYPE_F16) return scores_pick<__half>(*a, *b, dim, alpha, out, ldo, sms, err, st);
    return scores_pick<__nv_bfloat16>(*a, *b, dim, alpha, out, ldo, sms, err, st);
}

extern "C" int ap_softmax_loss_workspace(int device, uint32_t rows, uint32_t docs, uint32_t dim, int backward, size_t *bytes) {
    if (!bytes) return fail(AP_ERR_ARG, "softmax loss: null argument");
    if (rows == 0 || docs == 0 || dim == 0) return fail(AP_ERR_ARG, "softmax loss: %u queries, %u documents, %u values: none may be 0", rows, docs, dim);
    if (rows > (1u << 20) || docs > (1u << 30) || dim > (1u << 16))
        return fail(AP_ERR_LIMIT, "softmax loss: up to 2^20 queries, 2^30 documents, 2^16 values");
    if (!backward) { *bytes = forward_plan(rows, docs).bytes; return AP_OK; }
    int sms;
    AP_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    *bytes = backward_plan(rows, docs, dim, sms).bytes;
    return AP_OK;
}

extern "C" int ap_softmax_loss_forward_device(int device, uint32_t rows, uint32_t docs, uint32_t dim, uint32_t type, const void *queries, uint64_t ldq,
                                              const void *documents, uint64_t ldd, const uint32_t *target, float scale, float *loss, float *lse,
                                              void *workspace, size_t workspace_bytes, void *stream) {
    AP_TRY(check_loss("softmax loss", rows, docs, dim, type, queries, ldq, documents, ldd, target, scale));
    if (!loss || !lse || !workspace) return fail(AP_ERR_ARG, "softmax loss: null argument");
    if (!words(target, loss, lse)) return fail(AP_ERR_ARG, "softmax loss: target, loss and lse start on 4-byte boundaries");
    const ForwardPlan p = forward_plan(rows, docs);
    if (workspace_bytes < p.bytes) return fail(AP_ERR_ARG, "softmax loss: the workspace has %zu bytes, %zu are needed", workspace_bytes, p.bytes);
    if ((uintptr_t)workspace % 256) return fail(AP_ERR_ARG, "softmax loss: the workspace starts on a 256-byte boundary");
    DeviceScope scope;
    AP_TRY(scope.enter(device));
    LossCall c{rows, docs, dim, queries, documents, ldq, ldd, target, scale, 0, nullptr, (cudaStream_t)stream};
    AP_TRY(device_facts(device, &c.sms, &c.err));
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    if (type == AP_TYPE_F16) return rows <= 128 ? forward_run<__half, 1>(c, p, ws, loss, lse) : forward_run<__half, 2>(c, p, ws, loss, lse);
    return rows <= 128 ? forward_run<__nv_bfloat16, 1>(c, p, ws, loss, lse) : forward_run<__nv_bfloat16, 2>(c, p, ws, loss, lse);
}

extern "C" int ap_softmax_loss_backward_device(int device, uint32_t rows, uint32_t docs, uint32_t dim, uint32_t type, const void *queries, uint64_t ldq,
                                               const void *documents, uint64_t ldd, const uint32_t *target, float scale, const float *loss,
                                               const float *lse, const float *grad_loss, void *grad_queries, uint64_t ldgq, void *grad_documents,
                                               uint64_t ldgd, void *workspace, size_t workspace_bytes, void *stream) {
    AP_TRY(check_loss("softmax loss gradient", rows, docs, dim, type, queries, ldq, documents, ldd, target, scale));
    if (!loss || !lse || !grad_loss || !grad_queries || !grad_documents || !workspace) return fail(AP_ERR_ARG, "softmax loss gradient: null argument");
    if (!words(target, loss, lse, grad_loss)) return fail(AP_ERR_ARG, "softmax loss gradient: target, loss, lse and grad_loss start on 4-byte boundaries");
    if (ldgq < dim || ldgd < dim) return fail(AP_ERR_ARG, "softmax loss gradient: a row stride is shorter than a row");
    if (!aligned(grad_queries, ldgq * 2, 8) || (uintptr_t)grad_documents % 2) return fail(AP_ERR_ARG, "softmax loss gradient: rows of the queries' gradient start on 8-byte boundaries");
    DeviceScope scope;
    AP_TRY(scope.enter(device));
    LossCall c{rows, docs, dim, queries, documents, ldq, ldd, target, scale, 0, nullptr, (cudaStream_t)stream};
    AP_TRY(device_facts(device, &c.sms, &c.err));
    const BackwardPlan p = backward_plan(rows, docs, dim, c.sms);
    if (workspace_bytes < p.bytes) return fail(AP_ERR_ARG, "softmax loss gradient: the workspace has %zu bytes, %zu are needed", workspace_bytes, p.bytes);
    if ((uintptr_t)workspace % 256) return fail(AP_ERR_ARG, "softmax loss gradient: the workspace starts on a 256-byte boundary");
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    if (type == AP_TYPE_F16)
        return rows <= 128 ? backward_run<__half, 1>(c, p, ws, loss, lse, grad_loss, grad_queries, ldgq, grad_documents, ldgd)
                           : backward_run<__half, 2>(c, p, ws, loss, lse, grad_loss, grad_queries, ldgq, grad_documents, ldgd);
    return rows <= 128 ? backward_run<__nv_bfloat16, 1>(c, p, ws, loss, lse, grad_loss, grad_queries, ldgq, grad_documents, ldgd)
                       : backward_run<__nv_bfloat16, 2>(c, p, ws, loss, lse, grad_loss, grad_queries, ldgq, grad_documents, ldgd);
}
