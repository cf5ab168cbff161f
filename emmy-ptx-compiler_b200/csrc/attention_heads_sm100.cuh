// Device pieces shared by the tensor-core kernels of attention over heads: packed fp32 arithmetic, rounding pairs to 16
// bits, the relative position bias of a warp's block of scores, and the tensor maps of strided [batch, head, row, d]
// operands.
#pragma once
#include <limits.h>
#include <stddef.h>

#include "attention_heads.cuh"
#include "sm100_ptx.cuh"

namespace emmy {
namespace heads {

constexpr int kTile = 128;              // rows of a tile: tensor-memory lanes
constexpr int kHalf = 64;               // columns of a tile: rows of a stage
// bf16 operands of second products are cut from the fp32 pattern (one byte permute per pair): a conversion would run on the
// transcendental unit next to the exponentials. A cut loses half a step, 2^-8 of a value with mantissa 1, on average 2^-8 / ln 4 of
// values spread evenly in magnitude: they are scaled by 1 + 2^-8 / ln 4 first, which leaves no mean error and at most 1.28 times the
// 2^-8 of a rounding. f16 operands are converted: the same cut for f16 needs two more operations per value and was 5 % slower.
constexpr float kCutScale = 1.0028178f;
constexpr float kCutScaleLog2 = 0.0040594572f;      // its log2

__device__ __forceinline__ uint64_t as_u64(float2 v) { return *reinterpret_cast<uint64_t*>(&v); }
__device__ __forceinline__ float2 as_f2(uint64_t v) { return *reinterpret_cast<float2*>(&v); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(as_u64(a)), "l"(as_u64(b)), "l"(as_u64(c)));
    return as_f2(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(as_u64(a)), "l"(as_u64(b)));
    return as_f2(d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(as_u64(a)), "l"(as_u64(b)));
    return as_f2(d);
}
__device__ __forceinline__ float2 f2(uint32_t a, uint32_t b) { return make_float2(__uint_as_float(a), __uint_as_float(b)); }

// Nearest: outputs.
template <bool BF16>
__device__ __forceinline__ uint32_t round_pair(float lo, float hi) {
    if constexpr (BF16) {
        __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&v);
    } else {
        __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&v);
    }
}
// Operands of a second product: bf16 values already scaled by kCutScale are cut, f16 ones rounded.
template <bool BF16>
__device__ __forceinline__ uint32_t operand_pair(float2 v) {
    if constexpr (BF16) return __byte_perm(__float_as_uint(v.x), __float_as_uint(v.y), 0x7632);
    else return round_pair<false>(v.x, v.y);
}

// The same rounded (half a step away from zero on a tie): two additions more per pair.
template <bool BF16>
__device__ __forceinline__ uint32_t rounded_pair(float2 v) {
    if constexpr (BF16) return __byte_perm(__float_as_uint(v.x) + 0x8000u, __float_as_uint(v.y) + 0x8000u, 0x7632);
    else return round_pair<false>(v.x, v.y);
}

// ---- waits of a whole warp ---------------------------------------------------------------------------------------------------
// One poll by all lanes and a vote is the common case and costs some 50 cycles less than a loop per lane around it (the
// issuing warp makes three or four waits per tile: with the per-lane form they took longer than the products). The limit and the
// abort flag are those of bounded_wait / bounded_spin; the answer is the warp's. All of it is inlined: across a call the compiler keeps
// nothing in uniform registers, and every operand of every product was moved there again (64 cycles per product instruction against 43).
template <bool PARK>
__device__ __forceinline__ bool warp_poll(const WaitCtx& ctx, uint32_t bar, uint32_t parity, uint32_t code) {
    if (__all_sync(0xffffffffu, ptx::mbar_test_wait(bar, parity))) return true;
    uint64_t t0 = 0;
    for (uint32_t n = 1;; ++n) {
        if (__all_sync(0xffffffffu, PARK ? ptx::mbar_try_wait(bar, parity) : ptx::mbar_test_wait(bar, parity))) return true;
        if ((n & (PARK ? 15u : 63u)) == 0) {
            const uint64_t now = ptx::global_timer_ns();
            if (t0 == 0) t0 = now;
            const bool late = now - t0 > ctx.limit_ns;
            if (late) {
                atomicCAS(ctx.status_word, 0u, code);
                *ctx.abort_flag = 1;
            }
            if (__any_sync(0xffffffffu, late || *ctx.abort_flag != 0)) return false;
        }
    }
}
// Parks the warp while it waits.
__device__ __forceinline__ bool warp_wait(const WaitCtx& ctx, uint32_t bar, uint32_t parity, uint32_t code) { return warp_poll<true>(ctx, bar, parity, code); }
// Polls without parking (the issuing warp).
__device__ __forceinline__ bool warp_spin(const WaitCtx& ctx, uint32_t bar, uint32_t parity, uint32_t code) { return warp_poll<false>(ctx, bar, parity, code); }

// ---- the bias --------------------------------------------------------------------------------------------------------
// A warp works on 32 x 64 blocks of scores, which span 95 distances. Where they all fall into one run (far from the
// diagonal: every distance beyond max_distance) the bias is one number; else the warp copies the 95 values into its own
// stretch of shared memory. The run of a distance comes from a table over the distances between the first run's last and the last
// run's first, filled once per CTA, run by run (a binary search for every block took 1900 cycles of the 4000 a block cost);
// schemes that spread over more than kNear distances are searched. The range of the last single run is kept, so that neighbouring blocks of a
// far stretch cost two comparisons.
constexpr int kNear = 4096;
struct BiasShared {
    int first[kHeadsMaxRuns];
    float value[kHeadsMaxRuns];         // of the head, log2 units
    float by_dist[8][96];               // one row per warp
    uint8_t near_run[kNear];            // run of distance near_first + i
};
static_assert(offsetof(BiasShared, by_dist) % 16 == 0, "read as float4");
// The distances near_run covers: from the last one of run 0 to the first one of the last run.
struct NearRuns {
    int first, count;                   // count 0: not used
    __device__ __forceinline__ NearRuns(const HeadsParams& p) {
        first = p.n_runs > 1 ? p.run_first[1] - 1 : 0;
        const long long span = p.n_runs > 1 ? (long long)p.run_first[p.n_runs - 1] - first + 1 : 1;
        count = span <= kNear ? (int)span : 0;
    }
};
// The part of the shared tables that does not depend on the head: a warp per run, a lane per distance (a thread per run took 2000
// cycles of a CTA's set-up for 32 runs within 128).
__device__ __forceinline__ void load_runs(BiasShared& s, const HeadsParams& p, int warp, int warps, int lane) {
    const NearRuns near(p);
    for (int r = warp; r < p.n_runs; r += warps) {
        const int mine = p.run_first[r];
        if (lane == 0) s.first[r] = mine;
        if (near.count) {
            const int to = r + 1 == p.n_runs ? near.count : p.run_first[r + 1] - near.first;
            for (int i = (r == 0 ? 0 : mine - near.first) + lane; i < to; i += 32) s.near_run[i] = (uint8_t)r;
        }
    }
}
struct WarpBias {
    int lo, hi;                         // distances [lo, hi) have the bias `same`
    int run;                            // its run
    float same;
    NearRuns near;
    __device__ __forceinline__ WarpBias(const HeadsParams& p) : near(p) { reset(); }
    __device__ __forceinline__ void reset() { lo = 0; hi = 0; run = 0; same = 0.0f; }
    __device__ __forceinline__ int run_of(const BiasShared& s, int n_runs, int dist) const {
        if (near.count) return s.near_run[min(max(dist - near.first, 0), near.count - 1)];
        return heads_run_of(s.first, n_runs, dist);
    }
    // Distances d0 .. d0 + 94. True: all in one run. False: s.by_dist[warp][0 .. 94] holds their biases. `value`: by run.
    __device__ __forceinline__ bool block(BiasShared& s, const float* value, int warp, int lane, int n_runs, int d0) {
        if (d0 >= lo && d0 + 94 < hi) return true;
        int r[3];
#pragma unroll
        for (int k = 0; k < 3; ++k) r[k] = run_of(s, n_runs, d0 + 32 * k + lane);
        const int ra = __shfl_sync(0xffffffffu, r[0], 0), rb = __shfl_sync(0xffffffffu, r[2], 30);
        if (ra == rb) {
            lo = ra == 0 ? INT_MIN : s.first[ra];
            hi = ra + 1 == n_runs ? INT_MAX : s.first[ra + 1];
            run = ra;
            same = value[ra];
            return true;
        }
        __syncwarp();                   // the previous block's readers
#pragma unroll
        for (int k = 0; k < 3; ++k) s.by_dist[warp][32 * k + lane] = value[r[k]];
        __syncwarp();
        return false;
    }
};

// The products of a 64-column tile, issued by a whole warp for its elected lane. B operands are stages of 64 rows: D / 64 pieces of 64 x 128 bytes.
template <int D, bool BF16>
struct Products {
    static constexpr uint32_t kHi = ptx::smem_desc_sw128_hi(1024);
    static constexpr uint32_t kPiece = kHalf * 128;
    static constexpr uint32_t kScores = ptx::mma_idesc_f16(BF16, false, false, kTile, kHalf);
    static constexpr uint32_t kGrads = ptx::mma_idesc_f16(BF16, false, true, kTile, D);
    // scores: rows of A (tensor memory) times the stage's rows, contraction over the head dim
    static __device__ __forceinline__ void scores_ts(uint32_t lead, uint32_t d, uint32_t a, uint32_t stage) {
        const uint32_t lo = ptx::smem_desc_sw128_lo(stage, 16);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) ptx::mma_ts_lead(lead, d, a + kk * 8, lo + (((kk / 4) * kPiece + (kk % 4) * 32) >> 4), kHi, kScores, kk != 0);
    }
    // the same with A as 128 rows in shared memory
    static __device__ __forceinline__ void scores_ss(uint32_t lead, uint32_t d, uint32_t a, uint32_t stage) {
        const uint32_t lo_a = ptx::smem_desc_sw128_lo(a, 16), lo_b = ptx::smem_desc_sw128_lo(stage, 16);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
            ptx::mma_ss_lead(lead, d, lo_a + (((kk / 4) * (kTile * 128) + (kk % 4) * 32) >> 4), lo_b + (((kk / 4) * kPiece + (kk % 4) * 32) >> 4), kHi, kScores, kk != 0);
    }
    // gradients: A (tensor memory, 64 columns of values) times the stage, contraction over its rows
    static __device__ __forceinline__ void grads(uint32_t lead, uint32_t d, uint32_t a, uint32_t stage, bool first) {
        const uint32_t lo = ptx::smem_desc_sw128_lo(stage, kPiece);
#pragma unroll
        for (int kk = 0; kk < kHalf / 16; ++kk) ptx::mma_ts_lead(lead, d, a + kk * 8, lo + ((kk * 16 * 128) >> 4), kHi, kGrads, !first || kk != 0);
    }
};
// Part of a row of a 128-row tile in shared memory (pieces of 128 rows x 64 elements, 128-byte swizzle) into tensor memory, as the A
// operand of a product: columns of element pairs. Elements 32 first .. 32 (first + N) - 1; `taddr`: of the row's first element. (Threads
// reading their rows from global memory instead took 7000 cycles of a CTA's set-up.)
template <int N>
__device__ __forceinline__ void row_to_tmem(uint32_t taddr, uint32_t tile, int row, int first = 0) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int i = first + n;
        uint32_t r[16];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int piece = (i % 2) * 4 + k;
            ptx::ld_shared_16B(tile + (i / 2) * (kTile * 128) + row * 128 + ((piece ^ (row & 7)) << 4), r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]);
        }
        ptx::tmem_st_32x32b_x16(taddr + 16 * i, r);
    }
}

// ---- the order of the work items -----------------------------------------------------------------------------------------------
// Causal tiles differ in length. Dealt longest first over many units the SMs finish together; dealt unit by unit the last units'
// longest tiles run alone (16 units of 2048 keys on 148 SMs, dK and dV: 184 us against 149). But CTAs that run at the same time should share
// what they stream, so the units are taken in chunks whose streamed operands fit in a third of L2, each chunk longest first. chunk = 1: unit by
// unit (tiles of equal length).
// Division of 0 <= n < 2^31 by a number known at launch: a division instruction sequence takes some 150 cycles, a CTA's place in the work seven.
struct FastDiv {
    uint32_t mul, shift;
    __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift); }
};
inline FastDiv fast_div(int64_t d) {
    uint32_t shift = 0;
    while ((1ll << shift) < d) ++shift;
    return {(uint32_t)((((1ull << shift) - (uint64_t)d) << 32) / (uint64_t)d + 1), shift};
}
struct WorkItem {
    int unit, tile;                     // tile: 0 is the longest
};
struct WorkOrder {
    int units, tiles, chunk;
    FastDiv per_chunk, width, last_width;       // chunk * tiles; units of a chunk; of the last one
    __device__ __forceinline__ WorkItem operator()(int item) const {
        const int c = per_chunk(item), in_chunk = item - c * chunk * tiles;
        const bool last = (c + 1) * chunk > units;
        const int w = last ? units - c * chunk : chunk, tile = last ? last_width(in_chunk) : width(in_chunk);
        return {c * chunk + in_chunk - tile * w, tile};
    }
};
// `bytes`: streamed by one unit's tiles.
inline WorkOrder work_order(bool causal, int64_t units, int64_t tiles, int64_t bytes) {
    const int64_t fit = (42ll << 20) / (bytes > 0 ? bytes : 1);
    int64_t chunk = !causal || fit < 1 ? 1 : fit > units ? units : fit;
    if (chunk * tiles >= (1ll << 31)) chunk = 1;
    const int64_t rest = units % chunk;
    return {(int)units, (int)tiles, (int)chunk, fast_div(chunk * tiles), fast_div(chunk), fast_div(rest ? rest : chunk)};
}

// ---- strided operands ---------------------------------------------------------------------------------------------------
// A [batch, heads, rows, d] operand as a 4-D tensor map; dimensions with stride 0 (a broadcast) or extent 1 are given
// extent 1 and coordinate 0.
struct MapAt {
    int head, batch;                    // 1, or 0 where the coordinate is always 0
};

inline bool stride_fits(int64_t extent, int64_t s) { return extent <= 1 || s == 0 || (s % 8 == 0 && s < (1ll << 38)); }
// Whether TMA can address the operand (16-byte aligned base, strides in whole 16-byte units).
inline bool map_fits(const void* base, int64_t batch, int64_t heads, int64_t rows, const int64_t* s) {
    return aligned(base, 16) && stride_fits(batch, s[0]) && stride_fits(heads, s[1]) && stride_fits(rows, s[2]) && !(rows > 1 && s[2] == 0);
}
inline int make_map(CUtensorMap* map, MapAt* at, const void* base, int64_t batch, int64_t heads, int64_t rows, int d, const int64_t* s, int box_rows,
                    int box_heads) {
    at->batch = batch > 1 && s[0] != 0;
    at->head = heads > 1 && s[1] != 0;
    const uint64_t row_s = rows > 1 ? (uint64_t)s[2] : (uint64_t)d;
    const uint64_t extent[4] = {(uint64_t)d, (uint64_t)rows, at->head ? (uint64_t)heads : 1, at->batch ? (uint64_t)batch : 1};
    const uint64_t stride[3] = {row_s, at->head ? (uint64_t)s[1] : row_s, at->batch ? (uint64_t)s[0] : row_s};
    const uint32_t box[4] = {64, (uint32_t)box_rows, (uint32_t)box_heads, 1};
    return make_tensor_map_4d(map, base, extent, stride, box);
}

// 32 columns of an output row (from `col` on, a multiple of 32) into a tile of 128 rows staged for a TMA store: pieces of 128 rows x
// 64 columns, 128-byte swizzle. `w`: the 16-bit pairs.
__device__ __forceinline__ void stage_row(uint32_t tile, int row, int col, const uint32_t (&w)[16]) {
    const uint32_t at = tile + (col / 64) * (kTile * 128) + row * 128;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const uint32_t piece = (uint32_t)((col % 64) / 8 + q) ^ (uint32_t)(row & 7);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + piece * 16), "r"(w[4 * q]), "r"(w[4 * q + 1]), "r"(w[4 * q + 2]), "r"(w[4 * q + 3])
                     : "memory");
    }
}

}  // namespace heads
}  // namespace emmy
