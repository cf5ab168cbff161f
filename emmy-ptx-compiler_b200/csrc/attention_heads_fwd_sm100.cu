// Attention over heads, forward, on the tensor cores: f16 / bf16, d = 64 or 128.
//
// One CTA per (query tile, head, batch entry), two CTAs resident per SM (256 tensor-memory columns each), so that one's
// softmax overlaps the other's products:
//   warp 0    TMA: the Q tile once, 128-key K and V tiles, each re-armed as soon as the product that read it is done
//   warp 1    tcgen05.mma: S = Q K^T into tensor memory, O += P V with P read from tensor memory
//   warps 2-9 softmax, two threads per query row (64 keys of each tile apiece), one pass with a running maximum and sum;
//             the maximum is raised only when it grows by more than 2^8, so O is rescaled rarely
// Added to what plain attention does: the log-sum-exp of every row; grouped heads and strides through 4-D tensor maps; a
// key count per batch entry (V rows behind it are cleared in shared memory before the product reads them, scores are masked
// by selection, so nothing there is ever used); causal masks from either end; the relative position bias, one number for
// blocks far from the diagonal, else 95 looked-up values per warp.
//
// When there are few rows (single tokens against a cache) two things change. The query heads of a key head share one tile:
// rows are (head of the group, query), loaded by one TMA box over both dimensions, so the keys are read once per key
// head. And the keys are split over several CTAs, whose unnormalised outputs, maxima and sums a small kernel joins.
#include <math_constants.h>

#include <algorithm>

#include "attention_heads_sm100.cuh"

namespace emmy {
namespace heads {

constexpr int kFwdThreads = 320;

struct FwdParams {
    HeadsParams h;
    MapAt q_at, k_at, v_at, o_at;
    int packed;                         // rows of a tile: group x seq_q (1) or 128 queries of one head (0)
    int tiles;                          // query tiles per unit (batch entry and head, or key head when packed)
    int splits;                         // CTAs that share a tile's keys
    WorkOrder order;
    FastDiv by_splits, by_unit_heads, by_group;
    float* lse;
    float* part_o;                      // splits > 1: [split][row][D], rows as lse
    float2* part_ml;                    // [split][row]: maximum (log2 units), sum
    unsigned long long wait_limit_ns;
    uint32_t* status;
};

__device__ uint32_t g_fwd_status;

template <int D>
struct FwdSmem {
    static constexpr int kOperand = kTile * D * 2;
    static constexpr int kBarOffset = 3 * kOperand;
    static constexpr int kXchgOffset = kBarOffset + 256;
    static constexpr int kBiasOffset = kXchgOffset + 2048;
    static constexpr int kNeeded = kBiasOffset + (int)sizeof(BiasShared) + 1024;
    static constexpr int kTotal = kNeeded > 81920 ? kNeeded : 81920;        // never three CTAs (of 256 tensor-memory columns) on an SM
};

// The two warps that share rows publish values in shared memory and trade a flag, with the time limit and abort handling of
// every other wait. Returns false, warp-uniformly, when the wait was given up.
__device__ __forceinline__ bool trade(const WaitCtx& ctx, volatile uint32_t* flags, int half, int quarter, int lane, uint32_t token, uint32_t code) {
    __threadfence_block();
    __syncwarp();
    bool ok = true;
    if (lane == 0) {
        flags[half * 4 + quarter] = token;
        volatile uint32_t* other = flags + (half ^ 1) * 4 + quarter;
        uint64_t t0 = 0;
        for (uint32_t spin = 1; *other != token; ++spin) {
            if ((spin & 255u) == 0) {
                if (*ctx.abort_flag) { ok = false; break; }
                const uint64_t now = ptx::global_timer_ns();
                if (t0 == 0) t0 = now;
                else if (now - t0 > ctx.limit_ns) {
                    atomicCAS(ctx.status_word, 0u, code);
                    *ctx.abort_flag = 1;
                    ok = false;
                    break;
                }
            }
        }
    }
    ok = __all_sync(0xffffffffu, ok);
    __threadfence_block();
    return ok;
}

template <int D, bool BF16, bool BIAS>
__global__ void __launch_bounds__(kFwdThreads, 2)
heads_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                 const __grid_constant__ CUtensorMap map_o, const __grid_constant__ FwdParams p) {
    using S = FwdSmem<D>;
    constexpr int kChunks = D / 64;
    constexpr uint32_t kTmemCols = 256, kColO = 128;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));
    const uint32_t q_smem = smem_base, k_smem = smem_base + S::kOperand, v_smem = k_smem + S::kOperand;
    const uint32_t bar_base = smem_base + S::kBarOffset;
    const uint32_t q_full = bar_base, k_full = bar_base + 8, v_full = bar_base + 16, k_empty = bar_base + 24, v_empty = bar_base + 32,
                   s_full = bar_base + 40, p_full = bar_base + 48, o_full = bar_base + 56, o_staged = bar_base + 64;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_gen + S::kBarOffset + 80);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    volatile uint32_t* pair_flags = tmem_slot + 4;                                  // [2 buffers][2 halves][4 quarters]
    float* xchg = reinterpret_cast<float*>(smem_gen + S::kXchgOffset);              // [2][2][128]
    BiasShared& bias = *reinterpret_cast<BiasShared*>(smem_gen + S::kBiasOffset);

    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int item = p.by_splits(blockIdx.x), split = blockIdx.x - item * p.splits;
    const int unit_heads = p.packed ? p.h.kv_heads : p.h.heads;
    const WorkItem work = p.order(item);
    const int unit = work.unit, qt = p.h.causal ? p.tiles - 1 - work.tile : work.tile;
    const int b = p.by_unit_heads(unit), hu = unit - b * unit_heads;
    const int head0 = p.packed ? hu * p.h.group : hu, hk = p.packed ? hu : p.by_group(hu);
    const int row0 = qt * kTile;
    const int box_rows = p.packed ? p.h.group * p.h.seq_q : kTile;
    const int n_keys = heads_key_count(p.h, b), offset = heads_offset(p.h, n_keys);
    const int last_query = p.packed ? p.h.seq_q - 1 : min(row0 + kTile, p.h.seq_q) - 1;
    const int key_end = p.h.causal ? max(0, min(n_keys, last_query + offset + 1)) : n_keys;
    const int all_tiles = (key_end + kTile - 1) / kTile;
    const int tile_first = (int)((long long)all_tiles * split / p.splits);
    const int kv_tiles = (int)((long long)all_tiles * (split + 1) / p.splits) - tile_first;
    const WaitCtx wctx{abort_flag, p.status, p.wait_limit_ns};

    auto load_k = [&](int j) {
        ptx::mbar_arrive_expect_tx(k_full, S::kOperand);
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
            ptx::tma_load_4d(k_smem + c * (kTile * 128), &map_k, k_full, c * 64, (tile_first + j) * kTile, hk * p.k_at.head, b * p.k_at.batch);
    };
    auto load_v = [&](int j) {
        ptx::mbar_arrive_expect_tx(v_full, S::kOperand);
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
            ptx::tma_load_4d(v_smem + c * (kTile * 128), &map_v, v_full, c * 64, (tile_first + j) * kTile, hk * p.v_at.head, b * p.v_at.batch);
    };
    if (threadIdx.x == 0) {
        ptx::mbar_init(q_full, 1); ptx::mbar_init(k_full, 1); ptx::mbar_init(v_full, 1);
        ptx::mbar_init(k_empty, 1); ptx::mbar_init(v_empty, 1);
        ptx::mbar_init(s_full, 1); ptx::mbar_init(p_full, 8); ptx::mbar_init(o_full, 1); ptx::mbar_init(o_staged, 8);
        for (int q = 0; q < 16; ++q) pair_flags[q] = 0;
        *abort_flag = 0;
        ptx::mbar_fence_init();
        if (kv_tiles > 0) {                                     // the first loads fly while the CTA sets itself up
            ptx::mbar_arrive_expect_tx(q_full, box_rows * D * 2);
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
                ptx::tma_load_4d(q_smem + c * (kTile * 128), &map_q, q_full, c * 64, row0, head0 * p.q_at.head, b * p.q_at.batch);
            load_k(0);
            load_v(0);
        }
    }
    if constexpr (BIAS) {
        float run_bias = 0.0f;
        if ((int)threadIdx.x < p.h.n_runs) run_bias = heads_run_bias(p.h, threadIdx.x, head0);
        load_runs(bias, p.h, warp, kFwdThreads / 32, lane);
        if ((int)threadIdx.x < p.h.n_runs) bias.value[threadIdx.x] = run_bias;
    }
    if (warp == 1) {
        ptx::tmem_alloc(ptx::smem_u32(tmem_slot), kTmemCols);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        // ---- TMA producer ------------------------------------------------------------------------------
        if (lane == 0) {
            for (int j = 1; j < kv_tiles; ++j) {
                if (!bounded_wait(wctx, k_empty, (j & 1) ^ 1, 0x04010000u | (j & 0xffff))) break;
                load_k(j);
                if (!bounded_wait(wctx, v_empty, (j & 1) ^ 1, 0x04020000u | (j & 0xffff))) break;
                load_v(j);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---- MMA issuer: the whole warp, for its elected lane -----------------------------------------------
        {
            constexpr uint32_t idesc_s = ptx::mma_idesc_f16(BF16, false, false, kTile, kTile);
            constexpr uint32_t idesc_o = ptx::mma_idesc_f16(BF16, false, true, kTile, D);
            constexpr uint32_t hi = ptx::smem_desc_sw128_hi(1024);
            const uint32_t lead = ptx::elect_lead();
            const uint32_t q_lo = ptx::smem_desc_sw128_lo(q_smem, 16), k_lo = ptx::smem_desc_sw128_lo(k_smem, 16), v_lo = ptx::smem_desc_sw128_lo(v_smem, kTile * 128);
            const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
            const int tiles = __shfl_sync(0xffffffffu, kv_tiles, 0);
            auto wait = [&](uint32_t bar, uint32_t parity, uint32_t code) { return warp_spin(wctx, bar, parity, code); };
            const uint32_t s_tmem = tmem, o_tmem = tmem + kColO;
            bool ok = tiles == 0 || wait(q_full, 0, 0x04030000u);
            for (int j = 0; j < tiles && ok; ++j) {
                const uint32_t ph = j & 1;
                if (!(ok = wait(k_full, ph, 0x04040000u | (j & 0xffff)))) break;
                ptx::tc_fence_after_sync();
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {           // S = Q K^T, contraction over the head dim
                    const uint32_t off = ((kk / 4) * (kTile * 128) + (kk % 4) * 32) >> 4;
                    ptx::mma_ss_lead(lead, s_tmem, q_lo + off, k_lo + off, hi, idesc_s, kk != 0);
                }
                ptx::mma_commit_lead(lead, s_full);
                ptx::mma_commit_lead(lead, k_empty);
                if (!(ok = wait(p_full, ph, 0x04050000u | (j & 0xffff)))) break;
                if (!(ok = wait(v_full, ph, 0x04060000u | (j & 0xffff)))) break;
                ptx::tc_fence_after_sync();
#pragma unroll
                for (int kk = 0; kk < kTile / 16; ++kk)         // O += P V, contraction over the keys
                    ptx::mma_ts_lead(lead, o_tmem, s_tmem + kk * 8, v_lo + ((kk * 16 * 128) >> 4), hi, idesc_o, (j | kk) != 0);
                ptx::mma_commit_lead(lead, v_empty);
            }
            if (ok) ptx::mma_commit_lead(lead, o_full);
        }
        __syncwarp();
    } else {
        // ---- softmax: two threads per query row, 64 keys of each tile apiece ----------------------------------
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const int row_in_tile = quarter * 32 + lane;
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        const uint32_t s_row = tmem_base + lane_base + half * (kTile / 2);
        const uint32_t p_row = tmem_base + lane_base + half * (kTile / 4);
        const uint32_t o_row = tmem_base + lane_base + kColO + half * (D / 2);
        const int query = p.packed ? row_in_tile % p.h.seq_q : row0 + row_in_tile;
        // keys 0 .. sees - 1 are seen by this row
        const int sees = p.h.causal ? min(n_keys, query + offset + 1) : n_keys;
        float m_run = -CUDART_INF_F;      // the max the exponentials are taken against (log2 units)
        float l_run = 0.0f;               // running sum over this thread's columns
        bool ok = true;
        WarpBias wb(p.h);
        for (int j = 0; j < kv_tiles && ok; ++j) {
            const int key0 = (tile_first + j) * kTile + half * (kTile / 2);
            float c = p.h.scale_log2, add = 0.0f;               // a score in log2 units is c * s + add
            bool looked_up = false;
            if constexpr (BIAS) looked_up = !wb.block(bias, bias.value, warp - 2, lane, p.h.n_runs, key0 - (row0 + quarter * 32 + 31 + offset));
            ok = __all_sync(0xffffffffu, bounded_wait(wctx, s_full, j & 1, 0x04070000u | (j & 0xffff)));
            if (!ok) break;
            ptx::tc_fence_after_sync();
            uint32_t r[kTile / 2];
#pragma unroll
            for (int ch = 0; ch < kTile / 64; ++ch) ptx::tmem_ld_32x32b_x32(s_row + ch * 32, *reinterpret_cast<uint32_t(*)[32]>(&r[ch * 32]));
            ptx::tmem_ld_wait();
            if constexpr (BIAS) {
                if (looked_up) {
                    const float* at = bias.by_dist[warp - 2] + 31 - lane;
#pragma unroll
                    for (int i = 0; i < kTile / 2; ++i) r[i] = __float_as_uint(fmaf(__uint_as_float(r[i]), c, at[i]));
                    c = 1.0f;
                } else {
                    add = wb.same;
                }
            }
            const int valid = sees - key0;                      // of this thread's columns
            if (valid < kTile / 2) {
#pragma unroll
                for (int i = 0; i < kTile / 2; ++i)
                    if (i >= valid) r[i] = __float_as_uint(-CUDART_INF_F);
            }
            float ext[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) ext[i] = __uint_as_float(r[i]);
#pragma unroll
            for (int i = 8; i < kTile / 2; ++i) ext[i & 7] = fmaxf(ext[i & 7], __uint_as_float(r[i]));
            ext[0] = fmaxf(fmaxf(fmaxf(ext[0], ext[1]), fmaxf(ext[2], ext[3])), fmaxf(fmaxf(ext[4], ext[5]), fmaxf(ext[6], ext[7])));
            const float mine = fmaf(ext[0], c, add);
            // exchange with the thread that owns the other half of the row (after it both halves of S are in registers, so P may
            // overwrite S)
            volatile float* slot = xchg + (j & 1) * 256;
            slot[half * 128 + row_in_tile] = mine;
            ok = trade(wctx, pair_flags + (j & 1) * 8, half, quarter, lane, (uint32_t)j + 1, 0x04090000u | (j & 0xffff));
            if (!ok) break;
            const float m_tile = fmaxf(mine, slot[(half ^ 1) * 128 + row_in_tile]);
            const bool raise = m_tile > m_run + 8.0f;           // from -inf: with the first key the row sees
            const float m_new = raise ? m_tile : m_run;
            if (__any_sync(0xffffffffu, raise) && j > 0) {
                const float f = raise ? ptx::ex2_approx(m_run - m_new) : 1.0f;
#pragma unroll 1
                for (int col = 0; col < D / 2; col += 8) {      // few registers: the S row is still live
                    uint32_t o[8];
                    ptx::tmem_ld_32x32b_x8(o_row + col, o);
                    ptx::tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                    ptx::tmem_st_32x32b_x8(o_row + col, o);
                }
                l_run *= f;
            }
            m_run = m_new;
            const float ref = m_run == -CUDART_INF_F ? 0.0f : m_run;            // nothing seen so far: every exponential is 2^-inf
            const float shift = add - ref + (BF16 ? kCutScaleLog2 : 0.0f);
            const float2 c2 = make_float2(c, c), s2 = make_float2(shift, shift);
            float2 sum2[4] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
            for (int ch = 0; ch < kTile / 64; ++ch) {
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 y = fma2(f2(r[ch * 32 + 2 * i], r[ch * 32 + 2 * i + 1]), c2, s2);
                    const float2 e = make_float2(ptx::ex2_approx(y.x), ptx::ex2_approx(y.y));
                    sum2[i & 3] = add2(sum2[i & 3], e);
                    w[i] = operand_pair<BF16>(e);
                }
                ptx::tmem_st_32x32b_x16(p_row + ch * 16, w);
            }
            const float2 tot = add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3]));
            l_run += tot.x + tot.y;
            // V rows behind the key count hold whatever the caller left there: cleared before the product multiplies them by P's zeros
            const int live = n_keys - (tile_first + j) * kTile;
            if (live < kTile && n_keys < p.h.seq_k) {
                ok = __all_sync(0xffffffffu, bounded_wait(wctx, v_full, j & 1, 0x040b0000u | (j & 0xffff)));
                if (!ok) break;
                for (int e = live * 8 + (int)threadIdx.x - 64; e < kTile * 8; e += 256)         // 16-byte pieces of the rows
#pragma unroll
                    for (int ch = 0; ch < kChunks; ++ch)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(v_smem + ch * (kTile * 128) + e * 16), "r"(0) : "memory");
                ptx::fence_proxy_async_smem();
            }
            ptx::tmem_st_wait();
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(p_full);
        }
        // merge the two partial row sums, then write this thread's half of the output row
        if (ok) {
            volatile float* slot = xchg + (kv_tiles & 1) * 256;
            slot[half * 128 + row_in_tile] = l_run;
            ok = trade(wctx, pair_flags + (kv_tiles & 1) * 8, half, quarter, lane, (uint32_t)kv_tiles + 1, 0x040a0000u);
            if (ok) l_run += slot[(half ^ 1) * 128 + row_in_tile];
        }
        if (ok && __all_sync(0xffffffffu, bounded_wait(wctx, o_full, 0, 0x04080000u))) {
            ptx::tc_fence_after_sync();
            const bool live_row = p.packed ? row_in_tile < box_rows : query < p.h.seq_q;
            const int head = p.packed ? head0 + row_in_tile / p.h.seq_q : head0;
            const int64_t out_row = ((int64_t)b * p.h.heads + head) * p.h.seq_q + query;
            const bool empty = l_run == 0.0f;                   // the row saw no key
            if (p.splits > 1) {
                const int64_t at = (int64_t)split * p.h.batch * p.h.heads * p.h.seq_q + out_row;
#pragma unroll 1
                for (int ch = 0; ch < D / 16; ++ch) {           // this thread's D / 2 columns, eight at a time
                    uint32_t o[8];
                    ptx::tmem_ld_32x32b_x8(o_row + ch * 8, o);
                    ptx::tmem_ld_wait();
                    if (live_row && !empty) {
                        float4* dst = reinterpret_cast<float4*>(p.part_o + at * D + half * (D / 2) + ch * 8);
                        dst[0] = make_float4(__uint_as_float(o[0]), __uint_as_float(o[1]), __uint_as_float(o[2]), __uint_as_float(o[3]));
                        dst[1] = make_float4(__uint_as_float(o[4]), __uint_as_float(o[5]), __uint_as_float(o[6]), __uint_as_float(o[7]));
                    }
                }
                if (live_row && half == 0) p.part_ml[at] = make_float2(m_run, l_run);
            } else {
                if (live_row && half == 0)
                    p.lse[out_row] = empty ? -CUDART_INF_F : (m_run + log2f(l_run) - (BF16 ? kCutScaleLog2 : 0.0f)) * kLn2;
                // every product has completed, so the Q tile's shared memory is free: the output is staged there and leaves through TMA
                const float inv = empty ? 0.0f : (BF16 ? kCutScale : 1.0f) / l_run;
#pragma unroll 1
                for (int ch = 0; ch < D / 64; ++ch) {
                    uint32_t o[32];
                    ptx::tmem_ld_32x32b_x32(o_row + ch * 32, o);
                    ptx::tmem_ld_wait();
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        w[i] = empty ? 0u : round_pair<BF16>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
                    stage_row(q_smem, row_in_tile, half * (D / 2) + ch * 32, w);
                }
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(o_staged);
                if (threadIdx.x == 64 && bounded_wait(wctx, o_staged, 0, 0x040c0000u)) {
#pragma unroll
                    for (int c = 0; c < kChunks; ++c)
                        ptx::tma_store_4d(&map_o, q_smem + c * (kTile * 128), c * 64, row0, head0 * p.o_at.head, b * p.o_at.batch);
                    ptx::tma_store_commit();
                    ptx::tma_store_wait_read<0>();     // shared memory has been read; the grid's end covers the writes
                }
            }
        }
    }

    if (*abort_flag) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);         // copies in flight land before the shared memory is given up
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem_base, kTmemCols);
    }
}

// Joins the splits of every row: o = sum 2^(m_s - m) o_s / sum 2^(m_s - m) l_s. One warp per row.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) heads_join_kernel(const __grid_constant__ FwdParams p, uint16_t* __restrict__ O) {
    const int lane = threadIdx.x & 31;
    const int64_t rows = (int64_t)p.h.batch * p.h.heads * p.h.seq_q;
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= rows) return;
    float m = -CUDART_INF_F;
    for (int s = lane; s < p.splits; s += 32) {
        const float2 ml = p.part_ml[s * rows + row];
        if (ml.y != 0.0f) m = fmaxf(m, ml.x);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    const float ref = m == -CUDART_INF_F ? 0.0f : m;
    float acc[D / 32] = {}, l = 0.0f;
    for (int s = 0; s < p.splits; ++s) {
        const float2 ml = p.part_ml[s * rows + row];
        if (ml.y == 0.0f) continue;                             // this split saw no key of the row: its output was not written
        const float w = ptx::ex2_approx(ml.x - ref);
        l = fmaf(w, ml.y, l);
        const float* o = p.part_o + (s * rows + row) * D;
        if constexpr (D == 128) {
            const float4 v = reinterpret_cast<const float4*>(o)[lane];
            acc[0] = fmaf(w, v.x, acc[0]); acc[1] = fmaf(w, v.y, acc[1]); acc[2] = fmaf(w, v.z, acc[2]); acc[3] = fmaf(w, v.w, acc[3]);
        } else {
            const float2 v = reinterpret_cast<const float2*>(o)[lane];
            acc[0] = fmaf(w, v.x, acc[0]); acc[1] = fmaf(w, v.y, acc[1]);
        }
    }
    const int i = (int)(row % p.h.seq_q);
    const int64_t bh = row / p.h.seq_q;
    const bool empty = l == 0.0f;
    const float inv = empty ? 0.0f : (BF16 ? kCutScale : 1.0f) / l;
    uint16_t* out = O + (bh / p.h.heads) * p.h.o_s[0] + (bh % p.h.heads) * p.h.o_s[1] + i * p.h.o_s[2] + lane * (D / 32);
#pragma unroll
    for (int k = 0; k < D / 32; k += 2) *reinterpret_cast<uint32_t*>(out + k) = round_pair<BF16>(acc[k] * inv, acc[k + 1] * inv);
    if (lane == 0) p.lse[row] = empty ? -CUDART_INF_F : (ref + log2f(l) - (BF16 ? kCutScaleLog2 : 0.0f)) * kLn2;
}

template <int D, bool BF16>
static int launch(FwdParams& p, const FwdPlan& plan, const void* Q, const void* K, const void* V, void* O, cudaStream_t s) {
    CUtensorMap mq, mk, mv, mo;
    const int q_rows = plan.packed ? p.h.seq_q : kTile, q_heads = plan.packed ? p.h.group : 1;
    int rc = make_map(&mq, &p.q_at, Q, p.h.batch, p.h.heads, p.h.seq_q, D, p.h.q_s, q_rows, q_heads);
    if (rc == EMMYB200_OK) rc = make_map(&mk, &p.k_at, K, p.h.batch, p.h.kv_heads, p.h.seq_k, D, p.h.k_s, kTile, 1);
    if (rc == EMMYB200_OK) rc = make_map(&mv, &p.v_at, V, p.h.batch, p.h.kv_heads, p.h.seq_k, D, p.h.v_s, kTile, 1);
    if (rc == EMMYB200_OK) rc = make_map(&mo, &p.o_at, O, p.h.batch, p.h.heads, p.h.seq_q, D, p.h.o_s, q_rows, q_heads);
    if (rc != EMMYB200_OK) return rc;
    EMMY_CUDA(cudaGetSymbolAddress(reinterpret_cast<void**>(&p.status), g_fwd_status));
    const int64_t ctas = (int64_t)p.h.batch * (plan.packed ? p.h.kv_heads : p.h.heads) * p.tiles * p.splits;
    if (ctas >= (1ll << 31)) return fail(EMMYB200_ERR_SHAPE, "attention_heads_fwd: %lld tiles exceed the grid limit", (long long)ctas);
    const int unit_heads = plan.packed ? p.h.kv_heads : p.h.heads;
    p.order = work_order(p.h.causal != 0, (int64_t)p.h.batch * unit_heads, p.tiles, (int64_t)p.h.seq_k * D * 4 / (plan.packed ? 1 : p.h.group));
    p.by_splits = fast_div(p.splits);
    p.by_unit_heads = fast_div(unit_heads);
    p.by_group = fast_div(p.h.group);
    auto kernel = p.h.n_runs ? heads_fwd_kernel<D, BF16, true> : heads_fwd_kernel<D, BF16, false>;
    EMMY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, FwdSmem<D>::kTotal));
    kernel<<<(unsigned)ctas, kFwdThreads, FwdSmem<D>::kTotal, s>>>(mq, mk, mv, mo, p);
    rc = launch_status("heads_fwd_kernel");
    if (rc != EMMYB200_OK || p.splits == 1) return rc;
    const int64_t rows = (int64_t)p.h.batch * p.h.heads * p.h.seq_q;
    heads_join_kernel<D, BF16><<<(unsigned)((rows + 7) / 8), 256, 0, s>>>(p, static_cast<uint16_t*>(O));
    return launch_status("heads_join_kernel");
}

}  // namespace heads

FwdPlan heads_fwd_plan(const HeadsParams& p) {
    FwdPlan plan;
    // Packed rows: worth it whenever they fit one tile, since the tile's cost does not depend on how many of its rows are used. Not
    // with a bias (its values belong to a head), nor over broadcast query heads (no dimension to load them along).
    plan.packed = p.group > 1 && (int64_t)p.group * p.seq_q <= heads::kTile && p.n_runs == 0 && p.q_s[1] != 0;
    plan.tiles = plan.packed ? 1 : (p.seq_q + heads::kTile - 1) / heads::kTile;
    const int64_t items = (int64_t)p.batch * (plan.packed ? p.kv_heads : p.heads) * plan.tiles;
    // Splitting the keys costs a second launch and a set-up per CTA: worth it while there is less than one tile per SM (256 tiles
    // of 64 key tiles each: 152 us whole, 171 us in two; 32 tiles: 126 us whole, 35 us in eight; 8 tiles: 121 us whole, 22 us in
    // sixteen). Then as many CTAs as are resident at once, of at least four key tiles each, none of them shorter than it has to be.
    const int64_t key_tiles = (p.seq_k + heads::kTile - 1) / heads::kTile, slots = 2 * sm_count();
    plan.splits = 1;
    if (items < sm_count()) {
        const int64_t most = std::max<int64_t>(1, std::min<int64_t>(slots / items, key_tiles / 4));
        const int64_t each = (key_tiles + most - 1) / most;
        plan.splits = (int)((key_tiles + each - 1) / each);
    }
    plan.rows = (int64_t)p.batch * p.heads * p.seq_q;
    return plan;
}

bool heads_sm100_takes(const HeadsParams& p, int dtype, int d, const void* Q, const void* K, const void* V, const void* O) {
    using namespace heads;
    return (dtype == EMMYB200_F16 || dtype == EMMYB200_BF16) && (d == 64 || d == 128) && p.seq_k > 0 && p.seq_q > 0 &&
           map_fits(Q, p.batch, p.heads, p.seq_q, p.q_s) && map_fits(K, p.batch, p.kv_heads, p.seq_k, p.k_s) &&
           map_fits(V, p.batch, p.kv_heads, p.seq_k, p.v_s) && map_fits(O, p.batch, p.heads, p.seq_q, p.o_s);
}

int heads_fwd_sm100(int dtype, int d, const HeadsParams& hp, const FwdPlan& plan, const void* Q, const void* K, const void* V, void* O, float* lse,
                    void* workspace, cudaStream_t s) {
    heads::FwdParams p = {};
    p.h = hp;
    p.packed = plan.packed;
    p.tiles = plan.tiles;
    p.splits = plan.splits;
    p.lse = lse;
    p.part_ml = static_cast<float2*>(workspace);
    p.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + fwd_part_offset(plan));
    p.wait_limit_ns = wait_limit_ns();
    const bool bf16 = dtype == EMMYB200_BF16;
    if (d == 128) return bf16 ? heads::launch<128, true>(p, plan, Q, K, V, O, s) : heads::launch<128, false>(p, plan, Q, K, V, O, s);
    return bf16 ? heads::launch<64, true>(p, plan, Q, K, V, O, s) : heads::launch<64, false>(p, plan, Q, K, V, O, s);
}

int heads_fwd_read_status(uint32_t* out) {
    uint32_t zero = 0;
    EMMY_CUDA(cudaDeviceSynchronize());
    EMMY_CUDA(cudaMemcpyFromSymbol(out, heads::g_fwd_status, sizeof(uint32_t)));
    if (*out) EMMY_CUDA(cudaMemcpyToSymbol(heads::g_fwd_status, &zero, sizeof(uint32_t)));
    return EMMYB200_OK;
}

}  // namespace emmy
