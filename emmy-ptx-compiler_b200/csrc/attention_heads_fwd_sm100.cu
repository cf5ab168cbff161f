// Attention over heads, forward, on the tensor cores: f16 / bf16, d = 64 or 128.
//
// A CTA owns 128 query rows of a head and walks the keys 64 at a time. Warp 0 loads (TMA: the Q tile, rings of 64-row K and V
// stages), warp 1 issues the products (S = Q K^T into tensor memory, O += P V with P read from there, over the S it came from), and two groups of four warps
// take the 64-key tiles in turn, one thread per row: while one group takes exponentials the products of the other's tile run. The
// groups share nothing until the end: each keeps its own running maximum, sum and output accumulator, as if the row's keys had been
// split over two CTAs, and the two are joined in the epilogue. The maximum is raised only when it grows by more than 2^8, so O is
// rescaled rarely. (Before, two threads of different warps shared a row of a 128-key tile and traded its maximum through shared memory,
// with everything on one chain S -> maximum -> trade -> exponentials -> O: 2200 cycles per 128 x 128 tile with two CTAs on the SM.)
//   d = 128   one CTA per SM; Q is written to tensor memory once and read from there (a product with N = 64 and both operands in
//             shared memory takes 48 cycles per step instead of 32), and S has three buffers, so that a group's next S is there when its
//             tile is done (512 columns: S 3 x 64, O 2 x 128, Q 64)
//   d = 64    two CTAs per SM of 256 columns, one S buffer per group: the exponentials are the limit (512 cycles of the transcendental
//             unit per 128 x 64 tile against 320 of products), and the other CTA fills the gaps
//
// Beyond plain attention: the log-sum-exp of every row; grouped heads and strides through 4-D tensor maps; a key count per
// batch entry (V rows behind it are cleared in shared memory before the product reads them, scores are masked by selection, so nothing
// there is ever used); causal masks from either end; the relative position bias, one number for blocks far from the diagonal, else 95
// looked-up values per warp.
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
    static constexpr int kStage = kHalf * D * 2;
    static constexpr int kStagesK = 4, kStagesV = 6;                    // V is held from its load to the end of the softmax
    static constexpr int kBarOffset = (2 + kStagesK + kStagesV) * kStage;      // behind the Q tile and the rings
    static constexpr int kMlOffset = kBarOffset + 512;                  // [2 groups][128] maximum and sum
    static constexpr int kBiasOffset = kMlOffset + 2048;
    static constexpr int kTotal = kBiasOffset + (int)sizeof(BiasShared) + 1024;
    static_assert(D == 128 || (kTotal > 77824 && kTotal <= 115712), "two CTAs of 256 tensor-memory columns on an SM, never three");
};

template <int D, bool BF16, bool BIAS>
__global__ void __launch_bounds__(kFwdThreads, D == 64 ? 2 : 1)
heads_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                 const __grid_constant__ CUtensorMap map_o, const __grid_constant__ FwdParams p) {
    using S = FwdSmem<D>;
    using Mma = Products<D, BF16>;
    constexpr int kChunks = D / 64, kStagesK = S::kStagesK, kStagesV = S::kStagesV;
    constexpr bool kQInTmem = D == 128;
    constexpr int kBuffers = D == 128 ? 3 : 2;                          // of S: tile h uses buffer h mod kBuffers
    constexpr uint32_t kColO = 64 * kBuffers, kColQ = kColO + 2 * D, kTmemCols = D == 128 ? 512 : 256;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));
    const uint32_t q_smem = smem_base;
    auto k_smem = [&](int s) { return smem_base + (2 + s) * S::kStage; };
    auto v_smem = [&](int s) { return smem_base + (2 + kStagesK + s) * S::kStage; };
    const uint32_t bar_base = smem_base + S::kBarOffset;
    const uint32_t q_full = bar_base, q_ready = kQInTmem ? bar_base + 120 : q_full, acc_full = bar_base + 8, ml_ready = bar_base + 16, staged = bar_base + 24, s_full = bar_base + 32 /* per buffer */,
                   p_ready = bar_base + 64 /* per buffer: a group may be two tiles ahead of the issuer */, o_done = bar_base + 96 /* per group */,
                   k_full = bar_base + 128, k_empty = k_full + 8 * kStagesK,
                   v_full = k_empty + 8 * kStagesK, v_empty = v_full + 8 * kStagesV;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_gen + S::kBarOffset + 112);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    float2* ml = reinterpret_cast<float2*>(smem_gen + S::kMlOffset);
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
    const int all_tiles = (key_end + kHalf - 1) / kHalf;
    int first = 0, n_it = all_tiles;                                    // this CTA's tiles
    if (p.splits > 1) {
        first = (int)((long long)all_tiles * split / p.splits);
        n_it = (int)((long long)all_tiles * (split + 1) / p.splits) - first;
    }
    const WaitCtx wctx{abort_flag, p.status, p.wait_limit_ns};

    auto load_k = [&](int s, int it) {
        ptx::mbar_arrive_expect_tx(k_full + 8 * s, S::kStage);
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
            ptx::tma_load_4d(k_smem(s) + c * Mma::kPiece, &map_k, k_full + 8 * s, c * 64, (first + it) * kHalf, hk * p.k_at.head, b * p.k_at.batch);
    };
    auto load_v = [&](int s, int it) {
        ptx::mbar_arrive_expect_tx(v_full + 8 * s, S::kStage);
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
            ptx::tma_load_4d(v_smem(s) + c * Mma::kPiece, &map_v, v_full + 8 * s, c * 64, (first + it) * kHalf, hk * p.v_at.head, b * p.v_at.batch);
    };
    if (threadIdx.x == 0) {
        ptx::mbar_init(q_full, 1); ptx::mbar_init(acc_full, 1);
        if (kQInTmem) ptx::mbar_init(q_ready, 8); ptx::mbar_init(ml_ready, 8); ptx::mbar_init(staged, 8);
        for (int y = 0; y < kBuffers; ++y) { ptx::mbar_init(s_full + 8 * y, 1); ptx::mbar_init(p_ready + 8 * y, 4); }
        ptx::mbar_init(o_done, 1); ptx::mbar_init(o_done + 8, 1);
        for (int s = 0; s < kStagesK; ++s) { ptx::mbar_init(k_full + 8 * s, 1); ptx::mbar_init(k_empty + 8 * s, 1); }
        for (int s = 0; s < kStagesV; ++s) { ptx::mbar_init(v_full + 8 * s, 1); ptx::mbar_init(v_empty + 8 * s, 1); }
        *abort_flag = 0;
        ptx::mbar_fence_init();
        if (n_it > 0) {                                                 // the first loads fly while the CTA sets itself up
            ptx::mbar_arrive_expect_tx(q_full, box_rows * D * 2);
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
                ptx::tma_load_4d(q_smem + c * (kTile * 128), &map_q, q_full, c * 64, row0, head0 * p.q_at.head, b * p.q_at.batch);
            load_k(0, 0);
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
            int ks = 0, vs = 0;
            uint32_t k_phase = 1, v_phase = 1;
            for (int it = 0; it < n_it; ++it) {
                if (it > 0) {
                    if (!bounded_wait(wctx, k_empty + 8 * ks, k_phase, 0x04010000u | (it & 0xffff))) break;
                    load_k(ks, it);
                }
                if (!bounded_wait(wctx, v_empty + 8 * vs, v_phase, 0x04020000u | (it & 0xffff))) break;
                load_v(vs, it);
                if (++ks == kStagesK) { ks = 0; k_phase ^= 1; }
                if (++vs == kStagesV) { vs = 0; v_phase ^= 1; }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---- MMA issuer, the whole warp for its elected lane: S(0) .. | O += P(i) V(i), S(i + kBuffers) | ... -----------
        {
            const uint32_t lead = ptx::elect_lead();
            const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
            const int tiles = __shfl_sync(0xffffffffu, n_it, 0);
            int ks = 0, vs = 0, next = 0, at = 0;               // stages; buffers of the next S and of tile it
            uint32_t k_phase = 0, v_phase = 0, p_phase = 0;
            auto s_product = [&](int it) {
                if (!warp_spin(wctx, k_full + 8 * ks, k_phase, 0x04030000u | (it & 0xffff))) return false;
                ptx::tc_fence_after_sync();
                if constexpr (kQInTmem) Mma::scores_ts(lead, tmem + 64 * next, tmem + kColQ, k_smem(ks));
                else Mma::scores_ss(lead, tmem + 64 * next, q_smem, k_smem(ks));
                ptx::mma_commit_lead(lead, s_full + 8 * next);
                if (++next == kBuffers) next = 0;
                ptx::mma_commit_lead(lead, k_empty + 8 * ks);
                if (++ks == kStagesK) { ks = 0; k_phase ^= 1; }
                return true;
            };
            bool ok = tiles == 0 || warp_spin(wctx, q_ready, 0, 0x04040000u);
            for (int it = 0; it < kBuffers && it < tiles && ok; ++it) ok = s_product(it);
            for (int it = 0; it < tiles && ok; ++it) {
                if (!(ok = warp_spin(wctx, v_full + 8 * vs, v_phase, 0x04050000u | (it & 0xffff)))) break;
                if (!(ok = warp_spin(wctx, p_ready + 8 * at, p_phase, 0x04060000u | (it & 0xffff)))) break;
                ptx::tc_fence_after_sync();
                Mma::grads(lead, tmem + kColO + D * (it & 1), tmem + 64 * at, v_smem(vs), it < 2);
                ptx::mma_commit_lead(lead, o_done + 8 * (it & 1));
                ptx::mma_commit_lead(lead, v_empty + 8 * vs);
                if (it + kBuffers < tiles && !(ok = s_product(it + kBuffers))) break;
                if (++at == kBuffers) { at = 0; p_phase ^= 1; }
                if (++vs == kStagesV) { vs = 0; v_phase ^= 1; }
            }
            if (ok) ptx::mma_commit_lead(lead, acc_full);
        }
        __syncwarp();
    } else {
        // ---- softmax: one thread per query row; group x takes tiles x, x + 2, ... -----------------------------------------
        const int w = warp - 2, quarter = warp & 3, x = w >> 2;
        const int row_in_tile = quarter * 32 + lane;
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        const uint32_t o_row = tmem_base + lane_base + kColO + x * D;
        const int query = p.packed ? row_in_tile % p.h.seq_q : row0 + row_in_tile;
        const int sees = p.h.causal ? min(n_keys, query + offset + 1) : n_keys;         // keys 0 .. sees - 1
        float m_run = -CUDART_INF_F;      // the max the exponentials are taken against (log2 units)
        float l_run = 0.0f;
        bool ok = true;
        if (kQInTmem && n_it > 0 && (ok = warp_wait(wctx, q_full, 0, 0x040d0000u))) {            // each group brings half of Q to tensor memory
            row_to_tmem<D / 64>(tmem_base + lane_base + kColQ, q_smem, row_in_tile, x * (D / 64));
            ptx::tmem_st_wait();
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(q_ready);
        }
        WarpBias wb(p.h);
        int buffer = x;                                         // of tile it
        uint32_t buffer_phase = 0;
        for (int it = x; it < n_it && ok; it += 2) {
            const int key0 = (first + it) * kHalf;
            const uint32_t s_at = tmem_base + lane_base + 64 * buffer;
            float c = p.h.scale_log2, add = 0.0f;               // a score in log2 units is c * s + add
            bool looked_up = false;
            if constexpr (BIAS) looked_up = !wb.block(bias, bias.value, w, lane, p.h.n_runs, key0 - (row0 + quarter * 32 + 31 + offset));
            ok = warp_wait(wctx, s_full + 8 * buffer, buffer_phase, 0x04070000u | (it & 0xffff));
            if (!ok) break;
            ptx::tc_fence_after_sync();
            uint32_t r[64];
            ptx::tmem_ld_32x32b_x32(s_at, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
            ptx::tmem_ld_32x32b_x32(s_at + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
            ptx::tmem_ld_wait();
            if constexpr (BIAS) {
                if (looked_up) {
                    const float* at = bias.by_dist[w] + 31 - lane;
#pragma unroll
                    for (int i = 0; i < 64; ++i) r[i] = __float_as_uint(fmaf(__uint_as_float(r[i]), c, at[i]));
                    c = 1.0f;
                } else {
                    add = wb.same;
                }
            }
            const int valid = sees - key0;                      // columns that are seen
            if (valid < 64) {
#pragma unroll
                for (int i = 0; i < 64; ++i)
                    if (i >= valid) r[i] = __float_as_uint(-CUDART_INF_F);
            }
            float ext[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) ext[i] = __uint_as_float(r[i]);
#pragma unroll
            for (int i = 8; i < 64; ++i) ext[i & 7] = fmaxf(ext[i & 7], __uint_as_float(r[i]));
            ext[0] = fmaxf(fmaxf(fmaxf(ext[0], ext[1]), fmaxf(ext[2], ext[3])), fmaxf(fmaxf(ext[4], ext[5]), fmaxf(ext[6], ext[7])));
            const float m_tile = fmaf(ext[0], c, add);
            const bool raise = m_tile > m_run + 8.0f;           // from -inf: with the first key the row sees
            if (__any_sync(0xffffffffu, raise)) {
                const float f = raise ? ptx::ex2_approx(m_run - m_tile) : 1.0f;
                if (it >= 2) {                                  // O holds the group's earlier tiles, once the last of them has been added
                    ok = warp_wait(wctx, o_done + 8 * x, ((it - 2) >> 1) & 1, 0x04080000u | (it & 0xffff));
                    if (!ok) break;
                    ptx::tc_fence_after_sync();
#pragma unroll 1
                    for (int col = 0; col < D; col += 8) {      // few registers: the S row is still live
                        uint32_t o[8];
                        ptx::tmem_ld_32x32b_x8(o_row + col, o);
                        ptx::tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        ptx::tmem_st_32x32b_x8(o_row + col, o);
                    }
                }
                l_run *= f;
                if (raise) m_run = m_tile;
            }
            const float ref = m_run == -CUDART_INF_F ? 0.0f : m_run;            // nothing seen so far: every exponential is 2^-inf
            const float shift = add - ref + (BF16 ? kCutScaleLog2 : 0.0f);
            const float2 c2 = make_float2(c, c), s2 = make_float2(shift, shift);
            float2 sum2[4] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
                uint32_t pk[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 y = fma2(f2(r[ch * 32 + 2 * i], r[ch * 32 + 2 * i + 1]), c2, s2);
                    const float2 e = make_float2(ptx::ex2_approx(y.x), ptx::ex2_approx(y.y));
                    sum2[i & 3] = add2(sum2[i & 3], e);
                    pk[i] = operand_pair<BF16>(e);
                }
                ptx::tmem_st_32x32b_x16(s_at + ch * 16, pk);
            }
            const float2 tot = add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3]));
            l_run += tot.x + tot.y;
            // V rows behind the key count hold whatever the caller left there: cleared before the product multiplies them by P's zeros
            const int live = n_keys - key0;
            if (live < kHalf && n_keys < p.h.seq_k) {
                const int vs = it % kStagesV;
                ok = warp_wait(wctx, v_full + 8 * vs, (it / kStagesV) & 1, 0x04090000u | (it & 0xffff));
                if (!ok) break;
                for (int e = live * 8 + row_in_tile; e < kHalf * 8; e += 128)           // 16-byte pieces of the rows
#pragma unroll
                    for (int ch = 0; ch < kChunks; ++ch)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(v_smem(vs) + ch * Mma::kPiece + e * 16), "r"(0) : "memory");
                ptx::fence_proxy_async_smem();
            }
            ptx::tmem_st_wait();
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(p_ready + 8 * buffer);
            buffer += 2;
            if (buffer >= kBuffers) { buffer -= kBuffers; buffer_phase ^= 1; }
        }
        // ---- the two groups joined; each writes half of the columns ----------------------------------------------------------
        if (ok) {
            ml[x * 128 + row_in_tile] = make_float2(m_run, l_run);
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(ml_ready);
            ok = warp_wait(wctx, ml_ready, 0, 0x040a0000u) && warp_wait(wctx, acc_full, 0, 0x040b0000u);
        }
        if (ok) {
            ptx::tc_fence_after_sync();
            const float2 a = ml[row_in_tile], z = ml[128 + row_in_tile];
            const bool has_a = a.y != 0.0f, has_z = z.y != 0.0f;        // otherwise the group saw no key of the row
            const float m = fmaxf(has_a ? a.x : -CUDART_INF_F, has_z ? z.x : -CUDART_INF_F), ref = m == -CUDART_INF_F ? 0.0f : m;
            const float fa = has_a ? ptx::ex2_approx(a.x - ref) : 0.0f, fz = has_z ? ptx::ex2_approx(z.x - ref) : 0.0f;
            const float l = (has_a ? a.y * fa : 0.0f) + (has_z ? z.y * fz : 0.0f);
            const bool empty = !has_a && !has_z;
            const bool live_row = p.packed ? row_in_tile < box_rows : query < p.h.seq_q;
            const int head = p.packed ? head0 + row_in_tile / p.h.seq_q : head0;
            const int64_t rows = (int64_t)p.h.batch * p.h.heads * p.h.seq_q, out_row = ((int64_t)b * p.h.heads + head) * p.h.seq_q + query;
            const bool parts = p.splits > 1;
            const float inv = parts ? 1.0f : empty ? 0.0f : (BF16 ? kCutScale : 1.0f) / l;
            const float2 wa = make_float2(fa * inv, fa * inv), wz = make_float2(fz * inv, fz * inv);
#pragma unroll 1
            for (int ch = 0; ch < D / 64; ++ch) {               // this group's D / 2 columns, 32 at a time
                const int col = x * (D / 2) + ch * 32;
                uint32_t oa[32], oz[32];
                ptx::tmem_ld_32x32b_x32(tmem_base + lane_base + kColO + col, oa);
                ptx::tmem_ld_32x32b_x32(tmem_base + lane_base + kColO + D + col, oz);
                ptx::tmem_ld_wait();
                float2 o[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {                  // what a group without keys left in its accumulator is not looked at
                    const float2 va = has_a ? mul2(f2(oa[2 * i], oa[2 * i + 1]), wa) : make_float2(0.0f, 0.0f);
                    o[i] = has_z ? fma2(f2(oz[2 * i], oz[2 * i + 1]), wz, va) : va;
                }
                if (parts) {
                    if (live_row && !empty) {
                        float4* dst = reinterpret_cast<float4*>(p.part_o + (split * rows + out_row) * D + col);
#pragma unroll
                        for (int i = 0; i < 8; ++i) dst[i] = make_float4(o[2 * i].x, o[2 * i].y, o[2 * i + 1].x, o[2 * i + 1].y);
                    }
                } else {                                        // every product has completed: the output is staged over Q and leaves through TMA
                    uint32_t v[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = round_pair<BF16>(o[i].x, o[i].y);
                    stage_row(q_smem, row_in_tile, col, v);
                }
            }
            if (parts) {
                if (live_row && x == 0) p.part_ml[split * rows + out_row] = make_float2(m, empty ? 0.0f : l);
            } else {
                if (live_row && x == 0) p.lse[out_row] = empty ? -CUDART_INF_F : (m + log2f(l) - (BF16 ? kCutScaleLog2 : 0.0f)) * kLn2;
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(staged);
                if (w == 0 && lane == 0 && bounded_wait(wctx, staged, 0, 0x040c0000u)) {
#pragma unroll
                    for (int ch = 0; ch < kChunks; ++ch)        // rows that do not exist are dropped
                        ptx::tma_store_4d(&map_o, q_smem + ch * (kTile * 128), ch * 64, row0, head0 * p.o_at.head, b * p.o_at.batch);
                    ptx::tma_store_commit();
                    ptx::tma_store_wait_read<0>();              // shared memory has been read; the grid's end covers the writes
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
    if (rc == EMMYB200_OK) rc = make_map(&mk, &p.k_at, K, p.h.batch, p.h.kv_heads, p.h.seq_k, D, p.h.k_s, kHalf, 1);
    if (rc == EMMYB200_OK) rc = make_map(&mv, &p.v_at, V, p.h.batch, p.h.kv_heads, p.h.seq_k, D, p.h.v_s, kHalf, 1);
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

FwdPlan heads_fwd_plan(const HeadsParams& p, int64_t d) {
    FwdPlan plan;
    // Packed rows: worth it whenever they fit one tile, since the tile's cost does not depend on how many of its rows are used. Not
    // with a bias (its values belong to a head), nor over broadcast query heads (no dimension to load them along).
    plan.packed = p.group > 1 && (int64_t)p.group * p.seq_q <= heads::kTile && p.n_runs == 0 && p.q_s[1] != 0;
    plan.tiles = plan.packed ? 1 : (p.seq_q + heads::kTile - 1) / heads::kTile;
    const int64_t items = (int64_t)p.batch * (plan.packed ? p.kv_heads : p.heads) * plan.tiles;
    // Splitting the keys costs a second launch and a set-up per CTA: worth it while there is less than one tile per SM (caches of 8192
    // keys, d = 128: 256 tiles 140 us whole, 145 us in two; 32 tiles 60 us whole, 33 us in four, 36 us in eight; 8 tiles 57 us whole, 21 us in
    // eight to sixteen). Then at most as many CTAs as are resident at once, of at least four times 128 keys each, none of them shorter
    // than it has to be.
    const int64_t key_tiles = (p.seq_k + heads::kTile - 1) / heads::kTile, slots = (d == 64 ? 2 : 1) * sm_count();
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
