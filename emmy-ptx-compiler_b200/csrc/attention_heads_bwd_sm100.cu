// Attention over heads, backward, on the tensor cores: f16 / bf16, d = 64 or 128.
//
// With P_ij = exp(s_ij - lse_i) and dS_ij = P_ij (dO_i . v_j - D_i), D_i = dO_i . O_i, the gradients are five products per tile of
// queries x keys. Two kinds of CTAs recompute P, each writing what it owns, so nothing is accumulated across CTAs and results
// are the same every time; the two score-sized products are done in both, seven in all where one kernel with atomic
// additions into dQ would do five:
//
//   dkv_block   owns 128 keys of a key head and walks the queries of every query head that reads it, 64 at a time.
//               Everything is transposed, keys are rows: S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q.
//   dq_block    owns 128 queries and walks the keys, 64 at a time: S = Q K^T, dP = dO V^T, dQ += dS K.
//
// One CTA per SM, 320 threads: warp 0 TMA (rings of 64-row stages), warp 1 issues the products, and two groups of four warps
// do the arithmetic between them, taking the 64-column tiles in turn, one thread per row: while one group takes exponentials the products of
// the other's tile run. Tensor memory (512 columns) sets the shape: with 128-column tiles there is room for one tile of S and dP
// beside the accumulators, and a chain S -> exponentials -> P -> dV -> next S that left the tensor pipe idle for 40-58 % of the
// time (measured: 3600 and 3790 cycles per 128 x 128 tile where the products take 2048 and 1536). With 64 columns S and dP have two
// buffers each. P (16 bits, 32 columns) goes back over the S tile it came from, dS over dP.
// A product with N = 64 is bound by shared memory if both operands come from there (A is read again for every 64 columns: 48
// cycles per 16-deep step against 32 with A in tensor memory), so where there is room the operand that stays is written to tensor memory
// once and read from there: Q and dO in dq; K and V in dkv for d = 64.
//   columns, dkv: S 2 x 64, dP 2 x 64, dV d, dK d (K 32, V 32)      dq: S 2 x 64, dP 2 x 64, Q d / 2, dO d / 2, dQ d
//
// Row terms come from the rows kernel already negated and shifted: nlse2 = -lse log2(e) + shift, -inf for rows that see
// nothing or lie behind seq_q, so that P = 2^(scale log2(e) q.k + bias + nlse2) needs no test. The shift scales P by what
// 16 bits want: kCutScale before bf16 values are cut, 2^14 for f16, whose small probabilities would lose bits. dS inherits the factor
// and, in f16, a power of two per key head on top, chosen from the largest row norms of dO and V so that |dS| stays below 2^15: a
// tiny or huge incoming gradient keeps its bits. bf16 dS is rounded, not cut: it goes into two of the three gradients, and the two
// additions per pair cost 1 %. What is left of the factors is taken out at the end.
//
// Measured (bf16 unless said): 64 units of 4096 x 4096 x 128 in 1.66 ms, 0.83 PFLOP/s of the five products (1.16 of the seven done)
// with the power cap active; 64 heads over 16 key heads, 2048, causal: 0.26 ms; f16, d = 64, 96 units of 512 with bias: 76 us of this kernel.
// Bound by: long sequences the tensor pipe under the power cap; short ones a CTA's set-up and end (some 8000 cycles of 25000 for 12
// tiles of 64), with the bias the arithmetic between the products (one group's tile takes 2000 cycles near the diagonal).
#include <math_constants.h>

#include "attention_heads_sm100.cuh"

namespace emmy {
namespace heads {

constexpr int kBwdThreads = 320;
constexpr int kF16Shift = 14;

struct BwdParams {
    HeadsParams h;
    HeadsGrads g;
    MapAt q_at, k_at, v_at, do_at, dq_at, dk_at, dv_at;
    int q_tiles, k_tiles;
    WorkOrder order_dkv, order_dq;
    FastDiv by_heads, by_kv_heads, by_group;
    int dkv_blocks;                     // blocks from here on work on dQ
    unsigned long long wait_limit_ns;
    uint32_t* status;
};
struct BwdMaps {
    CUtensorMap q, d_o, k, v;           // stages of 64 rows
    CUtensorMap k_tile, v_tile, dq, dk, dv;     // 128 rows
};

__device__ uint32_t g_bwd_status;

template <int D>
struct BwdSmem {
    static constexpr int kStage = kHalf * D * 2;
    static constexpr int kStages = 4;                                   // dkv: of Q and of dO, beside 128 rows of K and V
    static constexpr int kStagesDq = 6;                                 // dq: of K and of V
    static constexpr int kRing = 12 * kStage;                           // either way: 4 + 2 x 4, 2 x 6 stages
    static constexpr int kRowsOffset = kRing;                           // dkv: [stage][nlse2 64, ndelta 64]
    static constexpr int kBarOffset = kRowsOffset + kStages * 512;
    static constexpr int kBiasOffset = kBarOffset + 512;
    static constexpr int kSumsOffset = kBiasOffset + (int)sizeof(BiasShared);
    static constexpr int kTotal = kSumsOffset + 8 * kHeadsMaxRuns * 4 + 1024;
};

// The power of two dS is scaled by in f16: |dS| 2^14 g <= 2^15 from |dO . v - D| <= 2 max|dO| max|v|, given the largest squared row norms.
__device__ __forceinline__ float ds_scale(float do_norm, float v_norm) {
    const float bound = sqrtf(do_norm) * sqrtf(v_norm);
    if (!(bound > 0.0f) || !(bound < CUDART_INF_F)) return 1.0f;
    return __int_as_float(((int)fminf(fmaxf(floorf(-log2f(bound)), -100.0f), 100.0f) + 127) << 23);
}

template <int D, bool BF16, bool BIAS>
__device__ __forceinline__ void dkv_block(const BwdMaps& m, const BwdParams& p, int item) {
    const CUtensorMap &map_q = m.q, &map_k = m.k_tile, &map_v = m.v_tile, &map_do = m.d_o, &map_dk = m.dk, &map_dv = m.dv;
    using S = BwdSmem<D>;
    using Mma = Products<D, BF16>;
    constexpr int kChunks = D / 64, kStages = S::kStages;
    constexpr bool kKvInTmem = D == 64;
    constexpr uint32_t kColS = 0, kColDP = 128, kColDV = 256, kColDK = 256 + D, kColK = 384, kColV = 416;      // K and V: D = 64 only
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));
    const uint32_t k_smem = smem_base, v_smem = smem_base + 2 * S::kStage;
    auto q_smem = [&](int s) { return smem_base + (4 + s) * S::kStage; };
    auto do_smem = [&](int s) { return smem_base + (4 + kStages + s) * S::kStage; };
    const uint32_t rows_smem = smem_base + S::kRowsOffset;
    const uint32_t bar_base = smem_base + S::kBarOffset;
    const uint32_t kv_full = bar_base, kv_ready = kKvInTmem ? bar_base + 8 : kv_full, acc_full = bar_base + 16, s_full = bar_base + 24 /* per group */, dp_full = bar_base + 40,
                   p_ready = bar_base + 56, ds_ready = bar_base + 72, staged = bar_base + 104, full = bar_base + 128, empty = full + 8 * kStages;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_gen + S::kBarOffset + 120);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    BiasShared& bias = *reinterpret_cast<BiasShared*>(smem_gen + S::kBiasOffset);

    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const WorkItem work = p.order_dkv(item);
    const int kt = work.tile, bk = work.unit;                   // causal: the first key tiles see the most queries
    const int b = p.by_kv_heads(bk), hk = bk - b * p.h.kv_heads;
    const int key0 = kt * kTile;
    const int n_keys = heads_key_count(p.h, b), offset = heads_offset(p.h, n_keys);
    const int q_tiles = (p.h.seq_q + kHalf - 1) / kHalf;
    const int first_qt = p.h.causal ? max(0, key0 - offset) / kHalf : 0;       // queries before it see none of these keys
    const int per_head = key0 < n_keys ? max(0, q_tiles - first_qt) : 0;
    const int n_it = per_head * p.h.group;
    const WaitCtx wctx{abort_flag, p.status, p.wait_limit_ns};

    auto load_stage = [&](int s, int gi, int qt) {
        const int h = hk * p.h.group + gi, row0 = qt * kHalf;
        ptx::mbar_arrive_expect_tx(full + 8 * s, 2 * S::kStage + 512);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            ptx::tma_load_4d(q_smem(s) + c * Mma::kPiece, &map_q, full + 8 * s, c * 64, row0, h * p.q_at.head, b * p.q_at.batch);
            ptx::tma_load_4d(do_smem(s) + c * Mma::kPiece, &map_do, full + 8 * s, c * 64, row0, h * p.do_at.head, b * p.do_at.batch);
        }
        const int64_t at = ((int64_t)b * p.h.heads + h) * p.g.pad_q + row0;
        ptx::bulk_load(rows_smem + s * 512, p.g.lse2 + at, 256, full + 8 * s);
        ptx::bulk_load(rows_smem + s * 512 + 256, p.g.delta + at, 256, full + 8 * s);
    };
    int load_it = 0, load_gi = 0, load_qt = first_qt, load_s = 0;               // the producer's next tile and stage
    uint32_t load_phase = 1;
    auto advance = [&]() {
        if (++load_s == kStages) { load_s = 0; load_phase ^= 1; }
        if (++load_qt == q_tiles) { load_qt = first_qt; ++load_gi; }
        ++load_it;
    };
    if (threadIdx.x == 0) {
        ptx::mbar_init(kv_full, 1); ptx::mbar_init(acc_full, 1);
        if (kKvInTmem) ptx::mbar_init(kv_ready, 8);
        for (int x = 0; x < 2; ++x) {
            ptx::mbar_init(s_full + 8 * x, 1); ptx::mbar_init(dp_full + 8 * x, 1); ptx::mbar_init(p_ready + 8 * x, 4); ptx::mbar_init(ds_ready + 8 * x, 4); ptx::mbar_init(staged + 8 * x, 4);
        }
        for (int s = 0; s < kStages; ++s) {
            ptx::mbar_init(full + 8 * s, 1); ptx::mbar_init(empty + 8 * s, 1);
        }
        *abort_flag = 0;
        ptx::mbar_fence_init();
        if (n_it > 0) {                                         // the first loads fly while the CTA sets itself up
            ptx::mbar_arrive_expect_tx(kv_full, 4 * S::kStage);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                ptx::tma_load_4d(k_smem + c * (kTile * 128), &map_k, kv_full, c * 64, key0, hk * p.k_at.head, b * p.k_at.batch);
                ptx::tma_load_4d(v_smem + c * (kTile * 128), &map_v, kv_full, c * 64, key0, hk * p.v_at.head, b * p.v_at.batch);
            }
            load_stage(load_s, load_gi, load_qt);
            advance();
        }
    }
    const int x = (warp - 2) >> 2;                              // group of the warps 2 to 9
    const int key = key0 + (warp & 3) * 32 + lane;
    float do_norm = 0.0f, v_norm = 0.0f;
    if (!BF16 && warp >= 2) {
        do_norm = __ldg(p.g.amax + bk);
        v_norm = __ldg(p.g.amax + (int64_t)p.h.batch * p.h.kv_heads + bk);
    }
    if constexpr (BIAS) load_runs(bias, p.h, warp, kBwdThreads / 32, lane);
    if (warp == 1) {
        ptx::tmem_alloc(ptx::smem_u32(tmem_slot), 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        // ---- TMA producer ------------------------------------------------------------------------------
        if (lane == 0) {
            for (; load_it < n_it; advance()) {
                if (!bounded_wait(wctx, empty + 8 * load_s, load_phase, 0x05010000u | (load_it & 0xffff))) break;
                load_stage(load_s, load_gi, load_qt);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---- MMA issuer: S(0) dP(0) S(1) dP(1) | dV(i) S(i+2) dK(i) dP(i+2) | ... ----------------------------------
        if (n_it > 0) {
            const uint32_t lead = ptx::elect_lead();
            const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
            const int tiles = __shfl_sync(0xffffffffu, n_it, 0);
            auto s_product = [&](int it, int s) {
                if constexpr (kKvInTmem) Mma::scores_ts(lead, tmem + kColS + 64 * (it & 1), tmem + kColK, q_smem(s));
                else Mma::scores_ss(lead, tmem + kColS + 64 * (it & 1), k_smem, q_smem(s));
                ptx::mma_commit_lead(lead, s_full + 8 * (it & 1));
            };
            auto dp_product = [&](int it, int s) {
                if constexpr (kKvInTmem) Mma::scores_ts(lead, tmem + kColDP + 64 * (it & 1), tmem + kColV, do_smem(s));
                else Mma::scores_ss(lead, tmem + kColDP + 64 * (it & 1), v_smem, do_smem(s));
                ptx::mma_commit_lead(lead, dp_full + 8 * (it & 1));
            };
            bool ok = warp_spin(wctx, kv_ready, 0, 0x05030000u);
            for (int it = 0; it < 2 && it < tiles && ok; ++it) {
                if (!(ok = warp_spin(wctx, full + 8 * it, 0, 0x05040000u | it))) break;
                ptx::tc_fence_after_sync();
                s_product(it, it);
                dp_product(it, it);
            }
            int s = 0, next = 2;                                // stages of tiles it and it + 2
            uint32_t next_phase = 0;
            for (int it = 0; it < tiles && ok; ++it) {
                const uint32_t x64 = 64 * (it & 1), phase = (it >> 1) & 1;
                const bool more = it + 2 < tiles;
                if (more && !(ok = warp_spin(wctx, full + 8 * next, next_phase, 0x05050000u | (it & 0xffff)))) break;
                if (!(ok = warp_spin(wctx, p_ready + 8 * (it & 1), phase, 0x05070000u | (it & 0xffff)))) break;
                ptx::tc_fence_after_sync();
                Mma::grads(lead, tmem + kColDV, tmem + kColS + x64, do_smem(s), it == 0);
                if (more) s_product(it + 2, next);
                if (!(ok = warp_spin(wctx, ds_ready + 8 * (it & 1), phase, 0x05080000u | (it & 0xffff)))) break;
                ptx::tc_fence_after_sync();
                Mma::grads(lead, tmem + kColDK, tmem + kColDP + x64, q_smem(s), it == 0);
                ptx::mma_commit_lead(lead, empty + 8 * s);
                if (more) dp_product(it + 2, next);
                if (++s == kStages) s = 0;
                if (++next == kStages) { next = 0; next_phase ^= 1; }
            }
            if (ok) ptx::mma_commit_lead(lead, acc_full);
        }
        __syncwarp();
    } else {
        // ---- probabilities and their gradients: rows are keys, columns queries; group x takes tiles x, x + 2, ... ---------
        const int w = warp - 2, quarter = warp & 3;
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        const uint32_t s_at = tmem_base + lane_base + kColS + x * 64, dp_at = tmem_base + lane_base + kColDP + x * 64;
        bool ok = true;
        if (kKvInTmem && n_it > 0 && (ok = warp_wait(wctx, kv_full, 0, 0x05090000u))) {          // group 0 writes K to tensor memory, group 1 V
            row_to_tmem<D / 32>(tmem_base + lane_base + (x ? kColV : kColK), x ? v_smem : k_smem, quarter * 32 + lane);
            ptx::tmem_st_wait();
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(kv_ready);
        }
        const float g_scale = BF16 ? 1.0f : ds_scale(do_norm, v_norm);
        const float2 g2 = make_float2(g_scale, g_scale);
        WarpBias wb(p.h);
        float* value = reinterpret_cast<float*>(smem_gen + S::kSumsOffset) + w * kHeadsMaxRuns;
        int bias_head = -1;
        int gi = 0, qt = first_qt, s = x;                       // this group's tile and its stage
        uint32_t full_phase = 0;
        if (x == 1 && ++qt == q_tiles) { qt = first_qt; ++gi; }
        for (int it = x; it < n_it && ok; it += 2) {
            const uint32_t phase = (it >> 1) & 1;
            const int q0 = qt * kHalf;                          // this thread's first query
            const float c = p.h.scale_log2;
            bool looked_up = false;
            if constexpr (BIAS) {
                // the table's column changes with the query head; every warp keeps a copy of its own, so that no two warps have to meet
                const int h = hk * p.h.group + gi;
                if (h != bias_head) {
                    bias_head = h;
                    __syncwarp();
                    for (int r = lane; r < p.h.n_runs; r += 32) value[r] = heads_run_bias(p.h, r, h);
                    __syncwarp();
                    wb.reset();
                }
                looked_up = !wb.block(bias, value, w, lane, p.h.n_runs, key0 + quarter * 32 - (q0 + 63 + offset));
            }
            ok = warp_wait(wctx, full + 8 * s, full_phase, 0x050a0000u | (it & 0xffff)) && warp_wait(wctx, s_full + 8 * x, phase, 0x050b0000u | (it & 0xffff));
            if (!ok) break;
            ptx::tc_fence_after_sync();
            const float4* nlse = reinterpret_cast<const float4*>(smem_gen + S::kRowsOffset + s * 512);
            const float4* ndelta = nlse + 16;
            // columns below `hidden` are not seen: queries before the key, or the whole row for keys behind the count
            const int hidden = key >= n_keys ? 64 : (p.h.causal ? key - offset - q0 : 0);
            const bool masked = __any_sync(0xffffffffu, hidden > 0);
            float2 e[32];
            uint32_t r[64];
            ptx::tmem_ld_32x32b_x32(s_at, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
            ptx::tmem_ld_32x32b_x32(s_at + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
            ptx::tmem_ld_wait();
            float cc = c, aa = 0.0f;
            if constexpr (BIAS) {
                aa = wb.same;
                if (looked_up) {
                    const float* at = bias.by_dist[w] + 63 + lane;
#pragma unroll
                    for (int i = 0; i < 64; ++i) r[i] = __float_as_uint(fmaf(__uint_as_float(r[i]), c, at[-i]));
                    cc = 1.0f;
                    aa = 0.0f;
                }
            }
            const float2 c2 = make_float2(cc, cc), a2 = make_float2(aa, aa);
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
#pragma unroll
                for (int i = ch * 16; i < ch * 16 + 16; i += 2) {
                    const float4 nl = nlse[i / 2];
                    float2 n0 = make_float2(nl.x, nl.y), n1 = make_float2(nl.z, nl.w);
                    if constexpr (BIAS) { n0 = add2(n0, a2); n1 = add2(n1, a2); }
                    const float2 y0 = fma2(f2(r[2 * i], r[2 * i + 1]), c2, n0), y1 = fma2(f2(r[2 * i + 2], r[2 * i + 3]), c2, n1);
                    e[i] = make_float2(ptx::ex2_approx(y0.x), ptx::ex2_approx(y0.y));
                    e[i + 1] = make_float2(ptx::ex2_approx(y1.x), ptx::ex2_approx(y1.y));
                }
                if (masked) {
#pragma unroll
                    for (int i = ch * 16; i < ch * 16 + 16; ++i) {
                        if (2 * i < hidden) e[i].x = 0.0f;
                        if (2 * i + 1 < hidden) e[i].y = 0.0f;
                    }
                }
                uint32_t pk[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) pk[i] = operand_pair<BF16>(e[ch * 16 + i]);
                ptx::tmem_st_32x32b_x16(s_at + ch * 16, pk);
            }
            ptx::tmem_st_wait();
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(p_ready + 8 * x);
            ok = warp_wait(wctx, dp_full + 8 * x, phase, 0x050c0000u | (it & 0xffff));
            if (!ok) break;
            ptx::tc_fence_after_sync();
            ptx::tmem_ld_32x32b_x32(dp_at, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
            ptx::tmem_ld_32x32b_x32(dp_at + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
            ptx::tmem_ld_wait();
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
                uint32_t pk[16];
#pragma unroll
                for (int i = ch * 16; i < ch * 16 + 16; i += 2) {
                    const float4 nd = ndelta[i / 2];
                    float2 d0 = mul2(e[i], add2(f2(r[2 * i], r[2 * i + 1]), make_float2(nd.x, nd.y)));
                    float2 d1 = mul2(e[i + 1], add2(f2(r[2 * i + 2], r[2 * i + 3]), make_float2(nd.z, nd.w)));
                    if (masked) {                                       // dP may hold anything there
                        if (2 * i < hidden) d0.x = 0.0f;
                        if (2 * i + 1 < hidden) d0.y = 0.0f;
                        if (2 * i + 2 < hidden) d1.x = 0.0f;
                        if (2 * i + 3 < hidden) d1.y = 0.0f;
                    }
                    if constexpr (!BF16) { d0 = mul2(d0, g2); d1 = mul2(d1, g2); }
                    pk[i - ch * 16] = rounded_pair<BF16>(d0);
                    pk[i - ch * 16 + 1] = rounded_pair<BF16>(d1);
                }
                ptx::tmem_st_32x32b_x16(dp_at + ch * 16, pk);
            }
            ptx::tmem_st_wait();
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(ds_ready + 8 * x);
            // two tiles on
            s += 2;
            if (s >= kStages) { s -= kStages; full_phase ^= 1; }
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (++qt == q_tiles) { qt = first_qt; ++gi; }
        }
        if (ok && n_it > 0) ok = warp_wait(wctx, acc_full, 0, 0x050d0000u);
        if (ok) {                                               // group 0 writes dV, group 1 dK
            ptx::tc_fence_after_sync();
            // dV's factor went with the cut of P; dS still has it
            const float f = (BF16 ? (x ? 1.0f / kCutScale : 1.0f) : 1.0f / (1 << kF16Shift)) * (x ? p.h.scale / g_scale : 1.0f);
            const uint32_t tile = smem_base + x * (2 * S::kStage);      // every load has been used: the tile is staged where the operands were
#pragma unroll 1
            for (int col = 0; col < D; col += 32) {
                uint32_t r[32], v[16];
                if (n_it > 0) {
                    ptx::tmem_ld_32x32b_x32(tmem_base + lane_base + (x ? kColDK : kColDV) + col, r);
                    ptx::tmem_ld_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) r[i] = 0;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = round_pair<BF16>(__uint_as_float(r[2 * i]) * f, __uint_as_float(r[2 * i + 1]) * f);
                stage_row(tile, quarter * 32 + lane, col, v);
            }
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(staged + 8 * x);
            if (quarter == 2 && lane == 0 && bounded_wait(wctx, staged + 8 * x, 0, 0x050e0000u)) {
#pragma unroll
                for (int c = 0; c < kChunks; ++c)               // rows behind seq_k are dropped
                    ptx::tma_store_4d(x ? &map_dk : &map_dv, tile + c * (kTile * 128), c * 64, key0, hk * (x ? p.dk_at.head : p.dv_at.head),
                                      b * (x ? p.dk_at.batch : p.dv_at.batch));
                ptx::tma_store_commit();
                ptx::tma_store_wait_read<0>();     // shared memory has been read; the grid's end covers the writes
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
        ptx::tmem_dealloc(tmem_base, 512);
    }
}

// The gradient of the bias, one warp's share: 32 x 64 blocks of dS. A block inside one run adds to a per-thread sum, which goes
// to the warp's sum of that run when the run changes; other blocks are added up along their 95 diagonals, without atomics: a partial
// sum moves one lane up per column, so that it follows its diagonal and is complete when it reaches lane 31. Four chains of 16 columns run side by
// side (one of 64 was bound by the shuffle's latency: 55 us of dq for 96 units of 512 x 512 x 64, 8 tiles each); what the lanes hold
// after a chain's last column are partial sums of the 32 diagonals that go on into the next. A scan over the diagonals that stops
// where a run begins then gives each run's sum to its last diagonal's lane.
struct RunSums {
    float acc;              // this thread's part of the run
    int run;
    __device__ __forceinline__ void flush(float* sums, int lane) {
        float v = acc;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
        if (lane == 0) sums[run] += v;
        acc = 0.0f;
    }
};

template <int D, bool BF16, bool BIAS>
__device__ __forceinline__ void dq_block(const BwdMaps& m, const BwdParams& p, int item) {
    const CUtensorMap &map_k = m.k, &map_v = m.v, &map_dq = m.dq;
    using S = BwdSmem<D>;
    using Mma = Products<D, BF16>;
    constexpr int kChunks = D / 64, kStages = S::kStagesDq;
    constexpr uint32_t kColS = 0, kColDP = 128, kColQ = 256, kColDO = 320, kColDQ = 384;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));
    auto k_smem = [&](int s) { return smem_base + s * S::kStage; };
    auto v_smem = [&](int s) { return smem_base + (kStages + s) * S::kStage; };
    const uint32_t bar_base = smem_base + S::kBarOffset;
    const uint32_t a_ready = bar_base, a_full = bar_base + 96, acc_full = bar_base + 8, s_full = bar_base + 16 /* per group */, dp_full = bar_base + 32, ds_ready = bar_base + 48, s_free = bar_base + 64, staged = bar_base + 80,
                   full = bar_base + 128, empty = full + 8 * kStages;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_gen + S::kBarOffset + 120);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    BiasShared& bias = *reinterpret_cast<BiasShared*>(smem_gen + S::kBiasOffset);

    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const WorkItem work = p.order_dq(item);
    const int bh = work.unit, qt = p.h.causal ? p.q_tiles - 1 - work.tile : work.tile;
    const int b = p.by_heads(bh), h = bh - b * p.h.heads, hk = p.by_group(h);
    const int row0 = qt * kTile;
    const int n_keys = heads_key_count(p.h, b), offset = heads_offset(p.h, n_keys);
    const int key_end = p.h.causal ? max(0, min(n_keys, min(row0 + kTile, p.h.seq_q) + offset)) : n_keys;
    const int n_it = (key_end + kHalf - 1) / kHalf;
    const WaitCtx wctx{abort_flag, p.status, p.wait_limit_ns};

    auto load_stage = [&](int s, int it) {
        ptx::mbar_arrive_expect_tx(full + 8 * s, 2 * S::kStage);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            ptx::tma_load_4d(k_smem(s) + c * Mma::kPiece, &map_k, full + 8 * s, c * 64, it * kHalf, hk * p.k_at.head, b * p.k_at.batch);
            ptx::tma_load_4d(v_smem(s) + c * Mma::kPiece, &map_v, full + 8 * s, c * 64, it * kHalf, hk * p.v_at.head, b * p.v_at.batch);
        }
    };
    if (threadIdx.x == 0) {
        ptx::mbar_init(a_ready, 8); ptx::mbar_init(a_full, 1); ptx::mbar_init(acc_full, 1); ptx::mbar_init(staged, 8);
        for (int x = 0; x < 2; ++x) {
            ptx::mbar_init(s_full + 8 * x, 1); ptx::mbar_init(dp_full + 8 * x, 1); ptx::mbar_init(ds_ready + 8 * x, 4); ptx::mbar_init(s_free + 8 * x, 4);
        }
        for (int s = 0; s < kStages; ++s) {
            ptx::mbar_init(full + 8 * s, 1); ptx::mbar_init(empty + 8 * s, 1);
        }
        *abort_flag = 0;
        ptx::mbar_fence_init();
        if (n_it > 0) {                                         // these fly while the CTA sets itself up; Q and dO where the last two stages will be
            ptx::mbar_arrive_expect_tx(a_full, 4 * S::kStage);
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
#pragma unroll
                for (int r = 0; r < kTile; r += kHalf) {
                    ptx::tma_load_4d(k_smem(kStages - 2) + c * (kTile * 128) + r * 128, &m.q, a_full, c * 64, row0 + r, h * p.q_at.head, b * p.q_at.batch);
                    ptx::tma_load_4d(v_smem(kStages - 2) + c * (kTile * 128) + r * 128, &m.d_o, a_full, c * 64, row0 + r, h * p.do_at.head, b * p.do_at.batch);
                }
            load_stage(0, 0);
        }
    }
    const int x = (warp - 2) >> 2;                              // group of the warps 2 to 9
    const int row = row0 + (warp & 3) * 32 + lane;
    // loads from here to the barrier are in flight together
    float nlse = 0.0f, ndelta = 0.0f, do_norm = 0.0f, v_norm = 0.0f, run_bias = 0.0f;
    if (BIAS && (int)threadIdx.x < p.h.n_runs) run_bias = heads_run_bias(p.h, threadIdx.x, h);
    if (warp >= 2) {
        const int64_t at_row = (int64_t)bh * p.g.pad_q + row;
        nlse = p.g.lse2[at_row];
        ndelta = p.g.delta[at_row];
        if (!BF16) {
            do_norm = __ldg(p.g.amax + b * p.h.kv_heads + hk);
            v_norm = __ldg(p.g.amax + (int64_t)p.h.batch * p.h.kv_heads + b * p.h.kv_heads + hk);
        }
    }
    if constexpr (BIAS) {
        load_runs(bias, p.h, warp, kBwdThreads / 32, lane);
        if ((int)threadIdx.x < p.h.n_runs) bias.value[threadIdx.x] = run_bias;
    }
    if (warp == 1) {
        ptx::tmem_alloc(ptx::smem_u32(tmem_slot), 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        // ---- TMA producer ------------------------------------------------------------------------------
        if (lane == 0) {
            int s = 1;
            uint32_t phase = 1;
            for (int it = 1; it < n_it; ++it) {
                if (it == kStages - 2 && !bounded_wait(wctx, a_ready, 0, 0x06010000u)) break;          // Q and dO have left the last stages
                if (!bounded_wait(wctx, empty + 8 * s, phase, 0x06010000u | (it & 0xffff))) break;
                load_stage(s, it);
                if (++s == kStages) { s = 0; phase ^= 1; }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---- MMA issuer: S(0) dP(0) S(1) dP(1) | S(i+2) dQ(i) dP(i+2) | ... ------------------------------------------
        if (n_it > 0) {
            const uint32_t lead = ptx::elect_lead();
            const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
            const int tiles = __shfl_sync(0xffffffffu, n_it, 0);
            auto s_product = [&](int it, int s) {
                Mma::scores_ts(lead, tmem + kColS + 64 * (it & 1), tmem + kColQ, k_smem(s));
                ptx::mma_commit_lead(lead, s_full + 8 * (it & 1));
            };
            auto dp_product = [&](int it, int s) {
                Mma::scores_ts(lead, tmem + kColDP + 64 * (it & 1), tmem + kColDO, v_smem(s));
                ptx::mma_commit_lead(lead, dp_full + 8 * (it & 1));
            };
            bool ok = warp_spin(wctx, a_ready, 0, 0x06030000u);
            for (int it = 0; it < 2 && it < tiles && ok; ++it) {
                if (!(ok = warp_spin(wctx, full + 8 * it, 0, 0x06040000u | it))) break;
                ptx::tc_fence_after_sync();
                s_product(it, it);
                dp_product(it, it);
            }
            int s = 0, next = 2;                                // stages of tiles it and it + 2
            uint32_t next_phase = 0;
            for (int it = 0; it < tiles && ok; ++it) {
                const uint32_t phase = (it >> 1) & 1;
                const bool more = it + 2 < tiles;
                if (more) {
                    if (!(ok = warp_spin(wctx, full + 8 * next, next_phase, 0x06050000u | (it & 0xffff)))) break;
                    // S(it) is in registers: its columns are free
                    if (!(ok = warp_spin(wctx, s_free + 8 * (it & 1), phase, 0x06060000u | (it & 0xffff)))) break;
                    ptx::tc_fence_after_sync();
                    s_product(it + 2, next);
                }
                if (!(ok = warp_spin(wctx, ds_ready + 8 * (it & 1), phase, 0x06070000u | (it & 0xffff)))) break;
                ptx::tc_fence_after_sync();
                Mma::grads(lead, tmem + kColDQ, tmem + kColDP + 64 * (it & 1), k_smem(s), it == 0);
                ptx::mma_commit_lead(lead, empty + 8 * s);
                if (more) dp_product(it + 2, next);
                if (++s == kStages) s = 0;
                if (++next == kStages) { next = 0; next_phase ^= 1; }
            }
            if (ok) ptx::mma_commit_lead(lead, acc_full);
        }
        __syncwarp();
    } else {
        // ---- probabilities and their gradients: rows are queries, columns keys; group x takes tiles x, x + 2, ... --------
        const int w = warp - 2, quarter = warp & 3;
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        const uint32_t s_at = tmem_base + lane_base + kColS + x * 64, dp_at = tmem_base + lane_base + kColDP + x * 64;
        bool ok = true;
        if (n_it > 0 && (ok = warp_wait(wctx, a_full, 0, 0x06020000u))) {        // group 0 writes Q to tensor memory, group 1 dO
            row_to_tmem<D / 32>(tmem_base + lane_base + (x ? kColDO : kColQ), x ? v_smem(kStages - 2) : k_smem(kStages - 2), quarter * 32 + lane);
            ptx::tmem_st_wait();
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(a_ready);
        }
        const float g_scale = BF16 ? 1.0f : ds_scale(do_norm, v_norm);
        const float2 nd2 = make_float2(ndelta, ndelta), g2 = make_float2(g_scale, g_scale);
        const int sees = p.h.causal ? min(n_keys, row + offset + 1) : n_keys;
        const bool want_bias = BIAS && p.g.dtable != nullptr;
        float* sums = reinterpret_cast<float*>(smem_gen + S::kSumsOffset) + w * kHeadsMaxRuns;      // this warp's, by run
        RunSums rs{0.0f, 0};
        WarpBias wb(p.h);
        if constexpr (BIAS) {
            for (int r = lane; r < p.h.n_runs; r += 32) sums[r] = 0.0f;
            __syncwarp();
        }
        int s = x;                                              // the tile's stage
        for (int it = x; it < n_it && ok; it += 2) {
            const uint32_t phase = (it >> 1) & 1;
            const int key0 = it * kHalf;
            const int d0 = key0 - (row0 + quarter * 32 + 31 + offset);
            float c = p.h.scale_log2, add = nlse;
            bool looked_up = false;
            if constexpr (BIAS) looked_up = !wb.block(bias, bias.value, w, lane, p.h.n_runs, d0);
            ok = warp_wait(wctx, s_full + 8 * x, phase, 0x06080000u | (it & 0xffff));
            if (!ok) break;
            ptx::tc_fence_after_sync();
            const int valid = sees - key0;                      // columns that are seen
            const bool masked = __any_sync(0xffffffffu, valid < 64);
            float2 e[32];
            uint32_t r[64];
            ptx::tmem_ld_32x32b_x32(s_at, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
            ptx::tmem_ld_32x32b_x32(s_at + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
            ptx::tmem_ld_wait();
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(s_free + 8 * x);
            if constexpr (BIAS) {
                if (looked_up) {
                    const float* at = bias.by_dist[w] + 31 - lane;
#pragma unroll
                    for (int i = 0; i < 64; ++i) r[i] = __float_as_uint(fmaf(__uint_as_float(r[i]), c, at[i]));
                    c = 1.0f;
                } else {
                    add += wb.same;
                }
            }
            const float2 c2 = make_float2(c, c), a2 = make_float2(add, add);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const float2 y = fma2(f2(r[2 * i], r[2 * i + 1]), c2, a2);
                e[i] = make_float2(ptx::ex2_approx(y.x), ptx::ex2_approx(y.y));
            }
            // K rows behind the key count hold whatever the caller left there: cleared before dQ's product multiplies them by dS's zeros
            const int live = n_keys - key0;
            if (live < kHalf && n_keys < p.h.seq_k) {           // S has been computed from them; its columns there are not used
                for (int k = live * 8 + (quarter * 32 + lane); k < kHalf * 8; k += 128)
#pragma unroll
                    for (int ch = 0; ch < kChunks; ++ch)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(k_smem(s) + ch * Mma::kPiece + k * 16), "r"(0) : "memory");
                ptx::fence_proxy_async_smem();
            }
            ok = warp_wait(wctx, dp_full + 8 * x, phase, 0x06090000u | (it & 0xffff));
            if (!ok) break;
            ptx::tc_fence_after_sync();
            ptx::tmem_ld_32x32b_x32(dp_at, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
            ptx::tmem_ld_32x32b_x32(dp_at + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
            ptx::tmem_ld_wait();
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
                uint32_t pk[16];
#pragma unroll
                for (int i = ch * 16; i < ch * 16 + 16; ++i) {
                    float2 ds = mul2(e[i], add2(f2(r[2 * i], r[2 * i + 1]), nd2));
                    if (masked) {
                        if (2 * i >= valid) ds.x = 0.0f;
                        if (2 * i + 1 >= valid) ds.y = 0.0f;
                    }
                    pk[i - ch * 16] = rounded_pair<BF16>(BF16 ? ds : mul2(ds, g2));
                    if constexpr (BIAS) {
                        r[2 * i] = __float_as_uint(ds.x);
                        r[2 * i + 1] = __float_as_uint(ds.y);
                    }
                }
                ptx::tmem_st_32x32b_x16(dp_at + ch * 16, pk);
            }
            ptx::tmem_st_wait();
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(ds_ready + 8 * x);
            if constexpr (BIAS) {
                if (want_bias) {
                    if (looked_up) {
                        const float go_on = lane == 0 ? 0.0f : 1.0f;
#pragma unroll
                        for (int i = 1; i < 16; ++i)
#pragma unroll
                            for (int chain = 0; chain < 64; chain += 16) {
                                const float below = __shfl_up_sync(0xffffffffu, __uint_as_float(r[chain + i - 1]), 1);
                                r[chain + i] = __float_as_uint(fmaf(below, go_on, __uint_as_float(r[chain + i])));
                            }
                        float* by_diag = bias.by_dist[w];                   // the biases have been read
                        if (lane == 31) {
#pragma unroll
                            for (int i = 0; i < 64; i += 4) *reinterpret_cast<uint4*>(by_diag + i) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
                        }
                        __syncwarp();
                        // lane l takes diagonals l, 32 + l, 64 + l; what lane k was left with by chain c belongs to diagonal 16 c + 46 - k
                        // (lane 31's is complete)
                        auto rest = [&](int chain, int t) {
                            const int from = 16 * chain + 46 - t;
                            const float v = __shfl_sync(0xffffffffu, __uint_as_float(r[16 * chain + 15]), from & 31);
                            return from >= 0 && from < 31 ? v : 0.0f;
                        };
                        float d3[3] = {by_diag[lane] + rest(0, lane),
                                       by_diag[32 + lane] + ((rest(0, 32 + lane) + rest(1, 32 + lane)) + rest(2, 32 + lane)),
                                       rest(2, 64 + lane) + rest(3, 64 + lane)};
                        // each run's sum by a scan that stops at the run's first diagonal, 32 diagonals at a time
                        int run[3], start[3];
#pragma unroll
                        for (int k = 0; k < 3; ++k) {
                            run[k] = wb.run_of(bias, p.h.n_runs, d0 + 32 * k + lane);
                            start[k] = run[k] == 0 ? 0 : max(0, bias.first[run[k]] - d0 - 32 * k);
                        }
#pragma unroll
                        for (int off = 1; off < 32; off <<= 1)
#pragma unroll
                            for (int k = 0; k < 3; ++k) {
                                const float v = __shfl_up_sync(0xffffffffu, d3[k], off);
                                if (lane - off >= start[k]) d3[k] += v;
                            }
#pragma unroll
                        for (int k = 0; k < 3; ++k) {
                            const int next = __shfl_down_sync(0xffffffffu, run[k], 1);
                            if (lane == 31 || next != run[k]) sums[run[k]] += d3[k];
                            __syncwarp();
                        }
                        __syncwarp();
                    } else {
                        if (rs.run != wb.run) {
                            rs.flush(sums, lane);
                            __syncwarp();
                            rs.run = wb.run;
                        }
                        float2 part[4] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                        for (int i = 0; i < 32; ++i) part[i & 3] = add2(part[i & 3], f2(r[2 * i], r[2 * i + 1]));
                        const float2 sum = add2(add2(part[0], part[1]), add2(part[2], part[3]));
                        rs.acc += sum.x + sum.y;
                    }
                }
            }
            s += 2;
            if (s >= kStages) s -= kStages;
        }
        if (ok && n_it > 0) ok = warp_wait(wctx, acc_full, 0, 0x060a0000u);
        if (ok) {
            ptx::tc_fence_after_sync();
            const float out = BF16 ? 1.0f / kCutScale : 1.0f / ((1 << kF16Shift) * g_scale);
            const float f = p.h.scale * out;
#pragma unroll 1
            for (int ch = 0; ch < D / 64; ++ch) {               // every load has been used: the tile is staged where the operands were
                uint32_t r[32], v[16];
                if (n_it > 0) {
                    ptx::tmem_ld_32x32b_x32(tmem_base + lane_base + kColDQ + x * (D / 2) + ch * 32, r);
                    ptx::tmem_ld_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) r[i] = 0;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = round_pair<BF16>(__uint_as_float(r[2 * i]) * f, __uint_as_float(r[2 * i + 1]) * f);
                stage_row(smem_base, quarter * 32 + lane, x * (D / 2) + ch * 32, v);
            }
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(staged);
            if (w == 0 && lane == 0 && bounded_wait(wctx, staged, 0, 0x060b0000u)) {
#pragma unroll
                for (int c = 0; c < kChunks; ++c)               // rows behind seq_q are dropped
                    ptx::tma_store_4d(&map_dq, smem_base + c * (kTile * 128), c * 64, row0, h * p.dq_at.head, b * p.dq_at.batch);
                ptx::tma_store_commit();
                ptx::tma_store_wait_read<0>();     // shared memory has been read; the grid's end covers the writes
            }
            __syncwarp();
            if constexpr (BIAS) {
                if (want_bias) {
                    rs.flush(sums, lane);
                    __syncwarp();
                    const float back = BF16 ? 1.0f / kCutScale : 1.0f / (1 << kF16Shift);
                    for (int r = lane; r < p.h.n_runs; r += 32)
                        p.g.run_sums[((int64_t)bh * p.g.q_tiles + qt * 8 + w) * p.h.n_runs + r] = sums[r] * back;
                }
            }
        }
    }

    if (*abort_flag) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem_base, 512);
    }
}

// Both in one launch: the dq blocks fill the SMs that the last dkv blocks leave idle.
template <int D, bool BF16, bool BIAS>
__global__ void __launch_bounds__(kBwdThreads, 1) heads_bwd_kernel(const __grid_constant__ BwdMaps m, const __grid_constant__ BwdParams p) {
    if ((int)blockIdx.x < p.dkv_blocks) dkv_block<D, BF16, BIAS>(m, p, blockIdx.x);
    else dq_block<D, BF16, BIAS>(m, p, blockIdx.x - p.dkv_blocks);
}

template <int D, bool BF16>
static int launch_bwd(BwdParams& p, cudaStream_t s) {
    const HeadsParams& h = p.h;
    BwdMaps m;
    int rc = make_map(&m.q, &p.q_at, p.g.q, h.batch, h.heads, h.seq_q, D, h.q_s, kHalf, 1);
    if (rc == EMMYB200_OK) rc = make_map(&m.d_o, &p.do_at, p.g.d_o, h.batch, h.heads, h.seq_q, D, h.do_s, kHalf, 1);
    if (rc == EMMYB200_OK) rc = make_map(&m.k, &p.k_at, p.g.k, h.batch, h.kv_heads, h.seq_k, D, h.k_s, kHalf, 1);
    if (rc == EMMYB200_OK) rc = make_map(&m.v, &p.v_at, p.g.v, h.batch, h.kv_heads, h.seq_k, D, h.v_s, kHalf, 1);
    if (rc == EMMYB200_OK) rc = make_map(&m.k_tile, &p.k_at, p.g.k, h.batch, h.kv_heads, h.seq_k, D, h.k_s, kTile, 1);
    if (rc == EMMYB200_OK) rc = make_map(&m.v_tile, &p.v_at, p.g.v, h.batch, h.kv_heads, h.seq_k, D, h.v_s, kTile, 1);
    if (rc == EMMYB200_OK) rc = make_map(&m.dq, &p.dq_at, p.g.dq, h.batch, h.heads, h.seq_q, D, h.dq_s, kTile, 1);
    if (rc == EMMYB200_OK) rc = make_map(&m.dk, &p.dk_at, p.g.dk, h.batch, h.kv_heads, h.seq_k, D, h.dk_s, kTile, 1);
    if (rc == EMMYB200_OK) rc = make_map(&m.dv, &p.dv_at, p.g.dv, h.batch, h.kv_heads, h.seq_k, D, h.dv_s, kTile, 1);
    if (rc != EMMYB200_OK) return rc;
    EMMY_CUDA(cudaGetSymbolAddress(reinterpret_cast<void**>(&p.status), g_bwd_status));
    const int64_t kv_ctas = (int64_t)h.batch * h.kv_heads * p.k_tiles, q_ctas = (int64_t)h.batch * h.heads * p.q_tiles;
    if (kv_ctas + q_ctas >= (1ll << 31)) return fail(EMMYB200_ERR_SHAPE, "attention_heads_bwd: the tiles exceed the grid limit");
    p.dkv_blocks = (int)kv_ctas;
    p.order_dkv = work_order(h.causal != 0, (int64_t)h.batch * h.kv_heads, p.k_tiles, (int64_t)h.seq_q * D * 4 * h.group);
    p.order_dq = work_order(h.causal != 0, (int64_t)h.batch * h.heads, p.q_tiles, (int64_t)h.seq_k * D * 4 / h.group);
    p.by_heads = fast_div(h.heads);
    p.by_kv_heads = fast_div(h.kv_heads);
    p.by_group = fast_div(h.group);
    auto kernel = h.n_runs ? heads_bwd_kernel<D, BF16, true> : heads_bwd_kernel<D, BF16, false>;
    EMMY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BwdSmem<D>::kTotal));
    kernel<<<(unsigned)(kv_ctas + q_ctas), kBwdThreads, BwdSmem<D>::kTotal, s>>>(m, p);
    return launch_status("heads_bwd_kernel");
}

}  // namespace heads

bool heads_bwd_sm100_takes(const HeadsParams& p, int dtype, int d, const HeadsGrads& g) {
    using namespace heads;
    return heads_sm100_takes(p, dtype, d, g.q, g.k, g.v, g.o) && map_fits(g.d_o, p.batch, p.heads, p.seq_q, p.do_s) &&
           map_fits(g.dq, p.batch, p.heads, p.seq_q, p.dq_s) && map_fits(g.dk, p.batch, p.kv_heads, p.seq_k, p.dk_s) &&
           map_fits(g.dv, p.batch, p.kv_heads, p.seq_k, p.dv_s);
}

float heads_bwd_shift(int dtype) { return dtype == EMMYB200_BF16 ? heads::kCutScaleLog2 : (float)heads::kF16Shift; }

int heads_bwd_sm100(int dtype, int d, const HeadsParams& hp, const HeadsGrads& g, cudaStream_t s) {
    heads::BwdParams p = {};
    p.h = hp;
    p.g = g;
    p.q_tiles = (hp.seq_q + heads::kTile - 1) / heads::kTile;
    p.k_tiles = (hp.seq_k + heads::kTile - 1) / heads::kTile;
    p.wait_limit_ns = wait_limit_ns();
    const bool bf16 = dtype == EMMYB200_BF16;
    if (d == 128) return bf16 ? heads::launch_bwd<128, true>(p, s) : heads::launch_bwd<128, false>(p, s);
    return bf16 ? heads::launch_bwd<64, true>(p, s) : heads::launch_bwd<64, false>(p, s);
}

int heads_bwd_read_status(uint32_t* out) {
    uint32_t zero = 0;
    EMMY_CUDA(cudaDeviceSynchronize());
    EMMY_CUDA(cudaMemcpyFromSymbol(out, heads::g_bwd_status, sizeof(uint32_t)));
    if (*out) EMMY_CUDA(cudaMemcpyToSymbol(heads::g_bwd_status, &zero, sizeof(uint32_t)));
    return EMMYB200_OK;
}

}  // namespace emmy
