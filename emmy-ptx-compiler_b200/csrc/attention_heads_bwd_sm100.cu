// Attention over heads, backward, on the tensor cores: f16 / bf16, d = 64 or 128.
//
// With P_ij = exp(s_ij - lse_i) and dS_ij = P_ij (dO_i . v_j - D_i), D_i = dO_i . O_i, the gradients are five products per
// 128 x 128 tile. Two kernels recompute P, each writing what its CTAs own, so nothing is accumulated across CTAs and results
// are the same every time; the two score-sized products are done in both, seven in all where one kernel with atomic
// additions into dQ would do five:
//
//   heads_dkv_kernel   a CTA owns 128 keys of a key head and walks the query tiles of every query head that reads it.
//                      Everything is transposed, keys are rows: S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q, with P^T
//                      and dS^T as tensor-memory operands. 4 x 128 columns: S^T (P^T over it), dP^T (dS^T over it), dV, dK.
//   heads_dq_kernel    a CTA owns 128 queries and walks the keys: S = Q K^T (two buffers, dS over them), dP = dO V^T,
//                      dQ += dS K.
//
// One CTA per SM, 320 threads: warp 0 TMA (two-stage rings), warp 1 issues the products, warps 2-9 do the arithmetic between
// them: two threads per row, 64 columns apiece, no exchange at all, since the row terms are known beforehand. A product's
// operand (P, dS) goes back to tensor memory in two blocks of 64 columns, each over the columns its own thread has read.
// The order of the products keeps the tensor pipe busy while the exponentials are taken: dV(i) S(i+1) dK(i) dP(i+1), and
// dP(i+1) dQ(i) S(i+2).
//
// Row terms come from the rows kernel already negated and shifted: nlse2 = -lse log2(e) + shift, -inf for rows that see
// nothing or lie behind seq_q, so that P = 2^(scale log2(e) q.k + bias + nlse2) needs no test. The shift scales P by what the
// rounding to 16 bits wants: 1 + delta before bf16 values are cut (kCutScale), 2^14 for f16, whose small probabilities would
// lose bits. dS inherits the factor and, in f16, a power of two per key head on top, chosen from the largest row norms of dO and V so that
// |dS| stays below 2^15: a tiny or huge incoming gradient keeps its bits. All factors but the cut's are exact and taken out at the end.
#include <math_constants.h>

#include "attention_heads_sm100.cuh"

namespace emmy {
namespace heads {

constexpr int kBwdThreads = 320;
constexpr int kF16Shift = 14;

struct BwdParams {
    HeadsParams h;
    HeadsGrads g;
    MapAt q_at, k_at, v_at, do_at;
    int q_tiles, k_tiles;
    unsigned long long wait_limit_ns;
    uint32_t* status;
};

__device__ uint32_t g_bwd_status;

template <int D>
struct BwdSmem {
    static constexpr int kOperand = kTile * D * 2;
    static constexpr int kRowsOffset = 6 * kOperand;                    // [2 stages][nlse2 128, ndelta 128]
    static constexpr int kBarOffset = kRowsOffset + 2048;
    static constexpr int kBiasOffset = kBarOffset + 256;
    static constexpr int kSumsOffset = kBiasOffset + (int)sizeof(BiasShared);
    static constexpr int kTotal = kSumsOffset + 8 * kHeadsMaxRuns * 4 + 1024;
};

// The power of two dS is scaled by in f16: |dS| 2^14 g <= 2^15 from |dO . v - D| <= 2 max|dO| max|v|. 1 in bf16.
template <bool BF16>
__device__ __forceinline__ float ds_scale(const HeadsGrads& g, int64_t bk, int64_t all) {
    if constexpr (BF16) return 1.0f;
    const float bound = sqrtf(g.amax[bk]) * sqrtf(g.amax[all + bk]);
    if (!(bound > 0.0f) || !(bound < CUDART_INF_F)) return 1.0f;
    return __int_as_float(((int)fminf(fmaxf(floorf(-log2f(bound)), -100.0f), 100.0f) + 127) << 23);
}

// Tensor-memory column of k-step kk (16 columns of a 128-column operand) inside its region: the two halves are 64 apart.
__device__ __forceinline__ uint32_t operand_col(int kk) { return kk < 4 ? kk * 8 : 64 + (kk - 4) * 8; }

template <int D, bool BF16, bool BIAS>
__global__ void __launch_bounds__(kBwdThreads, 1)
heads_dkv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                 const __grid_constant__ CUtensorMap map_do, const __grid_constant__ BwdParams p) {
    using S = BwdSmem<D>;
    constexpr int kChunks = D / 64;
    constexpr uint32_t kColS = 0, kColDP = 128, kColDV = 256, kColDK = 384;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));
    const uint32_t k_smem = smem_base, v_smem = smem_base + S::kOperand;
    auto q_smem = [&](int s) { return smem_base + (2 + s) * S::kOperand; };
    auto do_smem = [&](int s) { return smem_base + (4 + s) * S::kOperand; };
    const uint32_t rows_smem = smem_base + S::kRowsOffset;
    const uint32_t bar_base = smem_base + S::kBarOffset;
    const uint32_t kv_full = bar_base, s_full = bar_base + 8, dp_full = bar_base + 16, p_ready = bar_base + 24, ds_ready = bar_base + 32,
                   acc_full = bar_base + 40, q_full = bar_base + 48, q_empty = bar_base + 64, do_full = bar_base + 80, do_empty = bar_base + 96;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_gen + S::kBarOffset + 128);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    BiasShared& bias = *reinterpret_cast<BiasShared*>(smem_gen + S::kBiasOffset);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kt = blockIdx.x % p.k_tiles, bk = blockIdx.x / p.k_tiles;         // causal: the first key tiles see the most queries
    const int b = bk / p.h.kv_heads, hk = bk % p.h.kv_heads;
    const int key0 = kt * kTile;
    const int n_keys = heads_key_count(p.h, b), offset = heads_offset(p.h, n_keys);
    const int first_qt = p.h.causal ? max(0, key0 - offset) / kTile : 0;       // queries before it see none of these keys
    const int per_head = key0 < n_keys ? max(0, p.q_tiles - first_qt) : 0;
    const int n_it = per_head * p.h.group;
    const WaitCtx wctx{abort_flag, p.status, p.wait_limit_ns};

    if (threadIdx.x == 0) {
        ptx::mbar_init(kv_full, 1); ptx::mbar_init(s_full, 1); ptx::mbar_init(dp_full, 1);
        ptx::mbar_init(p_ready, 8); ptx::mbar_init(ds_ready, 8); ptx::mbar_init(acc_full, 1);
        for (int s = 0; s < 2; ++s) {
            ptx::mbar_init(q_full + 8 * s, 1); ptx::mbar_init(q_empty + 8 * s, 1);
            ptx::mbar_init(do_full + 8 * s, 1); ptx::mbar_init(do_empty + 8 * s, 1);
        }
        *abort_flag = 0;
        ptx::mbar_fence_init();
        ptx::prefetch_tensormap(&map_q); ptx::prefetch_tensormap(&map_k); ptx::prefetch_tensormap(&map_v); ptx::prefetch_tensormap(&map_do);
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
        if (lane == 0 && n_it > 0) {
            ptx::mbar_arrive_expect_tx(kv_full, 2 * S::kOperand);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                ptx::tma_load_4d(k_smem + c * (kTile * 128), &map_k, kv_full, c * 64, key0, hk * p.k_at.head, b * p.k_at.batch);
                ptx::tma_load_4d(v_smem + c * (kTile * 128), &map_v, kv_full, c * 64, key0, hk * p.v_at.head, b * p.v_at.batch);
            }
            for (int it = 0; it < n_it; ++it) {
                const int s = it & 1, h = hk * p.h.group + it / per_head, row0 = (first_qt + it % per_head) * kTile;
                const uint32_t empty = ((it >> 1) & 1) ^ 1;
                if (!bounded_wait(wctx, q_empty + 8 * s, empty, 0x05010000u | (it & 0xffff))) break;
                ptx::mbar_arrive_expect_tx(q_full + 8 * s, S::kOperand + 1024);
#pragma unroll
                for (int c = 0; c < kChunks; ++c)
                    ptx::tma_load_4d(q_smem(s) + c * (kTile * 128), &map_q, q_full + 8 * s, c * 64, row0, h * p.q_at.head, b * p.q_at.batch);
                const int64_t at = ((int64_t)b * p.h.heads + h) * p.g.pad_q + row0;
                ptx::bulk_load(rows_smem + s * 1024, p.g.lse2 + at, 512, q_full + 8 * s);
                ptx::bulk_load(rows_smem + s * 1024 + 512, p.g.delta + at, 512, q_full + 8 * s);
                if (!bounded_wait(wctx, do_empty + 8 * s, empty, 0x05020000u | (it & 0xffff))) break;
                ptx::mbar_arrive_expect_tx(do_full + 8 * s, S::kOperand);
#pragma unroll
                for (int c = 0; c < kChunks; ++c)
                    ptx::tma_load_4d(do_smem(s) + c * (kTile * 128), &map_do, do_full + 8 * s, c * 64, row0, h * p.do_at.head, b * p.do_at.batch);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---- MMA issuer ----------------------------------------------------------------------------------
        if (lane == 0 && n_it > 0) {
            constexpr uint32_t idesc_s = ptx::mma_idesc_f16(BF16, false, false, kTile, kTile);
            constexpr uint32_t idesc_d = ptx::mma_idesc_f16(BF16, false, true, kTile, D);
            // rows of `a` times rows of `b`, contraction over the head dim
            auto scores = [&](uint32_t col, uint32_t a, uint32_t bb) {
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint32_t off = (kk / 4) * (kTile * 128) + (kk % 4) * 32;
                    ptx::mma_ss(tmem_base + col, ptx::smem_desc_sw128(a + off, 16, 1024), ptx::smem_desc_sw128(bb + off, 16, 1024), idesc_s, kk != 0);
                }
            };
            // accumulator += operand in tensor memory times the rows of `bb`, contraction over those rows
            auto grads = [&](uint32_t col, uint32_t a_col, uint32_t bb, bool first) {
#pragma unroll
                for (int kk = 0; kk < kTile / 16; ++kk)
                    ptx::mma_ts(tmem_base + col, tmem_base + a_col + operand_col(kk), ptx::smem_desc_sw128(bb + kk * (16 * 128), kTile * 128, 1024), idesc_d,
                                !first || kk != 0);
            };
            bool ok = bounded_spin(wctx, kv_full, 0, 0x05030000u) && bounded_spin(wctx, q_full, 0, 0x05040000u);
            if (ok) {
                ptx::tc_fence_after_sync();
                scores(kColS, k_smem, q_smem(0));
                ptx::mma_commit(s_full);
                ok = bounded_spin(wctx, do_full, 0, 0x05050000u);
            }
            if (ok) {
                ptx::tc_fence_after_sync();
                scores(kColDP, v_smem, do_smem(0));
                ptx::mma_commit(dp_full);
            }
            for (int it = 0; it < n_it && ok; ++it) {
                const int s = it & 1;
                const uint32_t next = ((it + 1) >> 1) & 1;
                if (!(ok = bounded_spin(wctx, p_ready, it & 1, 0x05060000u | (it & 0xffff)))) break;
                ptx::tc_fence_after_sync();
                grads(kColDV, kColS, do_smem(s), it == 0);
                ptx::mma_commit(do_empty + 8 * s);
                if (it + 1 < n_it) {
                    if (!(ok = bounded_spin(wctx, q_full + 8 * (s ^ 1), next, 0x05070000u | (it & 0xffff)))) break;
                    ptx::tc_fence_after_sync();
                    scores(kColS, k_smem, q_smem(s ^ 1));
                    ptx::mma_commit(s_full);
                }
                if (!(ok = bounded_spin(wctx, ds_ready, it & 1, 0x05080000u | (it & 0xffff)))) break;
                ptx::tc_fence_after_sync();
                grads(kColDK, kColDP, q_smem(s), it == 0);
                ptx::mma_commit(q_empty + 8 * s);
                if (it + 1 < n_it) {
                    if (!(ok = bounded_spin(wctx, do_full + 8 * (s ^ 1), next, 0x05090000u | (it & 0xffff)))) break;
                    ptx::tc_fence_after_sync();
                    scores(kColDP, v_smem, do_smem(s ^ 1));
                    ptx::mma_commit(dp_full);
                }
            }
            if (ok) ptx::mma_commit(acc_full);
        }
        __syncwarp();
    } else {
        // ---- probabilities and their gradients: rows are keys, columns queries ---------------------------------------
        const int w = warp - 2, quarter = warp & 3, half = w >> 2;
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        const uint32_t s_at = tmem_base + lane_base + kColS + half * 64, dp_at = tmem_base + lane_base + kColDP + half * 64;
        const int key = key0 + quarter * 32 + lane;
        const float g_scale = ds_scale<BF16>(p.g, bk, (int64_t)p.h.batch * p.h.kv_heads);
        const float2 g2 = make_float2(g_scale, g_scale);
        bool ok = true;
        WarpBias wb;
        int bias_head = -1;
        for (int it = 0; it < n_it && ok; ++it) {
            const int s = it & 1;
            const int q0 = (first_qt + it % per_head) * kTile + half * 64;      // this thread's first query
            float c = p.h.scale_log2, add = 0.0f;
            bool looked_up = false;
            if constexpr (BIAS) {
                // the table's column changes with the query head; every warp keeps a copy of its own, so that no two warps have to meet
                const int h = hk * p.h.group + it / per_head;
                if (h != bias_head) {
                    bias_head = h;
                    __syncwarp();
                    float* value = reinterpret_cast<float*>(smem_gen + S::kSumsOffset) + w * kHeadsMaxRuns;
                    for (int r = lane; r < p.h.n_runs; r += 32) {
                        if (it == 0) bias.first[r] = p.h.run_first[r];          // every warp writes the same
                        value[r] = heads_run_bias(p.h, r, h);
                    }
                    __syncwarp();
                    wb.reset();
                }
                looked_up = !wb.block(bias, reinterpret_cast<float*>(smem_gen + S::kSumsOffset) + w * kHeadsMaxRuns, w, lane, p.h.n_runs,
                                      key0 + quarter * 32 - (q0 + 63 + offset));
                add = wb.same;
            }
            ok = __all_sync(0xffffffffu, bounded_wait(wctx, q_full + 8 * s, (it >> 1) & 1, 0x050a0000u | (it & 0xffff)) &&
                                             bounded_wait(wctx, s_full, it & 1, 0x050b0000u | (it & 0xffff)));
            if (!ok) break;
            ptx::tc_fence_after_sync();
            const float4* nlse = reinterpret_cast<const float4*>(smem_gen + S::kRowsOffset + s * 1024 + half * 256);
            const float4* ndelta = nlse + 32;
            // columns below `hidden` are not seen: queries before the key, or the whole row for keys behind the count
            const int hidden = key >= n_keys ? 64 : (p.h.causal ? key - offset - q0 : 0);
            const bool masked = __any_sync(0xffffffffu, hidden > 0);
            float2 e[32];
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
                uint32_t r[32];
                ptx::tmem_ld_32x32b_x32(s_at + ch * 32, r);
                ptx::tmem_ld_wait();
                if constexpr (BIAS) {
                    if (looked_up) {
                        const float* at = bias.by_dist[w] + 63 + lane - ch * 32;
#pragma unroll
                        for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(fmaf(__uint_as_float(r[i]), c, at[-i]));
                    }
                }
                const float cc = BIAS && looked_up ? 1.0f : c, aa = BIAS && looked_up ? 0.0f : add;
                const float2 c2 = make_float2(cc, cc), a2 = make_float2(aa, aa);
                uint32_t pk[16];
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    float4 nl = nlse[ch * 8 + i / 2];
                    float2 n0 = make_float2(nl.x, nl.y), n1 = make_float2(nl.z, nl.w);
                    if constexpr (BIAS) { n0 = add2(n0, a2); n1 = add2(n1, a2); }
                    const float2 y0 = fma2(f2(r[2 * i], r[2 * i + 1]), c2, n0), y1 = fma2(f2(r[2 * i + 2], r[2 * i + 3]), c2, n1);
                    e[ch * 16 + i] = make_float2(ptx::ex2_approx(y0.x), ptx::ex2_approx(y0.y));
                    e[ch * 16 + i + 1] = make_float2(ptx::ex2_approx(y1.x), ptx::ex2_approx(y1.y));
                }
                if (masked) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        if (ch * 32 + 2 * i < hidden) e[ch * 16 + i].x = 0.0f;
                        if (ch * 32 + 2 * i + 1 < hidden) e[ch * 16 + i].y = 0.0f;
                    }
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) pk[i] = operand_pair<BF16>(e[ch * 16 + i]);
                ptx::tmem_st_32x32b_x16(s_at + ch * 16, pk);
            }
            ptx::tmem_st_wait();
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(p_ready);
            ok = __all_sync(0xffffffffu, bounded_wait(wctx, dp_full, it & 1, 0x050c0000u | (it & 0xffff)));
            if (!ok) break;
            ptx::tc_fence_after_sync();
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
                uint32_t r[32], pk[16];
                ptx::tmem_ld_32x32b_x32(dp_at + ch * 32, r);
                ptx::tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const float4 nd = ndelta[ch * 8 + i / 2];
                    float2 e0 = e[ch * 16 + i], e1 = e[ch * 16 + i + 1];
                    if constexpr (!BF16) { e0 = mul2(e0, g2); e1 = mul2(e1, g2); }
                    float2 d0 = mul2(e0, add2(f2(r[2 * i], r[2 * i + 1]), make_float2(nd.x, nd.y)));
                    float2 d1 = mul2(e1, add2(f2(r[2 * i + 2], r[2 * i + 3]), make_float2(nd.z, nd.w)));
                    if (masked) {                                       // dP may hold anything there
                        if (ch * 32 + 2 * i < hidden) d0.x = 0.0f;
                        if (ch * 32 + 2 * i + 1 < hidden) d0.y = 0.0f;
                        if (ch * 32 + 2 * i + 2 < hidden) d1.x = 0.0f;
                        if (ch * 32 + 2 * i + 3 < hidden) d1.y = 0.0f;
                    }
                    pk[i] = operand_pair<BF16>(d0);
                    pk[i + 1] = operand_pair<BF16>(d1);
                }
                ptx::tmem_st_32x32b_x16(dp_at + ch * 16, pk);
            }
            ptx::tmem_st_wait();
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(ds_ready);
        }
        if (ok && n_it > 0) ok = __all_sync(0xffffffffu, bounded_wait(wctx, acc_full, 0, 0x050d0000u));
        if (ok) {
            ptx::tc_fence_after_sync();
            const float dv_scale = BF16 ? 1.0f : 1.0f / (1 << kF16Shift), dk_scale = dv_scale * p.h.scale / g_scale;
            uint16_t* dv = static_cast<uint16_t*>(p.g.dv) + b * p.h.dv_s[0] + hk * p.h.dv_s[1] + key * p.h.dv_s[2] + half * (D / 2);
            uint16_t* dk = static_cast<uint16_t*>(p.g.dk) + b * p.h.dk_s[0] + hk * p.h.dk_s[1] + key * p.h.dk_s[2] + half * (D / 2);
#pragma unroll 1
            for (int ch = 0; ch < 2 * (D / 64); ++ch) {                 // dV's, then dK's pieces of 32 columns
                const bool is_dk = ch >= D / 64;
                const int col = (is_dk ? ch - D / 64 : ch) * 32;
                uint32_t r[32];
                if (n_it > 0) {
                    ptx::tmem_ld_32x32b_x32(tmem_base + lane_base + (is_dk ? kColDK : kColDV) + half * (D / 2) + col, r);
                    ptx::tmem_ld_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) r[i] = 0;
                }
                const float f = is_dk ? dk_scale : dv_scale;
                if (key < p.h.seq_k) {
                    uint4* dst = reinterpret_cast<uint4*>((is_dk ? dk : dv) + col);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint32_t v[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = round_pair<BF16>(__uint_as_float(r[8 * q + 2 * i]) * f, __uint_as_float(r[8 * q + 2 * i + 1]) * f);
                        dst[q] = make_uint4(v[0], v[1], v[2], v[3]);
                    }
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
        ptx::tmem_dealloc(tmem_base, 512);
    }
}

// The gradient of the bias, one warp's share: 32 x 64 blocks of dS. A block inside one run adds to a per-thread sum, which goes
// to the warp's sum of that run when the run changes; other blocks are added up along their 95 diagonals. Diagonal sums need
// no atomics: a partial sum moves one lane up per column, so that it follows its diagonal and is complete when it reaches lane 31
// (or the last column); every step adds one column of all 32 diagonals that pass it.
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
__global__ void __launch_bounds__(kBwdThreads, 1)
heads_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                const __grid_constant__ CUtensorMap map_do, const __grid_constant__ BwdParams p) {
    using S = BwdSmem<D>;
    constexpr int kChunks = D / 64;
    constexpr uint32_t kColS = 0, kColDP = 256, kColDQ = 384;           // S: two buffers of 128 columns
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - ptx::smem_u32(smem_raw));
    const uint32_t q_smem = smem_base, do_smem = smem_base + S::kOperand;
    auto k_smem = [&](int s) { return smem_base + (2 + s) * S::kOperand; };
    auto v_smem = [&](int s) { return smem_base + (4 + s) * S::kOperand; };
    const uint32_t bar_base = smem_base + S::kBarOffset;
    const uint32_t q_full = bar_base, do_full = bar_base + 8, s_full = bar_base + 16 /* two */, dp_full = bar_base + 32, ds_ready = bar_base + 40,
                   acc_full = bar_base + 48, k_full = bar_base + 64, k_empty = bar_base + 80, v_full = bar_base + 96, v_empty = bar_base + 112;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_gen + S::kBarOffset + 128);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    BiasShared& bias = *reinterpret_cast<BiasShared*>(smem_gen + S::kBiasOffset);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int bh = blockIdx.x / p.q_tiles;
    const int qt = p.h.causal ? p.q_tiles - 1 - (int)(blockIdx.x % p.q_tiles) : (int)(blockIdx.x % p.q_tiles);
    const int b = bh / p.h.heads, h = bh % p.h.heads, hk = h / p.h.group;
    const int row0 = qt * kTile;
    const int n_keys = heads_key_count(p.h, b), offset = heads_offset(p.h, n_keys);
    const int key_end = p.h.causal ? max(0, min(n_keys, min(row0 + kTile, p.h.seq_q) + offset)) : n_keys;
    const int n_it = (key_end + kTile - 1) / kTile;
    const WaitCtx wctx{abort_flag, p.status, p.wait_limit_ns};

    if (threadIdx.x == 0) {
        ptx::mbar_init(q_full, 1); ptx::mbar_init(do_full, 1); ptx::mbar_init(s_full, 1); ptx::mbar_init(s_full + 8, 1);
        ptx::mbar_init(dp_full, 1); ptx::mbar_init(ds_ready, 8); ptx::mbar_init(acc_full, 1);
        for (int s = 0; s < 2; ++s) {
            ptx::mbar_init(k_full + 8 * s, 1); ptx::mbar_init(k_empty + 8 * s, 1);
            ptx::mbar_init(v_full + 8 * s, 1); ptx::mbar_init(v_empty + 8 * s, 1);
        }
        *abort_flag = 0;
        ptx::mbar_fence_init();
        ptx::prefetch_tensormap(&map_q); ptx::prefetch_tensormap(&map_k); ptx::prefetch_tensormap(&map_v); ptx::prefetch_tensormap(&map_do);
    }
    if (BIAS) load_bias(bias, p.h, h, threadIdx.x, kBwdThreads);
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
        if (lane == 0 && n_it > 0) {
            ptx::mbar_arrive_expect_tx(q_full, S::kOperand);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) ptx::tma_load_4d(q_smem + c * (kTile * 128), &map_q, q_full, c * 64, row0, h * p.q_at.head, b * p.q_at.batch);
            for (int it = 0; it < n_it; ++it) {
                const int s = it & 1, key0 = it * kTile;
                const uint32_t empty = ((it >> 1) & 1) ^ 1;
                if (!bounded_wait(wctx, k_empty + 8 * s, empty, 0x06010000u | (it & 0xffff))) break;
                ptx::mbar_arrive_expect_tx(k_full + 8 * s, S::kOperand);
#pragma unroll
                for (int c = 0; c < kChunks; ++c)
                    ptx::tma_load_4d(k_smem(s) + c * (kTile * 128), &map_k, k_full + 8 * s, c * 64, key0, hk * p.k_at.head, b * p.k_at.batch);
                if (it == 0) {
                    ptx::mbar_arrive_expect_tx(do_full, S::kOperand);
#pragma unroll
                    for (int c = 0; c < kChunks; ++c)
                        ptx::tma_load_4d(do_smem + c * (kTile * 128), &map_do, do_full, c * 64, row0, h * p.do_at.head, b * p.do_at.batch);
                }
                if (!bounded_wait(wctx, v_empty + 8 * s, empty, 0x06020000u | (it & 0xffff))) break;
                ptx::mbar_arrive_expect_tx(v_full + 8 * s, S::kOperand);
#pragma unroll
                for (int c = 0; c < kChunks; ++c)
                    ptx::tma_load_4d(v_smem(s) + c * (kTile * 128), &map_v, v_full + 8 * s, c * 64, key0, hk * p.v_at.head, b * p.v_at.batch);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---- MMA issuer ----------------------------------------------------------------------------------
        if (lane == 0 && n_it > 0) {
            constexpr uint32_t idesc_s = ptx::mma_idesc_f16(BF16, false, false, kTile, kTile);
            constexpr uint32_t idesc_d = ptx::mma_idesc_f16(BF16, false, true, kTile, D);
            auto scores = [&](uint32_t col, uint32_t a, uint32_t bb) {
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint32_t off = (kk / 4) * (kTile * 128) + (kk % 4) * 32;
                    ptx::mma_ss(tmem_base + col, ptx::smem_desc_sw128(a + off, 16, 1024), ptx::smem_desc_sw128(bb + off, 16, 1024), idesc_s, kk != 0);
                }
            };
            auto s_product = [&](int it) {
                if (!bounded_spin(wctx, k_full + 8 * (it & 1), (it >> 1) & 1, 0x06030000u | (it & 0xffff))) return false;
                ptx::tc_fence_after_sync();
                scores(kColS + 128 * (it & 1), q_smem, k_smem(it & 1));
                ptx::mma_commit(s_full + 8 * (it & 1));
                return true;
            };
            auto dp_product = [&](int it) {
                if (!bounded_spin(wctx, v_full + 8 * (it & 1), (it >> 1) & 1, 0x06040000u | (it & 0xffff))) return false;
                ptx::tc_fence_after_sync();
                scores(kColDP, do_smem, v_smem(it & 1));
                ptx::mma_commit(v_empty + 8 * (it & 1));
                ptx::mma_commit(dp_full);
                return true;
            };
            bool ok = bounded_spin(wctx, q_full, 0, 0x06050000u) && s_product(0) && bounded_spin(wctx, do_full, 0, 0x06060000u) && dp_product(0);
            if (ok && n_it > 1) ok = s_product(1);
            for (int it = 0; it < n_it && ok; ++it) {
                if (!(ok = bounded_spin(wctx, ds_ready, it & 1, 0x06070000u | (it & 0xffff)))) break;
                ptx::tc_fence_after_sync();
                if (it + 1 < n_it && !(ok = dp_product(it + 1))) break;
#pragma unroll
                for (int kk = 0; kk < kTile / 16; ++kk)         // dQ += dS K, contraction over the keys
                    ptx::mma_ts(tmem_base + kColDQ, tmem_base + kColS + 128 * (it & 1) + operand_col(kk),
                                ptx::smem_desc_sw128(k_smem(it & 1) + kk * (16 * 128), kTile * 128, 1024), idesc_d, (it | kk) != 0);
                ptx::mma_commit(k_empty + 8 * (it & 1));
                if (it + 2 < n_it && !(ok = s_product(it + 2))) break;
            }
            if (ok) ptx::mma_commit(acc_full);
        }
        __syncwarp();
    } else {
        // ---- probabilities and their gradients: rows are queries, columns keys ---------------------------------------
        const int w = warp - 2, quarter = warp & 3, half = w >> 2;
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        const int row = row0 + quarter * 32 + lane;
        const int64_t at_row = (int64_t)bh * p.g.pad_q + row;
        const float nlse = p.g.lse2[at_row], ndelta = p.g.delta[at_row];
        const float g_scale = ds_scale<BF16>(p.g, b * p.h.kv_heads + hk, (int64_t)p.h.batch * p.h.kv_heads);
        const float2 nd2 = make_float2(ndelta, ndelta), g2 = make_float2(g_scale, g_scale);
        const int sees = p.h.causal ? min(n_keys, row + offset + 1) : n_keys;
        const bool want_bias = BIAS && p.g.dtable != nullptr;
        float* sums = reinterpret_cast<float*>(smem_gen + S::kSumsOffset) + w * kHeadsMaxRuns;      // this warp's, by run
        RunSums rs{0.0f, 0};
        bool ok = true;
        WarpBias wb;
        wb.reset();
        if constexpr (BIAS) {
            for (int r = lane; r < p.h.n_runs; r += 32) sums[r] = 0.0f;
            __syncwarp();
        }
        for (int it = 0; it < n_it && ok; ++it) {
            const int key0 = it * kTile + half * 64;            // this thread's first key
            const uint32_t s_at = tmem_base + lane_base + kColS + 128 * (it & 1) + half * 64, dp_at = tmem_base + lane_base + kColDP + half * 64;
            const int d0 = key0 - (row0 + quarter * 32 + 31 + offset);
            float c = p.h.scale_log2, add = nlse;
            bool looked_up = false;
            if constexpr (BIAS) looked_up = !wb.block(bias, bias.value, w, lane, p.h.n_runs, d0);
            ok = __all_sync(0xffffffffu, bounded_wait(wctx, s_full + 8 * (it & 1), (it >> 1) & 1, 0x06080000u | (it & 0xffff)));
            if (!ok) break;
            ptx::tc_fence_after_sync();
            const int valid = sees - key0;                      // of this thread's columns
            const bool masked = __any_sync(0xffffffffu, valid < 64);
            float2 e[32];
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
                uint32_t r[32];
                ptx::tmem_ld_32x32b_x32(s_at + ch * 32, r);
                ptx::tmem_ld_wait();
                float cc = c, aa = add;
                if constexpr (BIAS) {
                    if (looked_up) {
                        const float* at = bias.by_dist[w] + 31 - lane + ch * 32;
#pragma unroll
                        for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(fmaf(__uint_as_float(r[i]), c, at[i]));
                        cc = 1.0f;
                    } else {
                        aa = add + wb.same;
                    }
                }
                const float2 c2 = make_float2(cc, cc), a2 = make_float2(aa, aa);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float2 y = fma2(f2(r[2 * i], r[2 * i + 1]), c2, a2);
                    e[ch * 16 + i] = make_float2(ptx::ex2_approx(y.x), ptx::ex2_approx(y.y));
                }
            }
            // K rows behind the key count hold whatever the caller left there: cleared before dQ's product multiplies them by dS's zeros
            const int live = n_keys - it * kTile;
            if (live < kTile && n_keys < p.h.seq_k) {           // S has been computed from them; its columns there are not used
                for (int x = live * 8 + (int)threadIdx.x - 64; x < kTile * 8; x += 256)
#pragma unroll
                    for (int ch = 0; ch < kChunks; ++ch)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(k_smem(it & 1) + ch * (kTile * 128) + x * 16), "r"(0) : "memory");
                ptx::fence_proxy_async_smem();
            }
            ok = __all_sync(0xffffffffu, bounded_wait(wctx, dp_full, it & 1, 0x06090000u | (it & 0xffff)));
            if (!ok) break;
            ptx::tc_fence_after_sync();
            float diag = 0.0f;                                  // a diagonal's partial sum, passing through this lane
            float2 same_sum = make_float2(0.0f, 0.0f);
            if (BIAS && looked_up) __syncwarp();                // the biases have been read: the diagonal sums take their place
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
                uint32_t r[32], pk[16];
                ptx::tmem_ld_32x32b_x32(dp_at + ch * 32, r);
                ptx::tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float2 ee = e[ch * 16 + i];
                    if constexpr (!BF16) ee = mul2(ee, g2);
                    float2 ds = mul2(ee, add2(f2(r[2 * i], r[2 * i + 1]), nd2));
                    if (masked) {
                        if (ch * 32 + 2 * i >= valid) ds.x = 0.0f;
                        if (ch * 32 + 2 * i + 1 >= valid) ds.y = 0.0f;
                    }
                    pk[i] = operand_pair<BF16>(ds);
                    if constexpr (BIAS) {
                        r[2 * i] = __float_as_uint(ds.x);
                        r[2 * i + 1] = __float_as_uint(ds.y);
                    }
                }
                ptx::tmem_st_32x32b_x16(s_at + ch * 16, pk);
                if (ch == 1) {
                    ptx::tmem_st_wait();
                    ptx::tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(ds_ready);
                }
                if constexpr (BIAS) {
                    if (want_bias) {
                        if (looked_up) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                const float below = __shfl_up_sync(0xffffffffu, diag, 1);
                                diag = (lane == 0 ? 0.0f : below) + __uint_as_float(r[i]);
                                if (lane == 31) bias.by_dist[w][ch * 32 + i] = diag;
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i) same_sum = add2(same_sum, f2(r[2 * i], r[2 * i + 1]));
                        }
                    }
                }
            }
            if constexpr (BIAS) {
                if (want_bias) {
                    if (looked_up) {
                        if (lane < 31) bias.by_dist[w][94 - lane] = diag;
                        __syncwarp();
                        // runs the block touches, one lane each
                        const int ra = heads_run_of(bias.first, p.h.n_runs, d0), rb = heads_run_of(bias.first, p.h.n_runs, d0 + 94);
                        for (int run = ra + lane; run <= rb; run += 32) {
                            const int from = run == ra ? 0 : bias.first[run] - d0, to = run == rb ? 95 : bias.first[run + 1] - d0;
                            float v = 0.0f;
                            for (int t = from; t < to; ++t) v += bias.by_dist[w][t];
                            sums[run] += v;
                        }
                        __syncwarp();
                    } else {
                        if (rs.run != wb.run) {
                            rs.flush(sums, lane);
                            __syncwarp();
                            rs.run = wb.run;
                        }
                        rs.acc += same_sum.x + same_sum.y;
                    }
                }
            }
        }
        if (ok && n_it > 0) ok = __all_sync(0xffffffffu, bounded_wait(wctx, acc_full, 0, 0x060a0000u));
        if (ok) {
            ptx::tc_fence_after_sync();
            const float out = BF16 ? 1.0f : 1.0f / ((1 << kF16Shift) * g_scale);
            const float f = p.h.scale * out;
            uint16_t* dq = static_cast<uint16_t*>(p.g.dq) + b * p.h.dq_s[0] + h * p.h.dq_s[1] + row * p.h.dq_s[2] + half * (D / 2);
#pragma unroll 1
            for (int ch = 0; ch < D / 64; ++ch) {
                uint32_t r[32];
                if (n_it > 0) {
                    ptx::tmem_ld_32x32b_x32(tmem_base + lane_base + kColDQ + half * (D / 2) + ch * 32, r);
                    ptx::tmem_ld_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) r[i] = 0;
                }
                if (row < p.h.seq_q) {
                    uint4* dst = reinterpret_cast<uint4*>(dq + ch * 32);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint32_t v[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = round_pair<BF16>(__uint_as_float(r[8 * q + 2 * i]) * f, __uint_as_float(r[8 * q + 2 * i + 1]) * f);
                        dst[q] = make_uint4(v[0], v[1], v[2], v[3]);
                    }
                }
            }
            if constexpr (BIAS) {
                if (want_bias) {
                    rs.flush(sums, lane);
                    __syncwarp();
                    const float back = BF16 ? 1.0f / kCutScale : out;
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

template <int D, bool BF16>
static int launch_bwd(BwdParams& p, cudaStream_t s) {
    const HeadsParams& h = p.h;
    CUtensorMap mq, mk, mv, mdo;
    int rc = make_map(&mq, &p.q_at, p.g.q, h.batch, h.heads, h.seq_q, D, h.q_s, kTile, 1);
    if (rc == EMMYB200_OK) rc = make_map(&mk, &p.k_at, p.g.k, h.batch, h.kv_heads, h.seq_k, D, h.k_s, kTile, 1);
    if (rc == EMMYB200_OK) rc = make_map(&mv, &p.v_at, p.g.v, h.batch, h.kv_heads, h.seq_k, D, h.v_s, kTile, 1);
    if (rc == EMMYB200_OK) rc = make_map(&mdo, &p.do_at, p.g.d_o, h.batch, h.heads, h.seq_q, D, h.do_s, kTile, 1);
    if (rc != EMMYB200_OK) return rc;
    EMMY_CUDA(cudaGetSymbolAddress(reinterpret_cast<void**>(&p.status), g_bwd_status));
    const int64_t kv_ctas = (int64_t)h.batch * h.kv_heads * p.k_tiles, q_ctas = (int64_t)h.batch * h.heads * p.q_tiles;
    if (kv_ctas >= (1ll << 31) || q_ctas >= (1ll << 31)) return fail(EMMYB200_ERR_SHAPE, "attention_heads_bwd: the tiles exceed the grid limit");
    auto dkv = h.n_runs ? heads_dkv_kernel<D, BF16, true> : heads_dkv_kernel<D, BF16, false>;
    auto dq = h.n_runs ? heads_dq_kernel<D, BF16, true> : heads_dq_kernel<D, BF16, false>;
    EMMY_CUDA(cudaFuncSetAttribute(dkv, cudaFuncAttributeMaxDynamicSharedMemorySize, BwdSmem<D>::kTotal));
    EMMY_CUDA(cudaFuncSetAttribute(dq, cudaFuncAttributeMaxDynamicSharedMemorySize, BwdSmem<D>::kTotal));
    dkv<<<(unsigned)kv_ctas, kBwdThreads, BwdSmem<D>::kTotal, s>>>(mq, mk, mv, mdo, p);
    rc = launch_status("heads_dkv_kernel");
    if (rc != EMMYB200_OK) return rc;
    dq<<<(unsigned)q_ctas, kBwdThreads, BwdSmem<D>::kTotal, s>>>(mq, mk, mv, mdo, p);
    return launch_status("heads_dq_kernel");
}

}  // namespace heads

bool heads_bwd_sm100_takes(const HeadsParams& p, int dtype, int d, const HeadsGrads& g) {
    using namespace heads;
    return heads_sm100_takes(p, dtype, d, g.q, g.k, g.v, g.q) && map_fits(g.d_o, p.batch, p.heads, p.seq_q, p.do_s) &&
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
