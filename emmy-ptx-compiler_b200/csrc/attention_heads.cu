// Entry points of attention over heads (forward with log-sum-exp, backward, relative position bias): argument checks, the
// choice between the tensor-core and the CUDA-core kernels, the workspace, and the two small kernels around the backward
// pass: row terms before it (D_i = dO_i . O_i, one pass over dO and O) and the bias gradient's ordered sum after it.
#include <algorithm>

#include "attention_heads.cuh"

namespace emmy {

int check_sm100();

// ---- before the backward pass -------------------------------------------------------------------------------------------
// Row terms of the padded row arrays: -D = -dO . O and -lse * log2(e) + shift. Rows behind seq_q and rows that saw nothing get
// -inf, which makes their probabilities 2^(s - inf) = 0 without a test in the kernels.
__device__ __forceinline__ void store_row(const HeadsParams& p, const HeadsGrads& g, int64_t bh, int row, float dot, float shift) {
    float l = -INFINITY;
    if (row < p.seq_q) {
        const float v = g.lse[bh * p.seq_q + row];
        l = v == -INFINITY ? -INFINITY : fmaf(v, -kLog2e, shift);
    }
    g.lse2[bh * g.pad_q + row] = l;
    g.delta[bh * g.pad_q + row] = -dot;
}

// Any type and alignment: one warp per row.
template <typename T>
__global__ void __launch_bounds__(256) heads_rows_kernel(HeadsParams p, HeadsGrads g, int d) {
    const int lane = threadIdx.x & 31;
    const int64_t row_at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row_at >= (int64_t)p.batch * p.heads * g.pad_q) return;
    const int row = (int)(row_at % g.pad_q);
    const int64_t bh = row_at / g.pad_q;
    const int b = (int)(bh / p.heads), h = (int)(bh % p.heads);
    float sum = 0.0f;
    if (row < p.seq_q) {
        const T* o = static_cast<const T*>(g.o) + b * p.o_s[0] + h * p.o_s[1] + row * p.o_s[2];
        const T* d_o = static_cast<const T*>(g.d_o) + b * p.do_s[0] + h * p.do_s[1] + row * p.do_s[2];
        for (int c = lane; c < d; c += 32) sum = fmaf(heads_load(o, c), heads_load(d_o, c), sum);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane == 0) store_row(p, g, bh, row, sum, 0.0f);
}

// 16-bit rows of 64 or 128 aligned elements, as the tensor-core kernels take them: bound by the bytes of dO and O. D / 8 lanes share a
// row with one 128-bit access each, four rows per thread in flight (262144 rows of 128, bf16: 30 us, 4.4 TB/s). A block's
// rows belong to one (batch entry, head). f16 (NORMS): also the largest squared row norms of dO and, in the blocks behind
// those, of V's rows below the key count; a maximum does not depend on the order it is taken in.
template <typename T, int D, bool NORMS>
__global__ void __launch_bounds__(256) heads_rows16_kernel(HeadsParams p, HeadsGrads g, float shift, int q_blocks) {
    constexpr int kLanes = D / 8, kRowsPerPass = 256 / kLanes, kPasses = 4, kRows = kRowsPerPass * kPasses;     // 64 or 128 rows
    const int sub = threadIdx.x % kLanes, first = threadIdx.x / kLanes;
    const bool is_q = !NORMS || (int)blockIdx.x < q_blocks;
    const int block = is_q ? blockIdx.x : blockIdx.x - q_blocks;
    const int pad_k = (p.seq_k + 127) / 128 * 128, per = (is_q ? g.pad_q : pad_k) / kRows;
    const int bh = block / per, row0 = block % per * kRows;
    const int heads = is_q ? p.heads : p.kv_heads;
    const int b = bh / heads, h = bh % heads;
    const T* x = is_q ? static_cast<const T*>(g.d_o) + b * p.do_s[0] + h * p.do_s[1] : static_cast<const T*>(g.v) + b * p.v_s[0] + h * p.v_s[1];
    const int64_t x_row = is_q ? p.do_s[2] : p.v_s[2];
    const T* o = is_q ? static_cast<const T*>(g.o) + b * p.o_s[0] + h * p.o_s[1] : x;
    const int64_t o_row = is_q ? p.o_s[2] : x_row;
    const int rows = is_q ? p.seq_q : heads_key_count(p, b);
    uint4 xv[kPasses], ov[kPasses];
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        const int row = row0 + i * kRowsPerPass + first;
        xv[i] = ov[i] = make_uint4(0, 0, 0, 0);
        if (row < rows) {
            xv[i] = __ldg(reinterpret_cast<const uint4*>(x + row * x_row) + sub);
            if (is_q) ov[i] = __ldg(reinterpret_cast<const uint4*>(o + row * o_row) + sub);
        }
    }
    float most = 0.0f;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        const T* xe = reinterpret_cast<const T*>(&xv[i]);
        const T* oe = reinterpret_cast<const T*>(&ov[i]);
        float dot = 0.0f, norm = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float v = heads_load(xe, k);
            dot = fmaf(heads_load(oe, k), v, dot);
            if (NORMS) norm = fmaf(v, v, norm);
        }
#pragma unroll
        for (int off = kLanes / 2; off > 0; off >>= 1) {
            dot += __shfl_xor_sync(0xffffffffu, dot, off);
            if (NORMS) norm += __shfl_xor_sync(0xffffffffu, norm, off);
        }
        if (is_q && sub == 0) store_row(p, g, bh, row0 + i * kRowsPerPass + first, dot, shift);
        if (NORMS) {
            nan |= !(norm == norm);
            most = fmaxf(most, norm);
        }
    }
    if (NORMS) {
        if (nan) most = INFINITY;               // as for an infinite norm: no scaling
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
        __shared__ float warp_most[8];
        if ((threadIdx.x & 31) == 0) warp_most[threadIdx.x >> 5] = most;
        __syncthreads();
        if (threadIdx.x == 0) {
#pragma unroll
            for (int k = 0; k < 8; ++k) most = fmaxf(most, warp_most[k]);
            const int64_t bk = is_q ? (int64_t)b * p.kv_heads + h / p.group : (int64_t)p.batch * p.kv_heads + bh;
            atomicMax(reinterpret_cast<unsigned int*>(g.amax) + bk, __float_as_uint(most));        // not negative: ordered as their bit patterns
        }
    }
}

template <typename T, bool NORMS>
static int launch_rows16(const HeadsParams& p, const HeadsGrads& g, int d, float shift, cudaStream_t s) {
    const int rows = d == 128 ? 64 : 128;
    const int64_t q_blocks = (int64_t)p.batch * p.heads * (g.pad_q / rows);
    const int64_t blocks = q_blocks + (NORMS ? (int64_t)p.batch * p.kv_heads * ((p.seq_k + 127) / 128 * (128 / rows)) : 0);
    if (blocks >= (1ll << 31)) return fail(EMMYB200_ERR_SHAPE, "attention_heads_bwd: the rows exceed the grid limit");
    if (d == 128) heads_rows16_kernel<T, 128, NORMS><<<(unsigned)blocks, 256, 0, s>>>(p, g, shift, (int)q_blocks);
    else heads_rows16_kernel<T, 64, NORMS><<<(unsigned)blocks, 256, 0, s>>>(p, g, shift, (int)q_blocks);
    return launch_status("heads_rows16_kernel");
}

// ---- after it -----------------------------------------------------------------------------------------------------------
// dtable[bucket][head]: the runs of the bucket over the batch and the query tiles, added up in a fixed order (a bucket may
// own several runs, or none: zero). One block per (bucket, head).
template <typename T>
__global__ void __launch_bounds__(128) heads_dtable_kernel(HeadsParams p, HeadsGrads g) {
    __shared__ float part[4];
    const int bucket = blockIdx.x / p.heads, h = blockIdx.x % p.heads;
    float sum = 0.0f;
    for (int r = 0; r < p.n_runs; ++r) {
        if (p.run_bucket[r] != bucket) continue;
        for (int i = threadIdx.x; i < p.batch * g.q_tiles; i += 128) {
            const int b = i / g.q_tiles, t = i % g.q_tiles;
            sum += g.run_sums[(((int64_t)b * p.heads + h) * g.q_tiles + t) * p.n_runs + r];
        }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) heads_store(static_cast<T*>(g.dtable), blockIdx.x, (part[0] + part[1]) + (part[2] + part[3]));
}

// ---- arguments ------------------------------------------------------------------------------------------------------------
static bool known_dtype(int t) { return t == EMMYB200_F32 || t == EMMYB200_F16 || t == EMMYB200_BF16; }

// An output must not write one element from two places: with the extents sorted by stride, each stride covers all below it.
static bool writes_once(const int64_t* stride, int64_t batch, int64_t heads, int64_t rows, int64_t d) {
    int64_t s[3] = {stride[0], stride[1], stride[2]}, n[3] = {batch, heads, rows};
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (s[j] < s[i]) { std::swap(s[i], s[j]); std::swap(n[i], n[j]); }
    int64_t covered = d;
    for (int i = 0; i < 3; ++i) {
        if (n[i] <= 1) continue;
        if (s[i] < covered) return false;
        covered = s[i] * (n[i] - 1) + covered;
    }
    return true;
}

static int check_desc(const emmyb200_attention_heads_desc* c, bool backward, const char* who) {
    if (c == nullptr) return fail(EMMYB200_ERR_ARG, "%s: null description", who);
    if (!known_dtype(c->dtype)) return fail(EMMYB200_ERR_UNSUPPORTED, "%s: dtype %d (f32, f16 and bf16 only)", who, c->dtype);
    if (c->flags & ~(EMMYB200_HEADS_CAUSAL | EMMYB200_HEADS_ALIGN_END)) return fail(EMMYB200_ERR_ARG, "%s: unknown flags 0x%x", who, c->flags);
    if (c->batch < 0 || c->heads < 0 || c->kv_heads < 0 || c->seq_q < 0 || c->seq_k < 0) return fail(EMMYB200_ERR_SHAPE, "%s: negative extent", who);
    const int64_t limit = 1ll << 30;
    if (c->batch >= limit || c->heads >= (1 << 20) || c->seq_q >= limit || c->seq_k >= limit)
        return fail(EMMYB200_ERR_SHAPE, "%s: extents must be below 2^30 (heads: 2^20)", who);
    if (c->batch * c->heads >= limit || c->batch * c->heads * ((c->seq_q > c->seq_k ? c->seq_q : c->seq_k) + 128) >= (1ll << 44))
        return fail(EMMYB200_ERR_SHAPE, "%s: batch * heads must be below 2^30, with the rows below 2^44", who);
    if (c->d % 32 != 0 || c->d < 32 || c->d > 128) return fail(EMMYB200_ERR_UNSUPPORTED, "%s: head dim %lld (a multiple of 32 up to 128)", who, (long long)c->d);
    if (c->heads != 0 && (c->kv_heads == 0 || c->heads % c->kv_heads != 0))
        return fail(EMMYB200_ERR_SHAPE, "%s: %lld query heads over %lld key heads (a multiple)", who, (long long)c->heads, (long long)c->kv_heads);
    if (c->heads == 0 && c->kv_heads != 0) return fail(EMMYB200_ERR_SHAPE, "%s: key heads without query heads", who);
    if (!(c->scale > 0.0f) || !(c->scale < INFINITY)) return fail(EMMYB200_ERR_ARG, "%s: scale must be a positive finite number", who);
    const int64_t* strides[8] = {c->q_stride, c->k_stride, c->v_stride, c->o_stride, c->do_stride, c->dq_stride, c->dk_stride, c->dv_stride};
    for (int t = 0; t < (backward ? 8 : 4); ++t)
        for (int i = 0; i < 3; ++i)
            if (strides[t][i] < 0) return fail(EMMYB200_ERR_SHAPE, "%s: negative stride", who);
    if (!backward && !writes_once(c->o_stride, c->batch, c->heads, c->seq_q, c->d)) return fail(EMMYB200_ERR_SHAPE, "%s: the strides of O overlap", who);
    if (backward && (!writes_once(c->dq_stride, c->batch, c->heads, c->seq_q, c->d) || !writes_once(c->dk_stride, c->batch, c->kv_heads, c->seq_k, c->d) ||
                     !writes_once(c->dv_stride, c->batch, c->kv_heads, c->seq_k, c->d)))
        return fail(EMMYB200_ERR_SHAPE, "%s: the strides of a gradient overlap", who);
    if (c->n_runs < 0 || c->n_runs > kHeadsMaxRuns) return fail(EMMYB200_ERR_ARG, "%s: %d runs of distances (at most %d)", who, c->n_runs, kHeadsMaxRuns);
    if (c->n_runs) {
        if (!known_dtype(c->bias_dtype)) return fail(EMMYB200_ERR_UNSUPPORTED, "%s: bias dtype %d (f32, f16 and bf16 only)", who, c->bias_dtype);
        if (c->buckets < 1 || c->buckets > kHeadsMaxRuns) return fail(EMMYB200_ERR_ARG, "%s: %d buckets (1 to %d)", who, c->buckets, kHeadsMaxRuns);
        if (c->bias_stride[0] < 0 || c->bias_stride[1] < 0) return fail(EMMYB200_ERR_SHAPE, "%s: negative stride", who);
        for (int r = 0; r < c->n_runs; ++r) {
            if (c->run_bucket[r] < 0 || c->run_bucket[r] >= c->buckets) return fail(EMMYB200_ERR_ARG, "%s: run %d names bucket %d of %d", who, r, c->run_bucket[r], c->buckets);
            if (r >= 1 && (c->run_first[r] < -(1 << 30) || c->run_first[r] > (1 << 30))) return fail(EMMYB200_ERR_ARG, "%s: run %d begins beyond 2^30", who, r);
            if (r >= 2 && c->run_first[r] <= c->run_first[r - 1]) return fail(EMMYB200_ERR_ARG, "%s: the runs' distances do not rise at run %d", who, r);
        }
    }
    return EMMYB200_OK;
}

static HeadsParams make_params(const emmyb200_attention_heads_desc* c, const int32_t* key_lens, const void* table) {
    HeadsParams p = {};
    p.batch = (int)c->batch; p.heads = (int)c->heads; p.kv_heads = (int)c->kv_heads; p.seq_q = (int)c->seq_q; p.seq_k = (int)c->seq_k;
    p.group = c->kv_heads ? (int)(c->heads / c->kv_heads) : 1;
    p.causal = (c->flags & EMMYB200_HEADS_CAUSAL) ? 1 : 0;
    p.at_end = (c->flags & EMMYB200_HEADS_ALIGN_END) ? 1 : 0;
    p.scale = c->scale;
    p.scale_log2 = c->scale * kLog2e;
    p.key_lens = key_lens;
    for (int i = 0; i < 3; ++i) {
        p.q_s[i] = c->q_stride[i]; p.k_s[i] = c->k_stride[i]; p.v_s[i] = c->v_stride[i]; p.o_s[i] = c->o_stride[i];
        p.do_s[i] = c->do_stride[i]; p.dq_s[i] = c->dq_stride[i]; p.dk_s[i] = c->dk_stride[i]; p.dv_s[i] = c->dv_stride[i];
    }
    p.table = table;
    p.table_dtype = c->bias_dtype;
    p.n_runs = c->n_runs;
    p.table_s[0] = c->bias_stride[0]; p.table_s[1] = c->bias_stride[1];
    for (int r = 0; r < c->n_runs; ++r) {
        p.run_first[r] = c->run_first[r];
        p.run_bucket[r] = (uint8_t)c->run_bucket[r];
    }
    return p;
}

// Workspace of a backward pass: [lse2][delta][run sums][amax], each 256-byte aligned. Large enough for either kind of kernels.
struct BwdLayout {
    int64_t pad_q, parts, delta_at, sums_at, amax_at, total;
};
static int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }
static BwdLayout bwd_layout(const emmyb200_attention_heads_desc* c) {
    BwdLayout w;
    w.pad_q = (c->seq_q + 127) / 128 * 128;
    w.parts = w.pad_q / 128 * 8;                // tensor cores: eight warps per 128 queries; CUDA cores: one part per 16 or 64
    const int64_t rows = round256(c->batch * c->heads * w.pad_q * 4);
    w.delta_at = rows;
    w.sums_at = 2 * rows;
    w.amax_at = w.sums_at + round256(c->n_runs ? c->batch * c->heads * w.parts * c->n_runs * 4 : 0);
    w.total = w.amax_at + (c->dtype == EMMYB200_F16 ? round256(2 * c->batch * c->kv_heads * 4) : 0);
    return w;
}

}  // namespace emmy

extern "C" int emmyb200_relative_runs(int buckets, int64_t max_distance, int bidirectional, int32_t* run_first, int32_t* run_bucket) {
    using namespace emmy;
    if (run_first == nullptr || run_bucket == nullptr) return fail(EMMYB200_ERR_ARG, "relative_runs: null output");
    const int m = bidirectional ? buckets / 2 : buckets, e = m / 2;
    if (buckets < 2 || buckets > kHeadsMaxRuns || (bidirectional && buckets % 2 != 0) || m < 2)
        return fail(EMMYB200_ERR_ARG, "relative_runs: %d buckets (2 to %d one-sided, an even number from 4 on when bidirectional)", buckets, kHeadsMaxRuns);
    if (max_distance <= e || max_distance > (1ll << 30)) return fail(EMMYB200_ERR_ARG, "relative_runs: max_distance %lld (above %d, at most 2^30)", (long long)max_distance, e);
    // lo[k]: the smallest n of bucket k. n belongs to bucket e + k or later when n >= e (max_distance / e)^(k / (m - e)); the
    // border is a whole number exactly where the power is one, which the long double power (error some 2^-62 of its value) hits to within 2^-56.
    int64_t lo[kHeadsMaxRuns + 1];
    for (int n = 0; n < e; ++n) lo[n] = n;
    for (int k = 0; k < m - e; ++k) {
        const long double x = e * powl((long double)max_distance / e, (long double)k / (m - e));
        const long double near = roundl(x);
        lo[e + k] = (int64_t)(fabsl(x - near) <= x * 0x1p-56L ? near : ceill(x));
    }
    lo[m] = INT64_MAX;
    int n = 0;
    run_first[n] = -(1 << 30);
    run_bucket[n++] = m - 1;
    for (int k = m - 2; k >= 0; --k)
        if (lo[k + 1] > lo[k]) {                // distances -(lo[k + 1] - 1) .. -lo[k]
            run_first[n] = (int32_t)-(lo[k + 1] - 1);
            run_bucket[n++] = k;
        }
    for (int k = 1; bidirectional && k < m; ++k)
        if (lo[k + 1] > lo[k]) {
            run_first[n] = (int32_t)lo[k];
            run_bucket[n++] = m + k;
        }
    return n;
}

extern "C" int64_t emmyb200_attention_heads_workspace_bytes(const emmyb200_attention_heads_desc* c, int backward) {
    using namespace emmy;
    if (check_desc(c, backward != 0, "attention_heads_workspace_bytes") != EMMYB200_OK) return -1;
    if (backward) return bwd_layout(c).total;
    if (c->batch * c->heads * c->seq_q * c->seq_k == 0 || c->dtype == EMMYB200_F32 || (c->d != 64 && c->d != 128)) return 0;
    return fwd_workspace(heads_fwd_plan(make_params(c, nullptr, nullptr), c->d), c->d);
}

extern "C" int emmyb200_attention_heads_fwd(const emmyb200_attention_heads_desc* c, const void* Q, const void* K, const void* V,
                                            const int32_t* key_lens, const void* table, void* O, float* lse, void* workspace,
                                            int64_t workspace_bytes, void* cuda_stream) {
    using namespace emmy;
    int rc = check_desc(c, false, "attention_heads_fwd");
    if (rc != EMMYB200_OK) return rc;
    if (c->batch == 0 || c->heads == 0 || c->seq_q == 0) return EMMYB200_OK;
    if (Q == nullptr || O == nullptr || lse == nullptr || (c->seq_k > 0 && (K == nullptr || V == nullptr))) return fail(EMMYB200_ERR_ARG, "attention_heads_fwd: null buffer");
    if (c->n_runs && table == nullptr) return fail(EMMYB200_ERR_ARG, "attention_heads_fwd: runs of distances without a table");
    const int64_t need = emmyb200_attention_heads_workspace_bytes(c, 0);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 256)))
        return fail(EMMYB200_ERR_ARG, "attention_heads_fwd: needs %lld bytes of 256-byte aligned workspace", (long long)need);
    rc = check_sm100();
    if (rc != EMMYB200_OK) return rc;
    const HeadsParams p = make_params(c, key_lens, table);
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    if (heads_sm100_takes(p, c->dtype, (int)c->d, Q, K, V, O)) return heads_fwd_sm100(c->dtype, (int)c->d, p, heads_fwd_plan(p, c->d), Q, K, V, O, lse, workspace, s);
    return heads_fwd_cores(c->dtype, (int)c->d, p, Q, K, V, O, lse, s);
}

extern "C" int emmyb200_attention_heads_bwd(const emmyb200_attention_heads_desc* c, const void* dO, const void* Q, const void* K,
                                            const void* V, const void* O, const float* lse, const int32_t* key_lens, const void* table,
                                            void* dQ, void* dK, void* dV, void* dtable, void* workspace, int64_t workspace_bytes,
                                            void* cuda_stream) {
    using namespace emmy;
    int rc = check_desc(c, true, "attention_heads_bwd");
    if (rc != EMMYB200_OK) return rc;
    const bool has_q = c->batch > 0 && c->heads > 0 && c->seq_q > 0, has_k = c->batch > 0 && c->heads > 0 && c->seq_k > 0;
    if (has_q && (dO == nullptr || Q == nullptr || O == nullptr || lse == nullptr || dQ == nullptr)) return fail(EMMYB200_ERR_ARG, "attention_heads_bwd: null buffer");
    if (has_k && (K == nullptr || V == nullptr || dK == nullptr || dV == nullptr)) return fail(EMMYB200_ERR_ARG, "attention_heads_bwd: null buffer");
    if (c->n_runs && c->heads > 0 && table == nullptr) return fail(EMMYB200_ERR_ARG, "attention_heads_bwd: runs of distances without a table");
    if (c->n_runs == 0 && dtable != nullptr) return fail(EMMYB200_ERR_ARG, "attention_heads_bwd: a table gradient without a table");
    const BwdLayout w = bwd_layout(c);
    if (w.total > 0 && (workspace == nullptr || workspace_bytes < w.total || !aligned(workspace, 256)))
        return fail(EMMYB200_ERR_ARG, "attention_heads_bwd: needs %lld bytes of 256-byte aligned workspace", (long long)w.total);
    if (!has_q && !has_k && dtable == nullptr) return EMMYB200_OK;
    rc = check_sm100();
    if (rc != EMMYB200_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
    const HeadsParams p = make_params(c, key_lens, table);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    HeadsGrads g = {};
    g.d_o = dO; g.q = Q; g.k = K; g.v = V; g.o = O; g.lse = lse; g.dq = dQ; g.dk = dK; g.dv = dV; g.dtable = dtable;
    g.pad_q = (int)w.pad_q;
    g.lse2 = reinterpret_cast<float*>(ws);
    g.delta = reinterpret_cast<float*>(ws + w.delta_at);
    g.run_sums = reinterpret_cast<float*>(ws + w.sums_at);
    g.amax = reinterpret_cast<float*>(ws + w.amax_at);
    const bool tensor_cores = has_q && has_k && heads_bwd_sm100_takes(p, c->dtype, (int)c->d, g);
    const bool norms = tensor_cores && c->dtype == EMMYB200_F16;
    const int cores_rows = 16 * heads_cores_rows(p);
    g.q_tiles = (int)(tensor_cores ? w.parts : (c->seq_q + cores_rows - 1) / cores_rows);
    if (tensor_cores) {
        if (norms) EMMY_CUDA(cudaMemsetAsync(g.amax, 0, 2 * c->batch * c->kv_heads * 4, s));
        rc = norms ? launch_rows16<__half, true>(p, g, (int)c->d, heads_bwd_shift(c->dtype), s)
                   : launch_rows16<__nv_bfloat16, false>(p, g, (int)c->d, heads_bwd_shift(c->dtype), s);
        if (rc != EMMYB200_OK) return rc;
    } else if (has_q) {
        const int64_t blocks = (c->batch * c->heads * w.pad_q + 7) / 8;
        if (blocks >= (1ll << 31)) return fail(EMMYB200_ERR_SHAPE, "attention_heads_bwd: %lld rows exceed the grid limit", (long long)blocks * 8);
        if (c->dtype == EMMYB200_F32) heads_rows_kernel<float><<<(unsigned)blocks, 256, 0, s>>>(p, g, (int)c->d);
        else if (c->dtype == EMMYB200_F16) heads_rows_kernel<__half><<<(unsigned)blocks, 256, 0, s>>>(p, g, (int)c->d);
        else heads_rows_kernel<__nv_bfloat16><<<(unsigned)blocks, 256, 0, s>>>(p, g, (int)c->d);
        rc = launch_status("heads_rows_kernel");
        if (rc != EMMYB200_OK) return rc;
    }
    if (has_q || has_k) {
        rc = tensor_cores ? heads_bwd_sm100(c->dtype, (int)c->d, p, g, s) : heads_bwd_cores(c->dtype, (int)c->d, p, g, s);
        if (rc != EMMYB200_OK) return rc;
    }
    if (dtable != nullptr && c->heads > 0) {
        const int blocks = c->buckets * (int)c->heads;
        if (c->bias_dtype == EMMYB200_F32) heads_dtable_kernel<float><<<blocks, 128, 0, s>>>(p, g);
        else if (c->bias_dtype == EMMYB200_F16) heads_dtable_kernel<__half><<<blocks, 128, 0, s>>>(p, g);
        else heads_dtable_kernel<__nv_bfloat16><<<blocks, 128, 0, s>>>(p, g);
        return launch_status("heads_dtable_kernel");
    }
    return EMMYB200_OK;
}
