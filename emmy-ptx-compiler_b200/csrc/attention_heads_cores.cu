// Attention over heads in fp32 arithmetic on the CUDA cores, forward and backward: fp32 buffers, head sizes the
// tensor-core kernels do not take (32, 96), and buffers that are not aligned for TMA.
//
// 64 x 64 tiles of queries and keys, 256 threads as 16 x 16; operands are widened to fp32 on their way into shared
// memory. Thread (ty, tx) owns rows 4 ty .. 4 ty + 3 and columns tx + 16 c of every product, so operand rows are read as
// 128-bit broadcasts and columns without bank conflicts (rows padded by 4 floats). Probabilities cross to the second
// product through shared memory, stored so that a thread's four rows are one 128-bit load. Sums stay in registers for the
// whole walk. Nothing is added atomically: a block owns its output rows, and the bias gradient goes through per-block
// sums that one last kernel adds up in order.
#include "attention_heads.cuh"

namespace emmy {

constexpr int kCt = kCoresTile;
constexpr int kCThreads = 256;
constexpr int kPRow = kCt + 4;          // pitch of the probability tile

// rows [row0, row0 + 64) of a strided [rows, D] operand, zeros from `limit` on
template <int D, typename T>
__device__ __forceinline__ void cores_stage(float* dst, const T* src, int64_t row_stride, int row0, int limit) {
    for (int e = threadIdx.x; e < kCt * D; e += kCThreads) {
        const int r = e / D, c = e % D;
        dst[r * (D + 4) + c] = row0 + r < limit ? heads_load(src, (int64_t)(row0 + r) * row_stride + c) : 0.0f;
    }
}

// s[r][c] = A[4 ty + r] . B[tx + 16 c]
template <int D>
__device__ __forceinline__ void cores_dot(const float* A, const float* B, int ty, int tx, float (&s)[4][4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[r][c] = 0.0f;
#pragma unroll 4
    for (int k = 0; k < D; k += 4) {
        float4 a[4], b[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) a[r] = *reinterpret_cast<const float4*>(A + (4 * ty + r) * (D + 4) + k);
#pragma unroll
        for (int c = 0; c < 4; ++c) b[c] = *reinterpret_cast<const float4*>(B + (tx + 16 * c) * (D + 4) + k);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                s[r][c] = fmaf(a[r].x, b[c].x, s[r][c]);
                s[r][c] = fmaf(a[r].y, b[c].y, s[r][c]);
                s[r][c] = fmaf(a[r].z, b[c].z, s[r][c]);
                s[r][c] = fmaf(a[r].w, b[c].w, s[r][c]);
            }
    }
}

// acc[r][c] += sum_j W[j][4 ty + r] * B[j][tx + 16 c]
template <int D>
__device__ __forceinline__ void cores_accumulate(const float* W, const float* B, int ty, int tx, float (&acc)[4][D / 16]) {
#pragma unroll 4
    for (int j = 0; j < kCt; ++j) {
        const float4 w = *reinterpret_cast<const float4*>(W + j * kPRow + 4 * ty);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            const float b = B[j * (D + 4) + tx + 16 * c];
            acc[0][c] = fmaf(w.x, b, acc[0][c]);
            acc[1][c] = fmaf(w.y, b, acc[1][c]);
            acc[2][c] = fmaf(w.z, b, acc[2][c]);
            acc[3][c] = fmaf(w.w, b, acc[3][c]);
        }
    }
}

struct CoresBias {          // in shared memory
    int first[kHeadsMaxRuns];
    float value[kHeadsMaxRuns];     // of this block's head, log2 units
    float by_dist[2 * kCt];         // of the current tile, by distance - (smallest distance of the tile)
    int run[2 * kCt];
};

__device__ __forceinline__ void cores_bias_head(CoresBias& cb, const HeadsParams& p, int head) {
    for (int r = threadIdx.x; r < p.n_runs; r += kCThreads) {
        cb.first[r] = p.run_first[r];
        cb.value[r] = heads_run_bias(p, r, head);
    }
}
// the 127 distances of a tile whose smallest is `d0`; the caller synchronises
__device__ __forceinline__ void cores_bias_tile(CoresBias& cb, const HeadsParams& p, int d0) {
    if (threadIdx.x < 2 * kCt) {
        const int r = heads_run_of(cb.first, p.n_runs, d0 + (int)threadIdx.x);
        cb.run[threadIdx.x] = r;
        cb.by_dist[threadIdx.x] = cb.value[r];
    }
}

// Score of (query row i, key j) of a tile in log2 units, -inf where the query does not see the key. i, j: within the tile.
__device__ __forceinline__ float cores_score(const HeadsParams& p, const CoresBias& cb, float dot, int i, int j, int row0, int key0, int offset,
                                             int n_keys) {
    float t = dot * p.scale_log2;
    if (p.n_runs) t += cb.by_dist[j - i + kCt - 1];
    const int key = key0 + j;
    if (key >= n_keys || (p.causal && key > row0 + i + offset)) t = -INFINITY;
    return t;
}

template <int D>
constexpr size_t cores_smem(int operands, int weights) {
    return sizeof(CoresBias) + sizeof(float) * ((size_t)operands * kCt * (D + 4) + (size_t)weights * kCt * kPRow);
}

template <int D, typename T>
__global__ void __launch_bounds__(kCThreads) heads_fwd_cores_kernel(HeadsParams p, const T* __restrict__ Q, const T* __restrict__ K,
                                                                     const T* __restrict__ V, T* __restrict__ O, float* __restrict__ lse) {
    extern __shared__ __align__(16) uint8_t cores_raw[];
    CoresBias& cb = *reinterpret_cast<CoresBias*>(cores_raw);
    float* q_s = reinterpret_cast<float*>(cores_raw + sizeof(CoresBias));
    float* k_s = q_s + kCt * (D + 4);
    float* v_s = k_s + kCt * (D + 4);
    float* w_s = v_s + kCt * (D + 4);
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const int q_tiles = (p.seq_q + kCt - 1) / kCt;
    const int row0 = (int)(blockIdx.x % q_tiles) * kCt;
    const int bh = blockIdx.x / q_tiles, b = bh / p.heads, h = bh % p.heads, hk = h / p.group;
    const int n_keys = heads_key_count(p, b), offset = heads_offset(p, n_keys);
    const T* q_u = Q + b * p.q_s[0] + h * p.q_s[1];
    const T* k_u = K + b * p.k_s[0] + hk * p.k_s[1];
    const T* v_u = V + b * p.v_s[0] + hk * p.v_s[1];

    cores_stage<D>(q_s, q_u, p.q_s[2], row0, p.seq_q);
    if (p.n_runs) cores_bias_head(cb, p, h);
    float m[4], l[4], acc[4][D / 16];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) acc[r][c] = 0.0f;
    }
    const int last_row = min(row0 + kCt, p.seq_q) - 1;
    const int key_end = p.causal ? min(n_keys, last_row + offset + 1) : n_keys;      // keys that some row of the tile sees
    for (int key0 = 0; key0 < key_end; key0 += kCt) {
        __syncthreads();
        cores_stage<D>(k_s, k_u, p.k_s[2], key0, n_keys);
        cores_stage<D>(v_s, v_u, p.v_s[2], key0, n_keys);
        if (p.n_runs) cores_bias_tile(cb, p, key0 - (row0 + kCt - 1 + offset));
        __syncthreads();
        float s[4][4];
        cores_dot<D>(q_s, k_s, ty, tx, s);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                s[r][c] = cores_score(p, cb, s[r][c], 4 * ty + r, tx + 16 * c, row0, key0, offset, n_keys);
                top = fmaxf(top, s[r][c]);
            }
#pragma unroll
            for (int off = 8; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            const float m_new = fmaxf(m[r], top);
            const float ref = m_new == -INFINITY ? 0.0f : m_new;        // nothing seen so far
            const float corr = exp2f(m[r] - ref);
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                s[r][c] = exp2f(s[r][c] - ref);
                sum += s[r][c];
            }
            l[r] = fmaf(l[r], corr, sum);                               // this thread's columns; added up over tx at the end
            m[r] = m_new;
#pragma unroll
            for (int c = 0; c < D / 16; ++c) acc[r][c] *= corr;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
            *reinterpret_cast<float4*>(w_s + (tx + 16 * c) * kPRow + 4 * ty) = make_float4(s[0][c], s[1][c], s[2][c], s[3][c]);
        __syncthreads();
        cores_accumulate<D>(w_s, v_s, ty, tx, acc);
    }
    T* o_u = O + b * p.o_s[0] + h * p.o_s[1];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        float sum = l[r];
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        const int row = row0 + 4 * ty + r;
        if (row >= p.seq_q) continue;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;              // a row that saw nothing: zeros (its sums are zero)
#pragma unroll
        for (int c = 0; c < D / 16; ++c) heads_store(o_u, (int64_t)row * p.o_s[2] + tx + 16 * c, sum == 0.0f ? 0.0f : acc[r][c] * inv);
        if (tx == 0) lse[(int64_t)bh * p.seq_q + row] = sum == 0.0f ? -INFINITY : fmaf(m[r], kLn2, logf(sum));
    }
}

// dK, dV of one key tile of one key head: walks the query tiles of every query head that reads it.
template <int D, typename T>
__global__ void __launch_bounds__(kCThreads) heads_dkv_cores_kernel(HeadsParams p, HeadsGrads g) {
    extern __shared__ __align__(16) uint8_t cores_raw[];
    CoresBias& cb = *reinterpret_cast<CoresBias*>(cores_raw);
    float* k_s = reinterpret_cast<float*>(cores_raw + sizeof(CoresBias));
    float* v_s = k_s + kCt * (D + 4);
    float* q_s = v_s + kCt * (D + 4);
    float* do_s = q_s + kCt * (D + 4);
    float* p_s = do_s + kCt * (D + 4);
    float* ds_s = p_s + kCt * kPRow;
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const int k_tiles = (p.seq_k + kCt - 1) / kCt;
    const int key0 = (int)(blockIdx.x % k_tiles) * kCt;
    const int bk = blockIdx.x / k_tiles, b = bk / p.kv_heads, hk = bk % p.kv_heads;
    const int n_keys = heads_key_count(p, b), offset = heads_offset(p, n_keys);
    float dk[4][D / 16], dv[4][D / 16];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < D / 16; ++c) dk[r][c] = dv[r][c] = 0.0f;
    if (key0 < n_keys) {
        cores_stage<D>(k_s, static_cast<const T*>(g.k) + b * p.k_s[0] + hk * p.k_s[1], p.k_s[2], key0, n_keys);
        cores_stage<D>(v_s, static_cast<const T*>(g.v) + b * p.v_s[0] + hk * p.v_s[1], p.v_s[2], key0, n_keys);
        const int first_row = p.causal ? max(0, key0 - offset) : 0;         // rows before it see none of the tile's keys
        for (int gi = 0; gi < p.group; ++gi) {
            const int h = hk * p.group + gi;
            const int64_t rows_at = ((int64_t)b * p.heads + h) * g.pad_q;
            const T* q_u = static_cast<const T*>(g.q) + b * p.q_s[0] + h * p.q_s[1];
            const T* do_u = static_cast<const T*>(g.d_o) + b * p.do_s[0] + h * p.do_s[1];
            __syncthreads();
            if (p.n_runs) cores_bias_head(cb, p, h);
            for (int row0 = first_row / kCt * kCt; row0 < p.seq_q; row0 += kCt) {
                __syncthreads();
                cores_stage<D>(q_s, q_u, p.q_s[2], row0, p.seq_q);
                cores_stage<D>(do_s, do_u, p.do_s[2], row0, p.seq_q);
                if (p.n_runs) cores_bias_tile(cb, p, key0 - (row0 + kCt - 1 + offset));
                __syncthreads();
                float s[4][4], dp[4][4];
                cores_dot<D>(q_s, k_s, ty, tx, s);
                cores_dot<D>(do_s, v_s, ty, tx, dp);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = row0 + 4 * ty + r;                      // below pad_q
                    const float lse2 = g.lse2[rows_at + row], delta = g.delta[rows_at + row];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float t = cores_score(p, cb, s[r][c], 4 * ty + r, tx + 16 * c, row0, key0, offset, n_keys);
                        const float pr = exp2f(t + lse2);
                        p_s[(4 * ty + r) * kPRow + tx + 16 * c] = pr;
                        ds_s[(4 * ty + r) * kPRow + tx + 16 * c] = pr * (dp[r][c] + delta);
                    }
                }
                __syncthreads();
                cores_accumulate<D>(p_s, do_s, ty, tx, dv);
                cores_accumulate<D>(ds_s, q_s, ty, tx, dk);
            }
        }
    }
    T* dk_u = static_cast<T*>(g.dk) + b * p.dk_s[0] + hk * p.dk_s[1];
    T* dv_u = static_cast<T*>(g.dv) + b * p.dv_s[0] + hk * p.dv_s[1];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int key = key0 + 4 * ty + r;
        if (key >= p.seq_k) continue;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            heads_store(dk_u, (int64_t)key * p.dk_s[2] + tx + 16 * c, dk[r][c] * p.scale);
            heads_store(dv_u, (int64_t)key * p.dv_s[2] + tx + 16 * c, dv[r][c]);
        }
    }
}

// dQ of one query tile, and this tile's part of the bias gradient: the 127 diagonals of every 64 x 64 tile of dS are added
// up one thread per distance, distances of one run by one thread, in a fixed order.
template <int D, typename T>
__global__ void __launch_bounds__(kCThreads) heads_dq_cores_kernel(HeadsParams p, HeadsGrads g) {
    extern __shared__ __align__(16) uint8_t cores_raw[];
    CoresBias& cb = *reinterpret_cast<CoresBias*>(cores_raw);
    float* k_s = reinterpret_cast<float*>(cores_raw + sizeof(CoresBias));
    float* v_s = k_s + kCt * (D + 4);
    float* q_s = v_s + kCt * (D + 4);
    float* do_s = q_s + kCt * (D + 4);
    float* ds_s = do_s + kCt * (D + 4);
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const int q_tiles = (p.seq_q + kCt - 1) / kCt;
    const int qt = blockIdx.x % q_tiles, row0 = qt * kCt;
    const int bh = blockIdx.x / q_tiles, b = bh / p.heads, h = bh % p.heads, hk = h / p.group;
    const int n_keys = heads_key_count(p, b), offset = heads_offset(p, n_keys);
    const T* k_u = static_cast<const T*>(g.k) + b * p.k_s[0] + hk * p.k_s[1];
    const T* v_u = static_cast<const T*>(g.v) + b * p.v_s[0] + hk * p.v_s[1];
    cores_stage<D>(q_s, static_cast<const T*>(g.q) + b * p.q_s[0] + h * p.q_s[1], p.q_s[2], row0, p.seq_q);
    cores_stage<D>(do_s, static_cast<const T*>(g.d_o) + b * p.do_s[0] + h * p.do_s[1], p.do_s[2], row0, p.seq_q);
    if (p.n_runs) cores_bias_head(cb, p, h);
    const bool want_bias = p.n_runs && g.dtable != nullptr;
    float run_sum = 0.0f;                                                   // thread r: of run r
    float lse2[4], delta[4], dq[4][D / 16];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        lse2[r] = g.lse2[(int64_t)bh * g.pad_q + row0 + 4 * ty + r];
        delta[r] = g.delta[(int64_t)bh * g.pad_q + row0 + 4 * ty + r];
#pragma unroll
        for (int c = 0; c < D / 16; ++c) dq[r][c] = 0.0f;
    }
    const int last_row = min(row0 + kCt, p.seq_q) - 1;
    const int key_end = p.causal ? min(n_keys, last_row + offset + 1) : n_keys;
    for (int key0 = 0; key0 < key_end; key0 += kCt) {
        __syncthreads();
        cores_stage<D>(k_s, k_u, p.k_s[2], key0, n_keys);
        cores_stage<D>(v_s, v_u, p.v_s[2], key0, n_keys);
        if (p.n_runs) cores_bias_tile(cb, p, key0 - (row0 + kCt - 1 + offset));
        __syncthreads();
        float s[4][4], dp[4][4];
        cores_dot<D>(q_s, k_s, ty, tx, s);
        cores_dot<D>(do_s, v_s, ty, tx, dp);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float t = cores_score(p, cb, s[r][c], 4 * ty + r, tx + 16 * c, row0, key0, offset, n_keys);
                s[r][c] = exp2f(t + lse2[r]) * (dp[r][c] + delta[r]);
            }
#pragma unroll
        for (int c = 0; c < 4; ++c)
            *reinterpret_cast<float4*>(ds_s + (tx + 16 * c) * kPRow + 4 * ty) = make_float4(s[0][c], s[1][c], s[2][c], s[3][c]);
        __syncthreads();
        cores_accumulate<D>(ds_s, k_s, ty, tx, dq);
        if (want_bias) {
            if (threadIdx.x < 2 * kCt - 1) {                                // distance index t = j - i + 63
                const int t = threadIdx.x;
                float sum = 0.0f;
                for (int i = max(0, kCt - 1 - t); i < min(kCt, 2 * kCt - 1 - t); ++i) sum += ds_s[(i + t - (kCt - 1)) * kPRow + i];
                cb.by_dist[t] = sum;                                        // the tile's biases have been used
            }
            __syncthreads();
            if ((int)threadIdx.x < p.n_runs) {
                const int r = threadIdx.x, d0 = key0 - (row0 + kCt - 1 + offset);
                const int from = r == 0 ? 0 : max(0, cb.first[r] - d0);
                const int to = r + 1 == p.n_runs ? 2 * kCt - 1 : min(2 * kCt - 1, cb.first[r + 1] - d0);
                for (int t = from; t < to; ++t) run_sum += cb.by_dist[t];
            }
        }
    }
    T* dq_u = static_cast<T*>(g.dq) + b * p.dq_s[0] + h * p.dq_s[1];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int row = row0 + 4 * ty + r;
        if (row >= p.seq_q) continue;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) heads_store(dq_u, (int64_t)row * p.dq_s[2] + tx + 16 * c, dq[r][c] * p.scale);
    }
    if (want_bias && (int)threadIdx.x < p.n_runs) g.run_sums[((int64_t)bh * g.q_tiles + qt) * p.n_runs + threadIdx.x] = run_sum;
}

template <int D, typename T>
static int fwd_launch(const HeadsParams& p, const void* Q, const void* K, const void* V, void* O, float* lse, cudaStream_t s) {
    const int64_t blocks = (int64_t)((p.seq_q + kCt - 1) / kCt) * p.batch * p.heads;
    if (blocks == 0) return EMMYB200_OK;
    if (blocks >= (1ll << 31)) return fail(EMMYB200_ERR_SHAPE, "attention_heads_fwd: %lld tiles exceed the grid limit", (long long)blocks);
    constexpr size_t smem = cores_smem<D>(3, 1);
    auto kernel = heads_fwd_cores_kernel<D, T>;
    EMMY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    kernel<<<(unsigned)blocks, kCThreads, smem, s>>>(p, static_cast<const T*>(Q), static_cast<const T*>(K), static_cast<const T*>(V), static_cast<T*>(O), lse);
    return launch_status("heads_fwd_cores_kernel");
}

template <int D, typename T>
static int bwd_launch(const HeadsParams& p, const HeadsGrads& g, cudaStream_t s) {
    const int64_t kv_blocks = (int64_t)((p.seq_k + kCt - 1) / kCt) * p.batch * p.kv_heads;
    const int64_t q_blocks = (int64_t)((p.seq_q + kCt - 1) / kCt) * p.batch * p.heads;
    if (kv_blocks >= (1ll << 31) || q_blocks >= (1ll << 31)) return fail(EMMYB200_ERR_SHAPE, "attention_heads_bwd: the tiles exceed the grid limit");
    if (kv_blocks > 0) {
        constexpr size_t smem = cores_smem<D>(4, 2);
        auto kernel = heads_dkv_cores_kernel<D, T>;
        EMMY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        kernel<<<(unsigned)kv_blocks, kCThreads, smem, s>>>(p, g);
        int rc = launch_status("heads_dkv_cores_kernel");
        if (rc != EMMYB200_OK) return rc;
    }
    if (q_blocks > 0) {
        constexpr size_t smem = cores_smem<D>(4, 1);
        auto kernel = heads_dq_cores_kernel<D, T>;
        EMMY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        kernel<<<(unsigned)q_blocks, kCThreads, smem, s>>>(p, g);
        return launch_status("heads_dq_cores_kernel");
    }
    return EMMYB200_OK;
}

template <typename T>
static int fwd_by_d(int d, const HeadsParams& p, const void* Q, const void* K, const void* V, void* O, float* lse, cudaStream_t s) {
    switch (d) {
        case 32: return fwd_launch<32, T>(p, Q, K, V, O, lse, s);
        case 64: return fwd_launch<64, T>(p, Q, K, V, O, lse, s);
        case 96: return fwd_launch<96, T>(p, Q, K, V, O, lse, s);
        default: return fwd_launch<128, T>(p, Q, K, V, O, lse, s);
    }
}
template <typename T>
static int bwd_by_d(int d, const HeadsParams& p, const HeadsGrads& g, cudaStream_t s) {
    switch (d) {
        case 32: return bwd_launch<32, T>(p, g, s);
        case 64: return bwd_launch<64, T>(p, g, s);
        case 96: return bwd_launch<96, T>(p, g, s);
        default: return bwd_launch<128, T>(p, g, s);
    }
}

int heads_fwd_cores(int dtype, int d, const HeadsParams& p, const void* Q, const void* K, const void* V, void* O, float* lse, cudaStream_t s) {
    if (dtype == EMMYB200_F32) return fwd_by_d<float>(d, p, Q, K, V, O, lse, s);
    if (dtype == EMMYB200_F16) return fwd_by_d<__half>(d, p, Q, K, V, O, lse, s);
    return fwd_by_d<__nv_bfloat16>(d, p, Q, K, V, O, lse, s);
}
int heads_bwd_cores(int dtype, int d, const HeadsParams& p, const HeadsGrads& g, cudaStream_t s) {
    if (dtype == EMMYB200_F32) return bwd_by_d<float>(d, p, g, s);
    if (dtype == EMMYB200_F16) return bwd_by_d<__half>(d, p, g, s);
    return bwd_by_d<__nv_bfloat16>(d, p, g, s);
}

}  // namespace emmy
