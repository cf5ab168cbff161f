// Attention over heads in fp32 arithmetic on the CUDA cores, forward and backward: fp32 buffers, head sizes the
// tensor-core kernels do not take (32, 96), and buffers that are not aligned for TMA.
//
// A block of 256 threads (16 x 16) owns 16 R rows (queries; keys in dkv) and walks the other side 64 at a time; operands are widened
// to fp32 on their way into shared memory. Thread (ty, tx) owns R rows and columns tx + 16 c of every product, so operand rows are
// read as 128-bit broadcasts and columns without bank conflicts (rows padded by 4 floats). Probabilities cross to the second
// product through shared memory, stored so that a thread's rows are one load. Sums stay in registers for the whole walk. Nothing
// is added atomically: a block owns its output rows, and the bias gradient goes through per-block sums that one last kernel adds up in
// order. R = 4 makes the best of every load (16 multiply-adds per 8 loads); R = 1 makes four times as many blocks of a quarter of the
// work, which is faster while R = 4 would leave SMs idle (8 units of 128 x 128 x 64: forward 34 -> 13 us, dkv and dq 48 + 46 -> 18 us together).
#include "attention_heads.cuh"

namespace emmy {

constexpr int kCt = kCoresTile;         // tile of the side that is walked
constexpr int kCThreads = 256;

// `rows` rows from row0 on of a strided [rows, D] operand, zeros from `limit` on. VEC: 16-byte aligned rows.
template <int D, int ROWS, bool VEC, typename T>
__device__ __forceinline__ void cores_stage(float* dst, const T* src, int64_t row_stride, int row0, int limit) {
    if constexpr (VEC) {
        constexpr int kElems = 16 / sizeof(T), kPerRow = D / kElems, kLoads = (ROWS * kPerRow + kCThreads - 1) / kCThreads;
        uint4 v[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int e = threadIdx.x + i * kCThreads, r = e / kPerRow, c = e % kPerRow;
            v[i] = make_uint4(0, 0, 0, 0);
            if (r < ROWS && row0 + r < limit) v[i] = __ldg(reinterpret_cast<const uint4*>(src + (row0 + r) * row_stride) + c);
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int e = threadIdx.x + i * kCThreads, r = e / kPerRow, c = e % kPerRow;
            const T* x = reinterpret_cast<const T*>(&v[i]);
            if (r < ROWS)
#pragma unroll
                for (int k = 0; k < kElems; k += 4)
                    *reinterpret_cast<float4*>(dst + r * (D + 4) + c * kElems + k) =
                        make_float4(heads_load(x, k), heads_load(x, k + 1), heads_load(x, k + 2), heads_load(x, k + 3));
        }
    } else {
#pragma unroll 4
        for (int e = threadIdx.x; e < ROWS * D; e += kCThreads) {
            const int r = e / D, c = e % D;
            dst[r * (D + 4) + c] = row0 + r < limit ? heads_load(src, (row0 + r) * row_stride + c) : 0.0f;
        }
    }
}

// s[r][c] = A[RA ty + r] . B[tx + 16 c]
template <int D, int RA, int CB>
__device__ __forceinline__ void cores_dot(const float* A, const float* B, int ty, int tx, float (&s)[RA][CB]) {
#pragma unroll
    for (int r = 0; r < RA; ++r)
#pragma unroll
        for (int c = 0; c < CB; ++c) s[r][c] = 0.0f;
#pragma unroll 4
    for (int k = 0; k < D; k += 4) {
        float4 a[RA], b[CB];
#pragma unroll
        for (int r = 0; r < RA; ++r) a[r] = *reinterpret_cast<const float4*>(A + (RA * ty + r) * (D + 4) + k);
#pragma unroll
        for (int c = 0; c < CB; ++c) b[c] = *reinterpret_cast<const float4*>(B + (tx + 16 * c) * (D + 4) + k);
#pragma unroll
        for (int r = 0; r < RA; ++r)
#pragma unroll
            for (int c = 0; c < CB; ++c) {
                s[r][c] = fmaf(a[r].x, b[c].x, s[r][c]);
                s[r][c] = fmaf(a[r].y, b[c].y, s[r][c]);
                s[r][c] = fmaf(a[r].z, b[c].z, s[r][c]);
                s[r][c] = fmaf(a[r].w, b[c].w, s[r][c]);
            }
    }
}

// R values of a row of weights: one load
template <int R>
__device__ __forceinline__ void load_weights(const float* at, float (&w)[R]) {
    if constexpr (R == 4) {
        const float4 v = *reinterpret_cast<const float4*>(at);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else {
        w[0] = *at;
    }
}
// acc[r][c] += sum_j W[j][R ty + r] * B[j][tx + 16 c] over 64 j
template <int D, int R>
__device__ __forceinline__ void cores_accumulate(const float* W, const float* B, int ty, int tx, float (&acc)[R][D / 16]) {
    constexpr int kPitch = 16 * R + 4;
#pragma unroll 8
    for (int j = 0; j < kCt; ++j) {
        float w[R];
        load_weights<R>(W + j * kPitch + R * ty, w);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            const float b = B[j * (D + 4) + tx + 16 * c];
#pragma unroll
            for (int r = 0; r < R; ++r) acc[r][c] = fmaf(w[r], b, acc[r][c]);
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
// the distances of a tile (at most 127) whose smallest is `d0`; the caller synchronises
__device__ __forceinline__ void cores_bias_tile(CoresBias& cb, const HeadsParams& p, int d0) {
    if (threadIdx.x < 2 * kCt) {
        const int r = heads_run_of(cb.first, p.n_runs, d0 + (int)threadIdx.x);
        cb.run[threadIdx.x] = r;
        cb.by_dist[threadIdx.x] = cb.value[r];
    }
}

// Score of (query row i, key j) of a tile in log2 units, -inf where the query does not see the key. i, j: within the tile.
template <int QT>       // query rows of the tile
__device__ __forceinline__ float cores_score(const HeadsParams& p, const CoresBias& cb, float dot, int i, int j, int row0, int key0, int offset,
                                             int n_keys) {
    float t = dot * p.scale_log2;
    if (p.n_runs) t += cb.by_dist[j - i + QT - 1];
    const int key = key0 + j;
    if (key >= n_keys || (p.causal && key > row0 + i + offset)) t = -INFINITY;
    return t;
}

// `walked` operands of 64 rows, `owned` ones of 16 R rows, `weights` tiles of 64 x 16 R
template <int D, int R>
constexpr size_t cores_smem(int walked, int owned, int weights) {
    return sizeof(CoresBias) + sizeof(float) * ((size_t)(walked * kCt + owned * 16 * R) * (D + 4) + (size_t)weights * kCt * (16 * R + 4));
}

template <int D, int R, bool VEC, typename T>
__global__ void __launch_bounds__(kCThreads) heads_fwd_cores_kernel(HeadsParams p, const T* __restrict__ Q, const T* __restrict__ K,
                                                                     const T* __restrict__ V, T* __restrict__ O, float* __restrict__ lse) {
    constexpr int QT = 16 * R, kPitch = QT + 4;
    extern __shared__ __align__(16) uint8_t cores_raw[];
    CoresBias& cb = *reinterpret_cast<CoresBias*>(cores_raw);
    float* q_s = reinterpret_cast<float*>(cores_raw + sizeof(CoresBias));
    float* k_s = q_s + QT * (D + 4);
    float* v_s = k_s + kCt * (D + 4);
    float* w_s = v_s + kCt * (D + 4);
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const int q_tiles = (p.seq_q + QT - 1) / QT;
    const int row0 = (int)(blockIdx.x % q_tiles) * QT;
    const int bh = blockIdx.x / q_tiles, b = bh / p.heads, h = bh % p.heads, hk = h / p.group;
    const int n_keys = heads_key_count(p, b), offset = heads_offset(p, n_keys);
    const T* q_u = Q + b * p.q_s[0] + h * p.q_s[1];
    const T* k_u = K + b * p.k_s[0] + hk * p.k_s[1];
    const T* v_u = V + b * p.v_s[0] + hk * p.v_s[1];

    cores_stage<D, QT, VEC>(q_s, q_u, p.q_s[2], row0, p.seq_q);
    if (p.n_runs) cores_bias_head(cb, p, h);
    float m[R], l[R], acc[R][D / 16];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) acc[r][c] = 0.0f;
    }
    const int last_row = min(row0 + QT, p.seq_q) - 1;
    const int key_end = p.causal ? min(n_keys, last_row + offset + 1) : n_keys;      // keys that some row of the tile sees
    for (int key0 = 0; key0 < key_end; key0 += kCt) {
        __syncthreads();
        cores_stage<D, kCt, VEC>(k_s, k_u, p.k_s[2], key0, n_keys);
        cores_stage<D, kCt, VEC>(v_s, v_u, p.v_s[2], key0, n_keys);
        if (p.n_runs) cores_bias_tile(cb, p, key0 - (row0 + QT - 1 + offset));
        __syncthreads();
        float s[R][4];
        cores_dot<D>(q_s, k_s, ty, tx, s);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                s[r][c] = cores_score<QT>(p, cb, s[r][c], R * ty + r, tx + 16 * c, row0, key0, offset, n_keys);
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
#pragma unroll
            for (int r = 0; r < R; ++r) w_s[(tx + 16 * c) * kPitch + R * ty + r] = s[r][c];
        __syncthreads();
        cores_accumulate<D, R>(w_s, v_s, ty, tx, acc);
    }
    T* o_u = O + b * p.o_s[0] + h * p.o_s[1];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float sum = l[r];
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        const int row = row0 + R * ty + r;
        if (row >= p.seq_q) continue;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;              // a row that saw nothing: zeros (its sums are zero)
#pragma unroll
        for (int c = 0; c < D / 16; ++c) heads_store(o_u, (int64_t)row * p.o_s[2] + tx + 16 * c, sum == 0.0f ? 0.0f : acc[r][c] * inv);
        if (tx == 0) lse[(int64_t)bh * p.seq_q + row] = sum == 0.0f ? -INFINITY : fmaf(m[r], kLn2, logf(sum));
    }
}

// dK, dV of one key tile of one key head: walks the query tiles of every query head that reads it.
template <int D, int R, bool VEC, typename T>
__device__ __forceinline__ void cores_dkv_block(const HeadsParams& p, const HeadsGrads& g, uint8_t* cores_raw, int block) {
    constexpr int KT = 16 * R, kPitch = KT + 4;
    CoresBias& cb = *reinterpret_cast<CoresBias*>(cores_raw);
    float* k_s = reinterpret_cast<float*>(cores_raw + sizeof(CoresBias));
    float* v_s = k_s + KT * (D + 4);
    float* q_s = v_s + KT * (D + 4);
    float* do_s = q_s + kCt * (D + 4);
    float* p_s = do_s + kCt * (D + 4);
    float* ds_s = p_s + kCt * kPitch;
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const int k_tiles = (p.seq_k + KT - 1) / KT;
    const int key0 = block % k_tiles * KT;
    const int bk = block / k_tiles, b = bk / p.kv_heads, hk = bk % p.kv_heads;
    const int n_keys = heads_key_count(p, b), offset = heads_offset(p, n_keys);
    float dk[R][D / 16], dv[R][D / 16];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < D / 16; ++c) dk[r][c] = dv[r][c] = 0.0f;
    if (key0 < n_keys) {
        cores_stage<D, KT, VEC>(k_s, static_cast<const T*>(g.k) + b * p.k_s[0] + hk * p.k_s[1], p.k_s[2], key0, n_keys);
        cores_stage<D, KT, VEC>(v_s, static_cast<const T*>(g.v) + b * p.v_s[0] + hk * p.v_s[1], p.v_s[2], key0, n_keys);
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
                float lse2[4], delta[4];                                    // rows below pad_q
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    lse2[r] = g.lse2[rows_at + row0 + 4 * ty + r];
                    delta[r] = g.delta[rows_at + row0 + 4 * ty + r];
                }
                cores_stage<D, kCt, VEC>(q_s, q_u, p.q_s[2], row0, p.seq_q);
                cores_stage<D, kCt, VEC>(do_s, do_u, p.do_s[2], row0, p.seq_q);
                if (p.n_runs) cores_bias_tile(cb, p, key0 - (row0 + kCt - 1 + offset));
                __syncthreads();
                float s[4][R], dp[4][R];
                cores_dot<D>(q_s, k_s, ty, tx, s);
                cores_dot<D>(do_s, v_s, ty, tx, dp);
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int c = 0; c < R; ++c) {
                        const float t = cores_score<kCt>(p, cb, s[r][c], 4 * ty + r, tx + 16 * c, row0, key0, offset, n_keys);
                        const float pr = exp2f(t + lse2[r]);
                        p_s[(4 * ty + r) * kPitch + tx + 16 * c] = pr;
                        ds_s[(4 * ty + r) * kPitch + tx + 16 * c] = pr * (dp[r][c] + delta[r]);
                    }
                __syncthreads();
                cores_accumulate<D, R>(p_s, do_s, ty, tx, dv);
                cores_accumulate<D, R>(ds_s, q_s, ty, tx, dk);
            }
        }
    }
    T* dk_u = static_cast<T*>(g.dk) + b * p.dk_s[0] + hk * p.dk_s[1];
    T* dv_u = static_cast<T*>(g.dv) + b * p.dv_s[0] + hk * p.dv_s[1];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int key = key0 + R * ty + r;
        if (key >= p.seq_k) continue;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            heads_store(dk_u, (int64_t)key * p.dk_s[2] + tx + 16 * c, dk[r][c] * p.scale);
            heads_store(dv_u, (int64_t)key * p.dv_s[2] + tx + 16 * c, dv[r][c]);
        }
    }
}

// dQ of one query tile, and this tile's part of the bias gradient: the diagonals of every tile of dS are added
// up one thread per distance, distances of one run by one thread, in a fixed order.
template <int D, int R, bool VEC, typename T>
__device__ __forceinline__ void cores_dq_block(const HeadsParams& p, const HeadsGrads& g, uint8_t* cores_raw, int block) {
    constexpr int QT = 16 * R, kPitch = QT + 4, kDists = QT + kCt - 1;
    CoresBias& cb = *reinterpret_cast<CoresBias*>(cores_raw);
    float* k_s = reinterpret_cast<float*>(cores_raw + sizeof(CoresBias));
    float* v_s = k_s + kCt * (D + 4);
    float* q_s = v_s + kCt * (D + 4);
    float* do_s = q_s + QT * (D + 4);
    float* ds_s = do_s + QT * (D + 4);
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const int q_tiles = (p.seq_q + QT - 1) / QT;
    const int qt = block % q_tiles, row0 = qt * QT;
    const int bh = block / q_tiles, b = bh / p.heads, h = bh % p.heads, hk = h / p.group;
    const int n_keys = heads_key_count(p, b), offset = heads_offset(p, n_keys);
    const T* k_u = static_cast<const T*>(g.k) + b * p.k_s[0] + hk * p.k_s[1];
    const T* v_u = static_cast<const T*>(g.v) + b * p.v_s[0] + hk * p.v_s[1];
    cores_stage<D, QT, VEC>(q_s, static_cast<const T*>(g.q) + b * p.q_s[0] + h * p.q_s[1], p.q_s[2], row0, p.seq_q);
    cores_stage<D, QT, VEC>(do_s, static_cast<const T*>(g.d_o) + b * p.do_s[0] + h * p.do_s[1], p.do_s[2], row0, p.seq_q);
    if (p.n_runs) cores_bias_head(cb, p, h);
    const bool want_bias = p.n_runs && g.dtable != nullptr;
    float run_sum = 0.0f;                                                   // thread r: of run r
    float lse2[R], delta[R], dq[R][D / 16];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        lse2[r] = g.lse2[(int64_t)bh * g.pad_q + row0 + R * ty + r];
        delta[r] = g.delta[(int64_t)bh * g.pad_q + row0 + R * ty + r];
#pragma unroll
        for (int c = 0; c < D / 16; ++c) dq[r][c] = 0.0f;
    }
    const int last_row = min(row0 + QT, p.seq_q) - 1;
    const int key_end = p.causal ? min(n_keys, last_row + offset + 1) : n_keys;
    for (int key0 = 0; key0 < key_end; key0 += kCt) {
        __syncthreads();
        cores_stage<D, kCt, VEC>(k_s, k_u, p.k_s[2], key0, n_keys);
        cores_stage<D, kCt, VEC>(v_s, v_u, p.v_s[2], key0, n_keys);
        const int d0 = key0 - (row0 + QT - 1 + offset);
        if (p.n_runs) cores_bias_tile(cb, p, d0);
        __syncthreads();
        float s[R][4], dp[R][4];
        cores_dot<D>(q_s, k_s, ty, tx, s);
        cores_dot<D>(do_s, v_s, ty, tx, dp);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float t = cores_score<QT>(p, cb, s[r][c], R * ty + r, tx + 16 * c, row0, key0, offset, n_keys);
                ds_s[(tx + 16 * c) * kPitch + R * ty + r] = exp2f(t + lse2[r]) * (dp[r][c] + delta[r]);
            }
        __syncthreads();
        cores_accumulate<D, R>(ds_s, k_s, ty, tx, dq);
        if (want_bias) {
            if (threadIdx.x < kDists) {                                     // distance index t = j - i + QT - 1
                const int t = threadIdx.x;
                float sum = 0.0f;
#pragma unroll 8
                for (int i = max(0, QT - 1 - t); i < min(QT, kDists - t); ++i) sum += ds_s[(i + t - (QT - 1)) * kPitch + i];
                cb.by_dist[t] = sum;                                        // the tile's biases have been used
            }
            __syncthreads();
            if ((int)threadIdx.x < p.n_runs) {
                const int r = threadIdx.x;
                const int from = r == 0 ? 0 : max(0, cb.first[r] - d0);
                const int to = r + 1 == p.n_runs ? kDists : min(kDists, cb.first[r + 1] - d0);
#pragma unroll 4
                for (int t = from; t < to; ++t) run_sum += cb.by_dist[t];
            }
        }
    }
    T* dq_u = static_cast<T*>(g.dq) + b * p.dq_s[0] + h * p.dq_s[1];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = row0 + R * ty + r;
        if (row >= p.seq_q) continue;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) heads_store(dq_u, (int64_t)row * p.dq_s[2] + tx + 16 * c, dq[r][c] * p.scale);
    }
    if (want_bias && (int)threadIdx.x < p.n_runs) g.run_sums[((int64_t)bh * g.q_tiles + qt) * p.n_runs + threadIdx.x] = run_sum;
}

// Both in one launch, so that neither waits for the other's last blocks.
template <int D, int R, bool VEC, typename T>
__global__ void __launch_bounds__(kCThreads) heads_bwd_cores_kernel(HeadsParams p, HeadsGrads g, int dkv_blocks) {
    extern __shared__ __align__(16) uint8_t cores_raw[];
    if ((int)blockIdx.x < dkv_blocks) cores_dkv_block<D, R, VEC, T>(p, g, cores_raw, blockIdx.x);
    else cores_dq_block<D, R, VEC, T>(p, g, cores_raw, blockIdx.x - dkv_blocks);
}

// 16-byte accesses: aligned bases, and strides in whole 16 bytes wherever they are used.
template <typename T>
static bool vec_ok(const void* base, const int64_t* s, int64_t batch, int64_t heads, int64_t rows) {
    constexpr int64_t kElems = 16 / sizeof(T);
    return aligned(base, 16) && (batch <= 1 || s[0] % kElems == 0) && (heads <= 1 || s[1] % kElems == 0) && (rows <= 1 || s[2] % kElems == 0);
}

template <int D, int R, bool VEC, typename T>
static int fwd_launch(const HeadsParams& p, const void* Q, const void* K, const void* V, void* O, float* lse, cudaStream_t s) {
    const int64_t blocks = (int64_t)((p.seq_q + 16 * R - 1) / (16 * R)) * p.batch * p.heads;
    if (blocks == 0) return EMMYB200_OK;
    if (blocks >= (1ll << 31)) return fail(EMMYB200_ERR_SHAPE, "attention_heads_fwd: %lld tiles exceed the grid limit", (long long)blocks);
    constexpr size_t smem = cores_smem<D, R>(2, 1, 1);
    auto kernel = heads_fwd_cores_kernel<D, R, VEC, T>;
    EMMY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    kernel<<<(unsigned)blocks, kCThreads, smem, s>>>(p, static_cast<const T*>(Q), static_cast<const T*>(K), static_cast<const T*>(V), static_cast<T*>(O), lse);
    return launch_status("heads_fwd_cores_kernel");
}

template <int D, int R, bool VEC, typename T>
static int bwd_launch(const HeadsParams& p, const HeadsGrads& grads, cudaStream_t s) {
    const int64_t q_tiles = (p.seq_q + 16 * R - 1) / (16 * R);
    const int64_t kv_blocks = (int64_t)((p.seq_k + 16 * R - 1) / (16 * R)) * p.batch * p.kv_heads, q_blocks = q_tiles * p.batch * p.heads;
    if (kv_blocks + q_blocks >= (1ll << 31)) return fail(EMMYB200_ERR_SHAPE, "attention_heads_bwd: the tiles exceed the grid limit");
    constexpr size_t dkv_smem = cores_smem<D, R>(2, 2, 2), dq_smem = cores_smem<D, R>(2, 2, 1), smem = dkv_smem > dq_smem ? dkv_smem : dq_smem;
    auto kernel = heads_bwd_cores_kernel<D, R, VEC, T>;
    EMMY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    kernel<<<(unsigned)(kv_blocks + q_blocks), kCThreads, smem, s>>>(p, grads, (int)kv_blocks);
    return launch_status("heads_bwd_cores_kernel");
}

// Rows per thread: 4 once that fills the SMs.
int heads_cores_rows(const HeadsParams& p) {
    const int64_t q_blocks = (int64_t)((p.seq_q + 63) / 64) * p.batch * p.heads;
    return q_blocks >= sm_count() ? 4 : 1;
}

template <int D, typename T>
static int fwd_pick(const HeadsParams& p, const void* Q, const void* K, const void* V, void* O, float* lse, cudaStream_t s) {
    const bool vec = vec_ok<T>(Q, p.q_s, p.batch, p.heads, p.seq_q) && vec_ok<T>(K, p.k_s, p.batch, p.kv_heads, p.seq_k) && vec_ok<T>(V, p.v_s, p.batch, p.kv_heads, p.seq_k);
    if (heads_cores_rows(p) == 4) return vec ? fwd_launch<D, 4, true, T>(p, Q, K, V, O, lse, s) : fwd_launch<D, 4, false, T>(p, Q, K, V, O, lse, s);
    return vec ? fwd_launch<D, 1, true, T>(p, Q, K, V, O, lse, s) : fwd_launch<D, 1, false, T>(p, Q, K, V, O, lse, s);
}
template <int D, typename T>
static int bwd_pick(const HeadsParams& p, const HeadsGrads& g, cudaStream_t s) {
    const bool vec = vec_ok<T>(g.q, p.q_s, p.batch, p.heads, p.seq_q) && vec_ok<T>(g.d_o, p.do_s, p.batch, p.heads, p.seq_q) &&
                     vec_ok<T>(g.k, p.k_s, p.batch, p.kv_heads, p.seq_k) && vec_ok<T>(g.v, p.v_s, p.batch, p.kv_heads, p.seq_k);
    if (heads_cores_rows(p) == 4) return vec ? bwd_launch<D, 4, true, T>(p, g, s) : bwd_launch<D, 4, false, T>(p, g, s);
    return vec ? bwd_launch<D, 1, true, T>(p, g, s) : bwd_launch<D, 1, false, T>(p, g, s);
}

template <typename T>
static int fwd_by_d(int d, const HeadsParams& p, const void* Q, const void* K, const void* V, void* O, float* lse, cudaStream_t s) {
    switch (d) {
        case 32: return fwd_pick<32, T>(p, Q, K, V, O, lse, s);
        case 64: return fwd_pick<64, T>(p, Q, K, V, O, lse, s);
        case 96: return fwd_pick<96, T>(p, Q, K, V, O, lse, s);
        default: return fwd_pick<128, T>(p, Q, K, V, O, lse, s);
    }
}
template <typename T>
static int bwd_by_d(int d, const HeadsParams& p, const HeadsGrads& g, cudaStream_t s) {
    switch (d) {
        case 32: return bwd_pick<32, T>(p, g, s);
        case 64: return bwd_pick<64, T>(p, g, s);
        case 96: return bwd_pick<96, T>(p, g, s);
        default: return bwd_pick<128, T>(p, g, s);
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
