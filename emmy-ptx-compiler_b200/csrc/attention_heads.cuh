// What the kernels of attention over heads (forward with log-sum-exp, backward, relative position bias) share: the launch
// parameters, where a query stands among the keys, the bias by runs of distance, and the layout of the backward pass's
// workspace.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"

namespace emmy {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kMaskedBias = -1e30f;           // a table entry at or below it masks its pairs
constexpr int kHeadsMaxRuns = EMMYB200_HEADS_MAX_RUNS;

struct HeadsParams {
    int batch, heads, kv_heads, group, seq_q, seq_k;
    int causal, at_end;
    float scale, scale_log2;                    // scale, scale * log2(e)
    const int32_t* key_lens;                    // device [batch] or null
    int64_t q_s[3], k_s[3], v_s[3], o_s[3], do_s[3], dq_s[3], dk_s[3], dv_s[3];
    // the bias: n_runs = 0 for none
    const void* table;
    int table_dtype, n_runs;
    int64_t table_s[2];
    int run_first[kHeadsMaxRuns];
    uint8_t run_bucket[kHeadsMaxRuns];
};

// Device pointers of a backward pass and its workspace.
struct HeadsGrads {
    const void *d_o, *q, *k, *v, *o;
    const float* lse;
    void *dq, *dk, *dv, *dtable;
    int pad_q;                  // rows per (batch entry, head) of lse2 and delta: seq_q rounded up to 128
    float* lse2;                // -lse * log2(e) + a shift (0 on the CUDA cores); -inf for rows that see nothing and rows behind seq_q:
                                // their probabilities 2^(s + lse2) come out 0
    float* delta;               // -D_i = -dO_i . O_i
    float* run_sums;            // [batch][heads][q_tiles][n_runs]: sums of dS by run, added up in order by the last kernel
    int q_tiles;                // parts a (batch entry, head) is summed in
    float* amax;                // f16 tensor-core path: [2][batch * kv_heads] largest row norms (squared) of dO and V
};

// Keys seen in batch entry b, and the key position of query 0.
__device__ __forceinline__ int heads_key_count(const HeadsParams& p, int b) {
    return p.key_lens ? min(max(p.key_lens[b], 0), p.seq_k) : p.seq_k;
}
__device__ __forceinline__ int heads_offset(const HeadsParams& p, int n_keys) { return p.at_end ? n_keys - p.seq_q : 0; }

template <typename T> __device__ __forceinline__ float heads_load(const T* p, int64_t i);
template <> __device__ __forceinline__ float heads_load<float>(const float* p, int64_t i) { return p[i]; }
template <> __device__ __forceinline__ float heads_load<__half>(const __half* p, int64_t i) { return __half2float(p[i]); }
template <> __device__ __forceinline__ float heads_load<__nv_bfloat16>(const __nv_bfloat16* p, int64_t i) { return __bfloat162float(p[i]); }
__device__ __forceinline__ void heads_store(float* p, int64_t i, float v) { p[i] = v; }
__device__ __forceinline__ void heads_store(__half* p, int64_t i, float v) { p[i] = __float2half_rn(v); }
__device__ __forceinline__ void heads_store(__nv_bfloat16* p, int64_t i, float v) { p[i] = __float2bfloat16_rn(v); }

// The bias of a run for one head, in log2 units (scores are kept as scale * log2(e) * q.k + this).
__device__ __forceinline__ float heads_run_bias(const HeadsParams& p, int run, int head) {
    const int64_t i = p.run_bucket[run] * p.table_s[0] + head * p.table_s[1];
    float v;
    if (p.table_dtype == EMMYB200_F32) v = static_cast<const float*>(p.table)[i];
    else if (p.table_dtype == EMMYB200_F16) v = __half2float(static_cast<const __half*>(p.table)[i]);
    else v = __bfloat162float(static_cast<const __nv_bfloat16*>(p.table)[i]);
    return v <= kMaskedBias ? -INFINITY : v * kLog2e;
}

// The run a distance falls into: the last r with first[r] <= dist (first[0] counts as minus infinity). `first` in
// shared memory.
__device__ __forceinline__ int heads_run_of(const int* first, int n_runs, int dist) {
    int lo = 0, hi = n_runs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= dist) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// ---- launches, implemented next to their kernels ------------------------------------------------------------------------
// CUDA cores, fp32 arithmetic: any dtype, d = 32, 64, 96 or 128, any alignment.
int heads_fwd_cores(int dtype, int d, const HeadsParams& p, const void* Q, const void* K, const void* V, void* O, float* lse, cudaStream_t s);
int heads_bwd_cores(int dtype, int d, const HeadsParams& p, const HeadsGrads& g, cudaStream_t s);
constexpr int kCoresTile = 64;                  // rows the CUDA-core kernels stage at a time
int heads_cores_rows(const HeadsParams& p);     // rows per thread; a block owns 16 times as many

// Tensor cores: 16-bit operands with d = 64 or 128 that TMA can address (heads_sm100_takes).
struct FwdPlan {
    int packed, tiles, splits;                  // see attention_heads_fwd_sm100.cu
    int64_t rows;                               // batch * heads * seq_q
};
FwdPlan heads_fwd_plan(const HeadsParams& p, int64_t d);
// Workspace of split keys: float2[splits][rows], then float[splits][rows][d].
inline int64_t fwd_part_offset(const FwdPlan& w) { return (w.splits * w.rows * 8 + 255) / 256 * 256; }
inline int64_t fwd_workspace(const FwdPlan& w, int64_t d) { return w.splits == 1 ? 0 : (fwd_part_offset(w) + w.splits * w.rows * d * 4 + 255) / 256 * 256; }
bool heads_sm100_takes(const HeadsParams& p, int dtype, int d, const void* Q, const void* K, const void* V, const void* O);
int heads_fwd_sm100(int dtype, int d, const HeadsParams& p, const FwdPlan& plan, const void* Q, const void* K, const void* V, void* O, float* lse,
                    void* workspace, cudaStream_t s);
bool heads_bwd_sm100_takes(const HeadsParams& p, int dtype, int d, const HeadsGrads& g);
float heads_bwd_shift(int dtype);               // of lse2
int heads_bwd_sm100(int dtype, int d, const HeadsParams& p, const HeadsGrads& g, cudaStream_t s);

}  // namespace emmy
