// Log probabilities of given tokens, the entropy of every row and its most likely alternatives, from logits [T, V] (the
// reference's sampler keeps none of them: layers/sampler.py:19-29 takes the argmax).
//
//     d_v = (x_v - max x) / temperature,  S = sum_v e^d_v,  A = sum_v e^d_v d_v
//     log p(v) = d_v - log S,   entropy = log S - A / S,   alternatives: the k largest logits, ties to the lower index
//
// All sums in 32 bits.  A logit of -inf has probability 0 and adds nothing; a row with a NaN, a +inf or nothing but -inf has no
// distribution and gives NaN.  A given token outside [0, V) has log probability -inf.
#include "common.h"

namespace m355 {

constexpr int kMaxTop = 64;                           // M355_MAX_TOP_LOGPROBS

// order of the logits as whole numbers: larger value first, lower index first among equals (-0 equals +0, NaN leads)
__device__ __forceinline__ uint64_t logit_key(float x, int32_t i) {
    x = x != x ? __builtin_bit_cast(float, 0x7fc00000u) : x + 0.f;
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const uint32_t o = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((uint64_t)o << 32) | (0xffffffffu - (uint32_t)i);
}

template <int DT>
__device__ __forceinline__ float logit_at(const void* row, int64_t i) {
    if constexpr (DT == M355_DTYPE_F32) return reinterpret_cast<const float*>(row)[i];
    else return unpack16_lo<DT == M355_DTYPE_F16>((uint32_t)reinterpret_cast<const uint16_t*>(row)[i]);
}

template <int DT>
__global__ __launch_bounds__(256) void token_logprobs_kernel(const uint8_t* __restrict__ logits, int64_t row_bytes, const int64_t* __restrict__ tokens,
                                                             int32_t given, int32_t V, int32_t k, float inv_t, float* __restrict__ logprobs,
                                                             float* __restrict__ entropy, float* __restrict__ top_logprobs,
                                                             int64_t* __restrict__ top_ids) {
    __shared__ float red[3][256];
    __shared__ uint64_t keys[256];
    const int tid = threadIdx.x;
    const int64_t t = blockIdx.x;
    const void* row = logits + t * row_bytes;
    float m = -INFINITY;
    for (int i = tid; i < V; i += 256) m = fmaxf(m, logit_at<DT>(row, i));
    red[0][tid] = m;
    __syncthreads();
    for (int s = 128; s; s >>= 1) {
        if (tid < s) red[0][tid] = fmaxf(red[0][tid], red[0][tid + s]);
        __syncthreads();
    }
    m = red[0][0];
    float S = 0.f, A = 0.f;
    for (int i = tid; i < V; i += 256) {
        const float d = (logit_at<DT>(row, i) - m) * inv_t, e = exp2_fast(d * kLog2e);
        S += e;
        A += e > 0.f ? e * d : 0.f;
    }
    red[1][tid] = S;
    red[2][tid] = A;
    __syncthreads();
    for (int s = 128; s; s >>= 1) {
        if (tid < s) { red[1][tid] += red[1][tid + s]; red[2][tid] += red[2][tid + s]; }
        __syncthreads();
    }
    S = red[1][0];
    const float log_s = logf(S);
    if (tid == 0) entropy[t] = log_s - red[2][0] / S;
    for (int g = tid; g < given; g += 256) {
        const int64_t v = tokens[t * given + g];
        logprobs[t * given + g] = v >= 0 && v < V ? (logit_at<DT>(row, v) - m) * inv_t - log_s : (S == S ? -INFINITY : S);
    }
    uint64_t last = ~0ull;
    for (int n = 0; n < k; ++n) {
        uint64_t best = 0;
        for (int i = tid; i < V; i += 256) {
            const uint64_t key = logit_key(logit_at<DT>(row, i), i);
            if (key < last && key > best) best = key;
        }
        keys[tid] = best;
        __syncthreads();
        for (int s = 128; s; s >>= 1) {
            if (tid < s) keys[tid] = keys[tid] > keys[tid + s] ? keys[tid] : keys[tid + s];
            __syncthreads();
        }
        last = keys[0];
        __syncthreads();
        if (tid == 0) {
            const int64_t v = 0xffffffffu - (uint32_t)last;
            top_ids[t * k + n] = v;
            top_logprobs[t * k + n] = (logit_at<DT>(row, v) - m) * inv_t - log_s;
        }
    }
}

}  // namespace m355

using namespace m355;

extern "C" int64_t m355_token_logprobs_workspace_bytes(int32_t T, int32_t V, int32_t top_k) {
    return 0;
}

extern "C" int m355_token_logprobs(const void* logits, int64_t row_stride, const int64_t* tokens, int32_t given, int32_t T, int32_t V,
                                   int32_t top_k, float temperature, float* logprobs, float* entropy, float* top_logprobs, int64_t* top_ids,
                                   void* workspace, int64_t workspace_bytes, int32_t dtype, void* stream) {
    if (T == 0) return M355_OK;
    if (!logits || !entropy || T < 0 || V <= 0 || given < 0 || top_k < 0 || row_stride < V) return M355_ERR_INVALID_ARG;
    if ((given > 0 && (!tokens || !logprobs)) || (top_k > 0 && (!top_logprobs || !top_ids))) return M355_ERR_INVALID_ARG;
    if (!(temperature > 0.f) || !(temperature < 1e30f) || !(1.f / temperature < 1e30f)) return M355_ERR_INVALID_ARG;
    if (top_k > kMaxTop || top_k > V) return M355_ERR_UNSUPPORTED;
    if (dtype != M355_DTYPE_BF16 && dtype != M355_DTYPE_F16 && dtype != M355_DTYPE_F32) return M355_ERR_UNSUPPORTED;
    const int esize = dtype == M355_DTYPE_F32 ? 4 : 2;
    if ((uintptr_t)logits % esize) return M355_ERR_INVALID_ARG;
#define M355_LOGPROBS(DT) hipLaunchKernelGGL((token_logprobs_kernel<DT>), dim3((unsigned)T), dim3(256), 0, (hipStream_t)stream, \
        (const uint8_t*)logits, row_stride * esize, tokens, given, V, top_k, 1.f / temperature, logprobs, entropy, top_logprobs, top_ids)
    if (dtype == M355_DTYPE_BF16) M355_LOGPROBS(M355_DTYPE_BF16);
    else if (dtype == M355_DTYPE_F16) M355_LOGPROBS(M355_DTYPE_F16);
    else M355_LOGPROBS(M355_DTYPE_F32);
#undef M355_LOGPROBS
    return check_launch();
}
