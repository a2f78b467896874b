// Log probabilities of given tokens, the entropy of every row and its most likely alternatives, from logits [T, V] (the
// reference's sampler keeps none of them: layers/sampler.py:19-29 takes the argmax).
//
//     d_v = (x_v - max x) / temperature,  S = sum_v e^d_v,  A = sum_v e^d_v d_v
//     log p(v) = d_v - log S,   entropy = log S - A / S,   alternatives: the k largest logits, ties to the lower index
//
// All sums in 32 bits.  A logit of -inf has probability 0 and adds nothing; a row with a NaN, a +inf or nothing but -inf has no
// distribution and gives NaN.  A given token outside [0, V) has log probability -inf.
//
// Bound by the logits' bytes, with the vector unit close behind (an exponential and seven plain instructions per logit), so a row
// is read once: a workgroup holds a block of 8192 logits in registers, brings its threads' (max, S, A) up to date - kept per
// thread, joined once at the end: a move of the maximum by e multiplies S by 2^e and turns A into 2^e (A + e S) - and
// keeps the k best so far in LDS.  Rows are cut into splits of whole blocks when there are fewer rows than the chip wants
// workgroups; a second launch joins them.
#include "common.h"
#include "scored_rules.h"

namespace m355 {

constexpr int kMaxTop = 64;                           // M355_MAX_TOP_LOGPROBS
constexpr int kPer = 32;                              // logits a thread holds of a block
constexpr int kBlock = 256 * kPer;
constexpr float kLn2 = 0.6931471805599453f;

// Order of the logits as whole numbers: larger value first, lower index first among equals (-0 equals +0, NaN leads).  Keys are
// distinct and never 0, which stands for "nothing".
__device__ __forceinline__ uint64_t logit_key(float x, uint32_t i) {
    x = x != x ? __builtin_bit_cast(float, 0x7fc00000u) : x + 0.f;
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const uint32_t o = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((uint64_t)o << 32) | (0xffffffffu - i);
}
__device__ __forceinline__ float key_logit(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __builtin_bit_cast(float, (o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

// max, S and A (in units of log 2) of a set of logits
struct RowSum { float m, S, A; };
// a maximum that moves from `a` up to `m`, in units of log 2; kept finite (2^it is 0 long before), so that 0 never meets infinity
__device__ __forceinline__ float log_move(float a, float m, float rate) { return fmaxf((a - m) * rate, -1e30f); }
__device__ __forceinline__ RowSum join(const RowSum a, const RowSum b, float rate) {
    const float m = fmaxf(a.m, b.m);
    if (m == -INFINITY) return {m, a.S + b.S, 0.f};
    const float da = a.m == -INFINITY ? 0.f : log_move(a.m, m, rate), db = b.m == -INFINITY ? 0.f : log_move(b.m, m, rate);
    const float ea = exp2_fast(da), eb = exp2_fast(db);
    return {m, ea * a.S + eb * b.S, ea * fmaf(da, a.S, a.A) + eb * fmaf(db, b.S, b.A)};
}

struct LogprobParams {
    const uint8_t* logits;
    int64_t row_bytes;
    const int64_t* tokens;
    int32_t given, T, V, k, splits, per_split;        // per_split: blocks of kBlock logits
    float inv_t, rate;                                // rate = log2(e) / temperature
    float *logprobs, *entropy, *top_logprobs;
    int64_t* top_ids;
    RowSum* part;                                     // splits > 1: [T][splits], and the keys [T][splits][k]
    uint64_t* part_keys;
};

template <int DT>
__device__ __forceinline__ float logit_at(const uint8_t* row, int64_t i) {
    if constexpr (DT == M355_DTYPE_F32) return reinterpret_cast<const float*>(row)[i];
    else return unpack16_lo<DT == M355_DTYPE_F16>((uint32_t)reinterpret_cast<const uint16_t*>(row)[i]);
}

// outputs of a row from its sums and its k best keys (in LDS), by the first `threads` threads
template <int DT>
__device__ __forceinline__ void finish_row(const LogprobParams& p, int64_t t, const RowSum r, const uint64_t* best, int tid, int threads) {
    const uint8_t* row = p.logits + t * p.row_bytes;
    const float log_s = logf(r.S);
    if (tid == 0) p.entropy[t] = log_s - kLn2 * r.A / r.S;
    for (int g = tid; g < p.given; g += threads) {
        const int64_t v = p.tokens[t * p.given + g];
        float lp = r.S != r.S || r.m == -INFINITY ? __builtin_nanf("") : -INFINITY;
        if (v >= 0 && v < p.V) lp = (logit_at<DT>(row, v) - r.m) * p.inv_t - log_s;
        p.logprobs[t * p.given + g] = lp;
    }
    for (int n = tid; n < p.k; n += threads) {
        const uint64_t key = best[n];
        p.top_ids[t * p.k + n] = 0xffffffffu - (uint32_t)key;
        p.top_logprobs[t * p.k + n] = (key_logit(key) - r.m) * p.inv_t - log_s;
    }
}

template <int DT>
__global__ __launch_bounds__(256, 4) void token_logprobs_kernel(const LogprobParams p) {
    constexpr int ES = DT == M355_DTYPE_F32 ? 4 : 2, VE = 16 / ES, NV = kPer / VE;      // logits per load, loads per block
    __shared__ uint64_t cand[kMaxTop * kPer];         // logits that may belong to the k best
    __shared__ __attribute__((aligned(16))) uint64_t lead[256];    // the threads' best
    __shared__ uint64_t best[2][kMaxTop];
    __shared__ RowSum red[256];
    __shared__ int32_t count;
    __shared__ uint64_t floor_key;
    const int tid = threadIdx.x;
    const int64_t t = blockIdx.x;
    const int sp = blockIdx.y, k = p.k;
    // rows of any alignment: loads start at the 16 bytes that hold the row's first logit, and what lies outside the row in the
    // first and last of them is taken for -inf (those 16 bytes hold a logit of the row: they are mapped)
    const uintptr_t addr = (uintptr_t)(p.logits + t * p.row_bytes);
    const uint8_t* row16 = reinterpret_cast<const uint8_t*>(addr & ~(uintptr_t)15);
    const int32_t skip = (int32_t)(addr & 15) / ES;
    const int32_t n_vec = (int32_t)(((int64_t)skip + p.V + VE - 1) / VE);
    const int32_t blocks = (n_vec + 256 * NV - 1) / (256 * NV);
    const int32_t b0 = sp * p.per_split, b1 = imin(blocks, b0 + p.per_split);

    u32x4 next[NV];
    auto fetch = [&](int blk) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int32_t i = imin((blk * NV + v) * 256 + tid, n_vec - 1);               // (past the end: masked below)
            next[v] = *reinterpret_cast<const u32x4*>(row16 + (int64_t)i * 16);
        }
    };
    if (tid < kMaxTop) best[0][tid] = 0;
    if (tid == 0) count = 0;
    int cur = 0;
    uint64_t least = 0;                               // the k-th best key so far (0: fewer than k)
    RowSum s = {-INFINITY, 0.f, 0.f};
    if (b0 < b1) fetch(b0);
    for (int blk = b0; blk < b1; ++blk) {
        float x[kPer];
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                if constexpr (DT == M355_DTYPE_F32) {
                    const uint32_t u = next[v][w];
                    x[VE * v + w] = __builtin_bit_cast(float, u);
                } else {
                    x[VE * v + 2 * w] = unpack16_lo<DT == M355_DTYPE_F16>(next[v][w]);
                    x[VE * v + 2 * w + 1] = unpack16_hi<DT == M355_DTYPE_F16>(next[v][w]);
                }
            }
        if (blk + 1 < b1) fetch(blk + 1);
        // index of element e of vector v: VE * vector - skip + e
        const int32_t i0 = (blk * NV * 256 + tid) * VE - skip;
        if (blk == 0 || (blk + 1) * NV * 256 >= n_vec) {
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                const int32_t i = i0 + (e / VE) * 256 * VE + e % VE;
                x[e] = i >= 0 && i < p.V ? x[e] : -INFINITY;
            }
        }
        float mx = x[0];
#pragma unroll
        for (int e = 1; e < kPer; ++e) mx = fmaxf(mx, x[e]);
        const float m = fmaxf(s.m, mx);
        if (s.m != -INFINITY && m > s.m) {
            const float d = log_move(s.m, m, p.rate), f = exp2_fast(d);
            s.A = f * fmaf(d, s.S, s.A);
            s.S *= f;
        }
        s.m = m;
        const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const float d = (x[e] - mu) * p.rate, w = exp2_fast(d);
            s.S += w;
            s.A = fmaf(w, fmaxf(d, -1e30f), s.A);     // (0 * -inf would be NaN)
        }
        if (k == 0) continue;

        // ---- the k best so far.  A thread has something to offer if its largest logit beats the k-th best (later indices lose
        // ties); NaN, which leads the order, shows in S.
        const bool offers = (s.S != s.S) || mx > key_logit(least) || least == 0;
        if (!__syncthreads_or(offers)) continue;
        bool by_floor = least == 0;
        for (;;) {
            uint64_t at_least = least + 1;
            if (by_floor) {
                // the k-th largest of the threads' best is a floor under the k-th best logit, and only k threads can hold
                // anything above it: at most k * kPer candidates, whatever the logits are
                uint64_t mine = 0;
#pragma unroll
                for (int e = 0; e < kPer; ++e) {
                    const int32_t i = i0 + (e / VE) * 256 * VE + e % VE;
                    const uint64_t key = logit_key(x[e], (uint32_t)i);
                    if (i >= 0 && i < p.V && key > mine) mine = key;
                }
                lead[tid] = mine;
                if (tid == 0) floor_key = 0;
                __syncthreads();
                int above = 0;
                for (int u = 0; u < 256; u += 2) {
                    const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(lead + u);
                    above += (two.x > mine ? 1 : 0) + (two.y > mine ? 1 : 0);
                }
                if (mine && above == k - 1) floor_key = mine;
                __syncthreads();
                if (floor_key > at_least) at_least = floor_key;
            }
            if (offers) {
#pragma unroll
                for (int e = 0; e < kPer; ++e) {
                    const int32_t i = i0 + (e / VE) * 256 * VE + e % VE;
                    const uint64_t key = logit_key(x[e], (uint32_t)i);
                    if (key >= at_least && i >= 0 && i < p.V) {
                        const int at = atomicAdd(&count, 1);
                        if (at < kMaxTop * kPer) cand[at] = key;
                    }
                }
            }
            __syncthreads();
            const int found = count;
            if (found <= kMaxTop * kPer) {
                // ranks among the k best so far and the candidates; the order in which they were entered does not matter
                if (tid < k) best[1 - cur][tid] = 0;
                __syncthreads();
                for (int c = tid; c < k + found; c += 256) {
                    const uint64_t key = c < k ? best[cur][c] : cand[c - k];
                    if (key == 0) continue;
                    int above = 0;
                    for (int j = 0; j < k; ++j) above += best[cur][j] > key ? 1 : 0;
                    for (int j = 0; j < found; ++j) above += cand[j] > key ? 1 : 0;
                    if (above < k) best[1 - cur][above] = key;
                }
                __syncthreads();
                cur = 1 - cur;
                least = best[cur][k - 1];
                if (tid == 0) count = 0;
                break;
            }
            __syncthreads();                          // too many to hold: raise the floor and collect again
            if (tid == 0) count = 0;
            __syncthreads();
            by_floor = true;
        }
    }

    red[tid] = s;
    __syncthreads();
    for (int n = 128; n; n >>= 1) {
        if (tid < n) red[tid] = join(red[tid], red[tid + n], p.rate);
        __syncthreads();
    }
    if (p.splits > 1) {
        if (tid == 0) p.part[t * p.splits + sp] = red[0];
        if (tid < k) p.part_keys[(t * p.splits + sp) * k + tid] = best[cur][tid];
        return;
    }
    finish_row<DT>(p, t, red[0], best[cur], tid, 256);
}

// Joins a row's splits: sums pairwise in split order, ranks of the splits' sorted keys by binary search in the other lists.
template <int DT>
__global__ __launch_bounds__(256) void token_logprobs_join_kernel(const LogprobParams p) {
    extern __shared__ __attribute__((aligned(16))) uint64_t lists[];              // [splits][k]
    __shared__ uint64_t best[kMaxTop];
    __shared__ RowSum sums[256];
    const int tid = threadIdx.x, k = p.k, n = p.splits;
    const int64_t t = blockIdx.x;
    for (int i = tid; i < n * k; i += 256) lists[i] = p.part_keys[t * n * k + i];
    if (tid < n) sums[tid] = p.part[t * n + tid];
    __syncthreads();
    for (int step = 1; step < n; step <<= 1) {
        const int at = tid * 2 * step;
        if (at + step < n) sums[at] = join(sums[at], sums[at + step], p.rate);
        __syncthreads();
    }
    for (int i = tid; i < n * k; i += 256) {
        const uint64_t key = lists[i];
        if (key == 0) continue;
        int above = 0;
        for (int l = 0; l < n && above < k; ++l) {
            int lo = 0, hi = k;                       // keys of list l above `key`: the list falls
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (lists[l * k + mid] > key) lo = mid + 1; else hi = mid;
            }
            above += lo;
        }
        if (above < k) best[above] = key;
    }
    __syncthreads();
    finish_row<DT>(p, t, sums[0], best, tid, 256);
}

// Splits of a row: as many as bring the launch to about 1024 workgroups, in whole blocks.
struct LogprobCut { int32_t splits, per_split; int64_t part_bytes, bytes; };
static LogprobCut logprob_cut(int64_t T, int64_t V, int64_t k) {
    const int64_t blocks = (V + 15 + kBlock - 1) / kBlock;             // (15: the logits of a load before the row's first)
    int64_t want = (1024 + T - 1) / T;
    if (want > 64) want = 64;
    if (want > blocks) want = blocks;
    LogprobCut c;
    c.per_split = (int32_t)((blocks + want - 1) / want);
    c.splits = (int32_t)((blocks + c.per_split - 1) / c.per_split);
    c.part_bytes = (T * c.splits * (int64_t)sizeof(RowSum) + 255) / 256 * 256;
    c.bytes = c.splits > 1 ? c.part_bytes + T * c.splits * k * (int64_t)sizeof(uint64_t) : 0;
    return c;
}

template <int DT>
static void launch_logprobs(const LogprobParams& p, hipStream_t st) {
    hipLaunchKernelGGL((token_logprobs_kernel<DT>), dim3((unsigned)p.T, (unsigned)p.splits), dim3(256), 0, st, p);
    if (p.splits > 1)
        hipLaunchKernelGGL((token_logprobs_join_kernel<DT>), dim3((unsigned)p.T), dim3(256), (size_t)p.splits * p.k * sizeof(uint64_t), st, p);
}

}  // namespace m355

using namespace m355;

extern "C" int64_t m355_token_logprobs_workspace_bytes(int32_t T, int32_t V, int32_t top_k) {
    if (T <= 0 || V <= 0 || top_k < 0 || top_k > kMaxTop) return 0;
    return logprob_cut(T, V, top_k).bytes;
}

extern "C" int m355_token_logprobs(const void* logits, int64_t row_stride, const int64_t* tokens, int32_t given, int32_t T, int32_t V,
                                   int32_t top_k, float temperature, float* logprobs, float* entropy, float* top_logprobs, int64_t* top_ids,
                                   void* workspace, int64_t workspace_bytes, int32_t dtype, void* stream) {
    if (T == 0) return M355_OK;
    if (!logits || !entropy || T < 0 || V <= 0 || V > 0x3fffffff || given < 0 || top_k < 0 || row_stride < V) return M355_ERR_INVALID_ARG;
    if ((given > 0 && (!tokens || !logprobs)) || (top_k > 0 && (!top_logprobs || !top_ids))) return M355_ERR_INVALID_ARG;
    if (!(temperature > 0.f) || !(temperature < 1e30f) || !(1.f / temperature < 1e30f)) return M355_ERR_INVALID_ARG;
    if (top_k > kMaxTop || top_k > V) return M355_ERR_UNSUPPORTED;
    if (dtype != M355_DTYPE_BF16 && dtype != M355_DTYPE_F16 && dtype != M355_DTYPE_F32) return M355_ERR_UNSUPPORTED;
    const int esize = dtype == M355_DTYPE_F32 ? 4 : 2;
    if ((uintptr_t)logits % esize) return M355_ERR_INVALID_ARG;
    const LogprobCut c = logprob_cut(T, V, top_k);
    if (c.bytes && (!workspace || workspace_bytes < c.bytes || ((uintptr_t)workspace & 255))) return M355_ERR_WORKSPACE;
    LogprobParams p = {};
    p.logits = (const uint8_t*)logits; p.row_bytes = row_stride * esize; p.tokens = tokens; p.given = given; p.T = T; p.V = V; p.k = top_k;
    p.splits = c.splits; p.per_split = c.per_split; p.inv_t = 1.f / temperature; p.rate = kLog2e / temperature;
    p.logprobs = logprobs; p.entropy = entropy; p.top_logprobs = top_logprobs; p.top_ids = top_ids;
    p.part = (RowSum*)workspace; p.part_keys = (uint64_t*)((uint8_t*)workspace + c.part_bytes);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == M355_DTYPE_BF16) launch_logprobs<M355_DTYPE_BF16>(p, st);
    else if (dtype == M355_DTYPE_F16) launch_logprobs<M355_DTYPE_F16>(p, st);
    else launch_logprobs<M355_DTYPE_F32>(p, st);
    return check_launch();
}
