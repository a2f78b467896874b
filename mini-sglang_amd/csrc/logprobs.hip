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
// is read once: a workgroup holds a block of 8192 logits in registers, the next one on its way, brings its threads' (max, S, A) up to date - kept per
// thread, joined once at the end: a move of the maximum by e multiplies S by 2^e and turns A into 2^e (A + e S) - and
// keeps the k best so far in LDS.  Rows are cut into splits of whole blocks when there are fewer rows than the chip wants
// workgroups; a second launch joins them.
//
// 1500 rows of 128256 fp32 logits, 5 alternatives: 147 us, 5.2 TB/s.  64 rows of bf16 (16 MB) are a matter of latency: 8.6 + 3.5 us
// without alternatives (start, one pass over 4 blocks, the second launch), 14.7 + 4.5 with 20 and 37 + 6 with 64, most of it the
// first block's floor.
#include "common.h"
#include "scored_rules.h"

namespace m355 {

constexpr int kMaxTop = 64;                           // M355_MAX_TOP_LOGPROBS
constexpr int kThreads = 512, kPer = 16;              // threads, and the logits each holds of a block
constexpr int kBlock = kThreads * kPer;
constexpr int kMaxSplits = 32;
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

// x of the lane on the other side of each of a wave's six halvings (VALU only; after step n all lanes of a group of 2^n hold the same)
template <int STEP>
__device__ __forceinline__ float other_lane(float x) {
    if constexpr (STEP < 4) {
        constexpr int ctrl = STEP == 0 ? kDppXor1 : STEP == 1 ? kDppXor2 : STEP == 2 ? kDppHalfMirror : kDppMirror;
        const int u = __builtin_bit_cast(int, x);
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(u, u, ctrl, 0xF, 0xF, true));
    } else {
        return __shfl_xor(x, 1 << STEP);
    }
}
template <int STEP = 0>
__device__ __forceinline__ RowSum wave_join(RowSum s, float rate) {
    if constexpr (STEP == 6) return s;
    else return wave_join<STEP + 1>(join(s, {other_lane<STEP>(s.m), other_lane<STEP>(s.S), other_lane<STEP>(s.A)}, rate), rate);
}
template <int STEP = 0>
__device__ __forceinline__ float wave_min(float x) {
    if constexpr (STEP == 6) return x;
    else return wave_min<STEP + 1>(fminf(x, other_lane<STEP>(x)));
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

// logit of given token g of a row; a token outside the vocabulary has none: -inf
template <int DT>
__device__ __forceinline__ float given_logit(const LogprobParams& p, int64_t t, int g) {
    const int64_t v = p.tokens[t * p.given + g];
    return v >= 0 && v < p.V ? logit_at<DT>(p.logits + t * p.row_bytes, v) : -INFINITY;
}

// Outputs of a row from its sums and its k best keys (in LDS).  `mine`: the logit of given token tid, fetched at the kernel's
// start, where its two dependent loads cost nothing.
template <int DT>
__device__ __forceinline__ void finish_row(const LogprobParams& p, int64_t t, const RowSum r, const uint64_t* best, float mine, int tid, int threads) {
    const float log_s = logf(r.S);
    if (tid == 0) p.entropy[t] = log_s - kLn2 * r.A / r.S;
    for (int g = tid; g < p.given; g += threads)
        p.logprobs[t * p.given + g] = ((g == tid ? mine : given_logit<DT>(p, t, g)) - r.m) * p.inv_t - log_s;
    for (int n = tid; n < p.k; n += threads) {
        const uint64_t key = best[n];
        p.top_ids[t * p.k + n] = 0xffffffffu - (uint32_t)key;
        p.top_logprobs[t * p.k + n] = (key_logit(key) - r.m) * p.inv_t - log_s;
    }
}

// n largest of the keys in list[0 .. count), into out[0 .. n) from the largest; ranks by counting, so the order in which the keys
// were entered does not matter.  list is padded to an even count by the caller's zeros; all threads take part.
template <int THREADS>
__device__ __forceinline__ void rank_keys(const uint64_t* list, int count, int n, uint64_t* out, int tid) {
    for (int c = tid; c < count; c += THREADS) {
        const uint64_t key = list[c];
        int above = 0;
#pragma unroll 4
        for (int j = 0; j < count; j += 2) {
            const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(list + j);
            above += (two.x > key ? 1 : 0) + (two.y > key ? 1 : 0);
        }
        if (key && above < n) out[above] = key;
    }
}

template <int DT>
__global__ __launch_bounds__(kThreads, 4) void token_logprobs_kernel(const LogprobParams p) {
    constexpr int ES = DT == M355_DTYPE_F32 ? 4 : 2, VE = 16 / ES, NV = kPer / VE;      // logits per load, loads per block
    constexpr int kCand = kMaxTop * kPer;
    __shared__ __attribute__((aligned(16))) uint64_t list[kMaxTop + kCand + 2];          // the k best so far, then the block's candidates
    __shared__ uint64_t ranked[kMaxTop];
    __shared__ __attribute__((aligned(16))) float group_max[64];
    __shared__ RowSum red[kThreads / 64];
    __shared__ int32_t count;
    __shared__ uint64_t floor_key;
    const int tid = threadIdx.x;
    const int64_t t = blockIdx.x;
    const int sp = blockIdx.y, k = p.k, k2 = (k + 1) & ~1;          // the list's candidates start at an even place
    // rows of any alignment: loads start at the 16 bytes that hold the row's first logit, and what lies outside the row in the
    // first and last of them is taken for -inf (those 16 bytes hold a logit of the row: they are mapped)
    const uintptr_t addr = (uintptr_t)(p.logits + t * p.row_bytes);
    const uint8_t* row16 = reinterpret_cast<const uint8_t*>(addr & ~(uintptr_t)15);
    const int32_t skip = (int32_t)(addr & 15) / ES;
    const int32_t n_vec = (int32_t)(((int64_t)skip + p.V + VE - 1) / VE);
    const int32_t blocks = (n_vec + kThreads * NV - 1) / (kThreads * NV);
    const int32_t b0 = sp * p.per_split, b1 = imin(blocks, b0 + p.per_split);

    u32x4 next[NV], cur[NV];
    auto fetch = [&](int blk) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int32_t i = imin((blk * NV + v) * kThreads + tid, n_vec - 1);               // (past the end: masked below)
            next[v] = *reinterpret_cast<const u32x4*>(row16 + (int64_t)i * 16);
        }
    };
    auto logit = [&](int e) {                         // element e of the block, unpacked where it is used: two registers hold four
        const uint32_t w = cur[e / VE][DT == M355_DTYPE_F32 ? e % VE : e % VE / 2];
        if constexpr (DT == M355_DTYPE_F32) return __builtin_bit_cast(float, w);
        else return e % 2 ? unpack16_hi<DT == M355_DTYPE_F16>(w) : unpack16_lo<DT == M355_DTYPE_F16>(w);
    };
    const float mine = p.splits == 1 && tid < p.given ? given_logit<DT>(p, t, tid) : 0.f;
    if (tid < kMaxTop) list[tid] = 0;
    if (tid == 0) count = 0;
    uint64_t least = 0;                               // the k-th best key so far (0: fewer than k)
    RowSum s = {-INFINITY, 0.f, 0.f};
    if (b0 < b1) fetch(b0);
    for (int blk = b0; blk < b1; ++blk) {
#pragma unroll
        for (int v = 0; v < NV; ++v) cur[v] = next[v];
        if (blk + 1 < b1) fetch(blk + 1);
        // index of element e: i0 + (e / VE) kThreads VE + e % VE
        const int32_t i0 = (blk * NV * kThreads + tid) * VE - skip;
        auto inside = [&](int e) { const int32_t i = i0 + (e / VE) * kThreads * VE + e % VE; return i >= 0 && i < p.V; };
        if (blk == 0 || (blk + 1) * NV * kThreads >= n_vec) {
            constexpr uint32_t low = DT == M355_DTYPE_F32 ? 0xff800000u : (DT == M355_DTYPE_F16 ? 0xfc00u : 0xff80u);
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                if (inside(e)) continue;
                uint32_t w = cur[e / VE][DT == M355_DTYPE_F32 ? e % VE : e % VE / 2];
                if constexpr (DT == M355_DTYPE_F32) w = low;
                else w = e % 2 ? (w & 0xffffu) | (low << 16) : (w & 0xffff0000u) | low;
                cur[e / VE][DT == M355_DTYPE_F32 ? e % VE : e % VE / 2] = w;
            }
        }
        float mx = logit(0);
#pragma unroll
        for (int e = 1; e < kPer; ++e) mx = fmaxf(mx, logit(e));
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
            const float d = (logit(e) - mu) * p.rate, w = exp2_fast(d);
            s.S += w;
            s.A = fmaf(w, fmaxf(d, -1e30f), s.A);     // (0 * -inf would be NaN)
            if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);               // (a few at a time: registers are occupancy here)
        }
        if (k == 0) continue;

        // ---- the k best so far.  A thread has something to offer if its largest logit beats the k-th best (later indices lose
        // ties); NaN, which leads the order, shows in S.
        const bool offers = (s.S != s.S) || mx > key_logit(least) || least == 0;
        if (!__syncthreads_or(offers)) continue;
        // A floor under the k-th best, so that few logits are looked at one by one.  First the k-th largest of 64 groups of threads' largest
        // logits; k groups hold a logit at or above it.  Where so many logits tie with it that they do not fit the list, the k-th largest KEY
        // of the threads' best: keys are distinct, so only k threads hold anything at or above it - k * kPer candidates at
        // most, whatever the logits are.
        for (int round = least ? 1 : 0;; ++round) {
            float floor = -INFINITY;
            uint64_t at_least = least + 1;
            if (round == 0) {
                float g = fmaxf(mx, other_lane<0>(mx));
                g = fmaxf(g, other_lane<1>(g));
                if constexpr (kThreads == 512) g = fmaxf(g, other_lane<2>(g));
                if (tid % (kThreads / 64) == 0) group_max[tid / (kThreads / 64)] = g;
                __syncthreads();
                const float mine = group_max[tid & 63];
                int above = 0;
#pragma unroll 4
                for (int u = 0; u < 64; u += 4) {
                    const f32x4 four = *reinterpret_cast<const f32x4*>(group_max + u);
                    above += (four[0] > mine ? 1 : 0) + (four[1] > mine ? 1 : 0) + (four[2] > mine ? 1 : 0) + (four[3] > mine ? 1 : 0);
                }
                floor = wave_min(above < k ? mine : INFINITY);
            } else if (round == 1) {
                floor = key_logit(least);
            } else {
                uint64_t mine = 0;
#pragma unroll 1
                for (int e = 0; e < kPer; ++e) {
                    const int32_t i = i0 + (e / VE) * kThreads * VE + e % VE;
                    if (i < 0 || i >= p.V) continue;
                    const uint64_t key = logit_key(logit_at<DT>(row16, (int64_t)i + skip), (uint32_t)i);
                    if (key > mine) mine = key;
                }
                list[k2 + tid] = mine;
                if (tid == 0) floor_key = 0;
                __syncthreads();
                int above = 0;
#pragma unroll 4
                for (int u = 0; u < kThreads; ++u) above += list[k2 + u] > mine ? 1 : 0;
                if (mine && above == k - 1) floor_key = mine;
                __syncthreads();
                if (floor_key > at_least) at_least = floor_key;
            }
            if (offers) {
#pragma unroll
                for (int e = 0; e < kPer; ++e) {
                    float x = logit(e);
                    if (!(x < floor)) {               // rare (NaN is not below anything); the empty asm keeps all of it in here
                        int32_t i = i0;
                        asm volatile("" : "+v"(i), "+v"(x));
                        i += (e / VE) * kThreads * VE + e % VE;
                        const uint64_t key = logit_key(x, (uint32_t)i);
                        if (i >= 0 && i < p.V && key >= at_least) {
                            const int at = atomicAdd(&count, 1);
                            if (at < kCand) list[k2 + at] = key;
                        }
                    }
                }
            }
            __syncthreads();
            const int found = count;
            if (found <= kCand) {
                if (tid < kMaxTop) ranked[tid] = 0;
                if (tid < 2) list[k2 + found + tid] = 0;
                __syncthreads();
                rank_keys<kThreads>(list, k2 + found, k, ranked, tid);
                __syncthreads();
                if (tid < k) list[tid] = ranked[tid];
                least = ranked[k - 1];
                if (tid == 0) count = 0;
                break;
            }
            __syncthreads();
            if (tid == 0) count = 0;
            round = round < 1 ? 1 : round;            // (on to the exact floor)
            __syncthreads();
        }
    }

    // ---- the threads' sums: across the wave, then across the waves
    s = wave_join(s, p.rate);
    if ((tid & 63) == 0) red[tid >> 6] = s;
    __syncthreads();
    s = red[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) s = join(s, red[w], p.rate);
    if (p.splits > 1) {
        if (tid == 0) p.part[t * p.splits + sp] = s;
        if (tid < k) p.part_keys[(t * p.splits + sp) * k + tid] = list[tid];
        return;
    }
    finish_row<DT>(p, t, s, list, mine, tid, kThreads);
}

// Joins a row's splits: sums pairwise in split order, the k best of the splits' falling key lists by rank.  The k-th best is at
// least every list's k-th key, and at least the smallest of the lists' c-th keys with c = ceil(k / lists) (k keys are at or above it):
// what lies below is left out before ranks are counted.
template <int DT>
__global__ __launch_bounds__(256) void token_logprobs_join_kernel(const LogprobParams p) {
    __shared__ __attribute__((aligned(16))) uint64_t all[kMaxSplits * kMaxTop], list[kMaxSplits * kMaxTop + 2];
    __shared__ uint64_t best[kMaxTop];
    __shared__ RowSum sums[kMaxSplits];
    __shared__ int32_t count;
    const int tid = threadIdx.x, k = p.k, n = p.splits;
    const int64_t t = blockIdx.x;
    const float mine = tid < p.given ? given_logit<DT>(p, t, tid) : 0.f;
    if (tid == 0) count = 0;
    if (tid < n) sums[tid] = p.part[t * n + tid];
    for (int i = tid; i < n * k; i += 256) all[i] = p.part_keys[t * n * k + i];
    __syncthreads();
    if (k) {
        const int c = (k + n - 1) / n - 1;
        uint64_t least = 1, low = ~0ull;
        for (int l = 0; l < n; ++l) {
            const uint64_t last = all[l * k + k - 1], cth = all[l * k + c];
            if (last > least) least = last;
            if (cth < low) low = cth;
        }
        if (low > least) least = low;
        for (int i = tid; i < n * k; i += 256)
            if (all[i] >= least) list[atomicAdd(&count, 1)] = all[i];
    }
    __syncthreads();
    const int found = count;
    if (tid < 2) list[found + tid] = 0;
    if (tid < 64) {                                   // the splits' sums, by one wave (n <= 32)
        const RowSum s = wave_join(tid < n ? sums[tid] : RowSum{-INFINITY, 0.f, 0.f}, p.rate);
        if (tid == 0) sums[0] = s;
    }
    __syncthreads();
    rank_keys<256>(list, found, k, best, tid);
    __syncthreads();
    finish_row<DT>(p, t, sums[0], best, mine, tid, 256);
}

// Splits of a row, in whole blocks: as many as fit the chip at once, two workgroups a CU (64 rows of 128256 bf16 logits, 20
// alternatives, before the candidates moved up to the list: 8 splits 16.6 + 4.5 us for the two launches, 16 splits 20.8 + 6.2, 4 splits
// of half the threads 21.6 + 4.4).
struct LogprobCut { int32_t splits, per_split; int64_t part_bytes, bytes; };
static LogprobCut logprob_cut(int64_t T, int64_t V, int64_t k) {
    const int64_t blocks = (V + 15 + kBlock - 1) / kBlock;             // (15: the logits of a load before the row's first)
    int64_t want = T < 512 ? 512 / T : 1;
    if (want > kMaxSplits) want = kMaxSplits;
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
    hipLaunchKernelGGL((token_logprobs_kernel<DT>), dim3((unsigned)p.T, (unsigned)p.splits), dim3(kThreads), 0, st, p);
    if (p.splits > 1)
        hipLaunchKernelGGL((token_logprobs_join_kernel<DT>), dim3((unsigned)p.T), dim3(256), 0, st, p);
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
