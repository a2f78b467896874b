// Parameters and score arithmetic shared by the scored-attention kernels (attention over the paged pools with capped or
// biased scores, interval masks, or a tree of drafted tokens behind the prefix).
#pragma once
#include "common.h"
#include "scored_rules.h"

namespace m355 {

struct ScoredParams {
    const uint16_t *q, *k_pool, *v_pool;
    const int32_t* page_table;
    const int64_t *page_table_ids, *seq_lens, *prefix_lens;   // seq_lens null: prefix + rows (trees); prefix_lens null: one row per request
    const int32_t* cu_q;                                      // null with prefix_lens
    uint16_t* out;
    int64_t q_stride, o_stride, row_elems, pt_stride, S;
    int32_t pt_rows, pt_cols, B, T, Hq, Hkv, G, ps, ps_shift;
    float scale_log2;                                         // scale log2(e): scores are kept in log2 units
    float cap_log2, cap_rate;                                 // cap log2(e) and 2 scale log2(e) / cap; cap_log2 0: not capped
    const float* slopes;                                      // [Hq] or null
    int32_t window;                                           // 0: none
    const int32_t *doc_starts, *bidir;                        // [T], [B], or null
    const uint32_t* mask;                                     // trees: [T, words] ancestor bits; null otherwise
    int32_t words;
    const int64_t* positions;                                 // trees: position of every node (read when slopes are given)
    // the launch: row blocks per request, KV splits per row block and their length in tokens (the last split takes what is left)
    int32_t blocks, splits, chunk;
    float* part;                                              // splits > 1: [T * Hq][splits][D + 4] unnormalised O, m, l
    int32_t* part_n;                                          // [T * Hq] splits that hold a part; 1: the row is already final
};

__device__ __forceinline__ ReqSpan load_span(const ScoredParams& p, int b) {
    const int64_t tokens = (int64_t)p.pt_cols * p.ps;
    if (!p.cu_q) {
        const int64_t L = p.seq_lens[b];
        return req_span(b, b + 1, L - 1, L, p.T, tokens);
    }
    const int64_t q0 = p.cu_q[b], q1 = p.cu_q[b + 1], P = p.prefix_lens[b];
    return req_span(q0, q1, P, p.seq_lens ? p.seq_lens[b] : P + (q1 - q0), p.T, tokens);
}

__device__ __forceinline__ const int32_t* table_row(const ScoredParams& p, int b) {
    int64_t r = p.page_table_ids[b];
    r = r < 0 ? 0 : (r >= p.pt_rows ? p.pt_rows - 1 : r);
    return p.page_table + r * p.pt_stride;
}

// Token range of a row block and of the rows' limits inside it: every row of the block sees [lo_max, hi_min), none sees a key
// outside [lo_min, hi_max).
struct BlockRange { int32_t lo_min, hi_max, lo_max, hi_min; };

// Rows j0 .. j1 of a request.  Without documents both limits grow with the row, so the first and the last row tell; a tree's
// rows all see the prefix and at most the whole tree.
__device__ __forceinline__ BlockRange block_range(const ScoredParams& p, const ReqSpan& r, int b, int j0, int j1) {
    if (p.mask) return {0, r.L, 0, imin(r.P, r.L)};
    const int32_t bd = p.bidir ? p.bidir[b] : 0;
    const KeyRange a = visible_range(r.P + j0, r.L, p.window, 0, bd), z = visible_range(r.P + j1, r.L, p.window, 0, bd);
    return {a.lo, z.hi, z.lo, a.hi};
}

// bits of the keys of a 32-key tile that a row sees
__device__ __forceinline__ uint32_t row_bits(const ScoredParams& p, const ReqSpan& r, int64_t t, int32_t lo, int32_t hi, int32_t base) {
    return p.mask ? tree_bits(p.mask + t * p.words, p.words, r.P, hi, base) : range_bits(lo, hi, base);
}

// cap tanh(scale s / cap) log2(e) from the raw product s: tanh(x) = 1 - 2 / (1 + e^2x), exact at both ends (e^2x = 0 and inf);
// near 0 its absolute error is a unit or two of cap 2^-24, which is what counts in an exponent.
__device__ __forceinline__ float cap_score(const ScoredParams& p, float s) {
    return fmaf(-2.f * p.cap_log2, __builtin_amdgcn_rcpf(1.f + exp2_fast(s * p.cap_rate)), p.cap_log2);
}

// Two 16-bit values of a dword: does one of them have all exponent bits set (infinity or NaN), and the dword without those
template <bool F16>
__device__ __forceinline__ bool has_nonfinite(uint32_t w) {
    constexpr uint32_t e = F16 ? 0x7c00u : 0x7f80u;
    return (w & e) == e || ((w >> 16) & e) == e;
}
template <bool F16>
__device__ __forceinline__ uint32_t finite_only(uint32_t w) {
    constexpr uint32_t e = F16 ? 0x7c00u : 0x7f80u;
    if ((w & e) == e) w &= 0xffff0000u;
    if (((w >> 16) & e) == e) w &= 0x0000ffffu;
    return w;
}
template <bool F16>
__device__ __forceinline__ bool frag_nonfinite(bf16x8 f) {
    const u32x4 w = __builtin_bit_cast(u32x4, f);
    return has_nonfinite<F16>(w[0]) || has_nonfinite<F16>(w[1]) || has_nonfinite<F16>(w[2]) || has_nonfinite<F16>(w[3]);
}
template <bool F16>
__device__ __forceinline__ bf16x8 frag_finite(bf16x8 f) {
    const u32x4 w = __builtin_bit_cast(u32x4, f);
    return __builtin_bit_cast(bf16x8, u32x4{finite_only<F16>(w[0]), finite_only<F16>(w[1]), finite_only<F16>(w[2]), finite_only<F16>(w[3])});
}
// the infinities and NaN of four consecutive values, 0 for the others
template <bool F16>
__device__ __forceinline__ f32x4 nonfinite4(uint2 w) {
    const uint32_t x = w.x & ~finite_only<F16>(w.x), y = w.y & ~finite_only<F16>(w.y);
    return f32x4{unpack16_lo<F16>(x), unpack16_hi<F16>(x), unpack16_lo<F16>(y), unpack16_hi<F16>(y)};
}

__device__ __forceinline__ int32_t slot_of(const ScoredParams& p, const int32_t* pt_row, int32_t tok) {
    const int32_t pg = p.ps_shift >= 0 ? tok >> p.ps_shift : tok / p.ps;
    return pool_slot(pt_row[pg], p.ps, tok - pg * p.ps, p.S);
}

}  // namespace m355
