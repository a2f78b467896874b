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
    float scale, cap;                                         // cap 0: scores are not capped
    const float* slopes;                                      // [Hq] or null
    int32_t window;                                           // 0: none
    const int32_t *doc_starts, *bidir;                        // [T], [B], or null
    const uint32_t* mask;                                     // trees: [T, words] ancestor bits; null otherwise
    int32_t words;
    const int64_t* positions;                                 // trees: position of every node (read when slopes are given)
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

__device__ __forceinline__ int32_t slot_of(const ScoredParams& p, const int32_t* pt_row, int32_t tok) {
    const int32_t pg = p.ps_shift >= 0 ? tok >> p.ps_shift : tok / p.ps;
    return pool_slot(pt_row[pg], p.ps, tok - pg * p.ps, p.S);
}

}  // namespace m355
