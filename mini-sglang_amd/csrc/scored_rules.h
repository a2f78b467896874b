// Which keys a query row of the scored attention sees, and where they live: the index rules as plain functions, shared by
// the kernels and by the tests, which build them for the host (no HIP header is included here).
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define M355_HD __host__ __device__ __forceinline__
#else
#define M355_HD inline
#endif

namespace m355 {

M355_HD int32_t imin(int32_t a, int32_t b) { return a < b ? a : b; }
M355_HD int32_t imax(int32_t a, int32_t b) { return a > b ? a : b; }

// keys [lo, hi) of the query at position `pos` of a request that holds `len` tokens: causal, not before the start of the
// query's document, not further back than the window, and up to `bidir` for everybody (a prompt prefix that attends both
// ways).  A mask that leaves nothing gives lo >= hi.
struct KeyRange { int32_t lo, hi; };
M355_HD KeyRange visible_range(int32_t pos, int32_t len, int32_t window, int32_t doc_start, int32_t bidir) {
    int32_t lo = imax(doc_start, 0);
    if (window > 0) lo = imax(lo, pos - window + 1);
    return {lo, imin(imax(pos + 1, bidir), len)};
}

// the lowest n bits, for any n
M355_HD uint32_t low_bits(int32_t n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); }

// bit x: key base + x lies in [lo, hi)
M355_HD uint32_t range_bits(int32_t lo, int32_t hi, int32_t base) { return low_bits(hi - base) & ~low_bits(lo - base); }

// Tree of drafted tokens behind a prefix of P keys: bit x tells whether key base + x is visible to a node whose ancestor mask
// is mask[0 .. words) (bit j: node j).  Keys below P are all visible, keys at or past hi = P + nodes none.
M355_HD uint32_t tree_bits(const uint32_t* mask, int32_t words, int32_t P, int32_t hi, int32_t base) {
    const int32_t o = base - P;                                        // node of the tile's first key
    uint32_t bits;
    if (o < 0) {
        bits = low_bits(-o);                                           // (o <= -32: the whole tile is prefix)
        if (o > -32 && words > 0) bits |= mask[0] << -o;
    } else {
        const int32_t w = o >> 5, sh = o & 31;
        bits = w < words ? mask[w] >> sh : 0u;
        if (sh && w + 1 < words) bits |= mask[w + 1] << (32 - sh);
    }
    return bits & low_bits(hi - base);
}

// Pool slot of a token: page table entries outside the pool are brought back into it, so that no table content makes a
// kernel read outside the pools.
M355_HD int32_t pool_slot(int32_t page, int32_t ps, int32_t offset, int64_t S) {
    int64_t s = (int64_t)page * ps + offset;
    s = s < 0 ? 0 : (s >= S ? S - 1 : s);
    return (int32_t)s;
}

// Full parts that `units` units of work are cut into for `slots` workgroups: every unit ends in a part that is half full on average,
// so the rest would run at once; at least half the slots, where the units alone nearly fill them.  The single-token kernel, which
// memory alone bounds, keeps a few more places free for workgroups without work.
M355_HD float full_parts(float slots, float units, bool few) {
    const float rest = slots - (few ? 0.75f : 0.5f) * units;
    return rest > 0.5f * slots ? rest : 0.5f * slots;
}

// A request's rows as the kernels use them: q rows q0 .. q0 + E, positions P + j, L cached tokens - whatever the device
// arrays hold, every row lies inside the T rows of q and every token inside the table row.
struct ReqSpan { int32_t q0, E, P, L; };
M355_HD ReqSpan req_span(int64_t q0, int64_t q1, int64_t P, int64_t L, int64_t T, int64_t table_tokens) {
    if (q0 < 0) q0 = 0;
    if (q1 > T) q1 = T;
    if (q1 < q0) q1 = q0;
    if (L > table_tokens) L = table_tokens;
    if (L < 0) L = 0;
    if (P < -1) P = -1;
    if (P > 0x3fffffff) P = 0x3fffffff;
    if (q0 > T) { q0 = T; q1 = T; }
    return {(int32_t)q0, (int32_t)(q1 - q0), (int32_t)P, (int32_t)L};
}

}  // namespace m355
