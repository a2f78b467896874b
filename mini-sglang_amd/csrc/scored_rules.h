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

// ---- Parts.  Keys are cut into parts where there are too few (request, kv head, row block) units for the chip.  The host sizes grid
// and workspace from the call's bounds (scored_cut), the device lays the parts out from the batch's own lengths (find_share); both by
// these functions, so that no batch within its bounds can want more parts than are reserved.
constexpr int32_t kFewRows = 16, kWideRows = 128;                      // rows of a workgroup in the two kernels

// Full parts that `units` units of work are cut into for `slots` workgroups: every unit ends in a part that is half full on average,
// so the rest would run at once; at least half the slots, where the units alone nearly fill them.  The single-token kernel, which
// memory alone bounds, keeps a few more places free for workgroups without work.
M355_HD float full_parts(float slots, float units, bool few) {
    const float rest = slots - (few ? 0.75f : 0.5f) * units;
    return rest > 0.5f * slots ? rest : 0.5f * slots;
}

// Row blocks of a request with E rows of G heads, `most` of them: a request with more rows than the call's bound promised keeps to the
// blocks that were reserved for it and takes nobody else's.
M355_HD int32_t row_blocks(int32_t E, int32_t G, int32_t block_rows, int32_t most) { return imin((E * G + block_rows - 1) / block_rows, most); }

// keys of a full part; work: sum over units of their keys
M355_HD int32_t part_size(float work, float units, float slots, bool few) {
    const float size = work / full_parts(slots, units, few);
    return (int32_t)(size < 1e9f ? size : 1e9f) + 1;
}

// Workgroups of one (request, kv head, part) lie 8 apart (part_item): its parts come in whole rounds of the 8 XCDs, `step` of them at
// a time for these kv heads.
M355_HD int32_t round_step(int32_t Hkv) { return 8 / imin(Hkv & -Hkv, 8); }

// Parts of each unit of a request: ceil(keys / size) of one length, none shorter than scored_cut says; several row blocks take the
// nearest number that gives whole rounds (61 to 72 workgroups an XCD instead of 64 cost a second round: 73 us for 58).  Rounding adds
// step / 2 parts at most, which is what scored_cut reserves: a number below step / 2 stays as it is, it would grow up to eightfold (40/10
// heads of 128, 20 requests of 64 rows over 1000 tokens: 54 us with one part, 94 with four; 9/3 heads of 64, 40 of 64 over 2000: 37
// with three, 49 with eight).
M355_HD int32_t request_parts(int32_t keys, int32_t blocks, int32_t size, int32_t Hkv, bool few) {
    const int32_t shortest_max = few ? 128 : 256, shortest_min = few ? 128 : 64;
    const int32_t least = imax(size, imax(shortest_min, imin(shortest_max, keys / 16)));
    const int32_t nsp = imax(1, (keys + least - 1) / least), step = round_step(Hkv);
    return blocks > 1 && nsp * Hkv >= 8 && nsp >= step / 2 ? (nsp + step / 2) / step * step : nsp;
}

// Workgroup i of a request with n parts a unit: its row block, and u = part * kv heads + kv head.  In whole rounds the row blocks of one
// u lie 8 apart, on one XCD, whose L2 then reads their keys once; otherwise they lie side by side.
struct PartItem { int32_t rb, u; };
M355_HD PartItem part_item(int32_t i, int32_t blocks, int32_t n, int32_t Hkv) {
    if (blocks <= 1) return {0, i};
    if (n * Hkv % 8) return {i % blocks, i / blocks};
    const int32_t y = i >> 3;
    return {y % blocks, (y / blocks) * 8 + (i & 7)};
}

// How a call is cut, from its sizes alone (so that the workspace query and the launch agree).  The rows a request brings choose the
// kernel.  Keys are split where there are fewer (request, kv head, row block) units than twice the workgroups that the chip
// holds at once; find_share then lays out the parts.  A part is at least 256 keys (128 in the few-row kernel), or a sixteenth of the
// request where that is shorter: a single short request is a matter of latency (8 nodes over 700 tokens: 64 keys 9.8 + 4.2 us,
// 128 keys 13.4 + 3.5, 256 keys 15.6 + 3.8; over 4 250 tokens: 256 keys 12.3 + 4.8, 128 keys 11.8 + 6.3).
struct ScoredCut { bool wide; int32_t blocks, slots, max_parts; int64_t grid, part_bytes, bytes; };
inline ScoredCut scored_cut(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int32_t D, int64_t ext, int64_t max_len) {
    constexpr int64_t kCus = 256;
    ScoredCut c = {};
    const int64_t G = Hq / Hkv;
    if (ext > T) ext = T;
    const int64_t rows = ext * G, rb = rows > kFewRows ? kWideRows : kFewRows;
    c.wide = rows > kFewRows;
    c.blocks = (int32_t)((rows + rb - 1) / rb);
    // workgroups a CU holds: two by the LDS at head_dim 128, three by the registers and four by the LDS at 64 (16 draft trees over
    // 500 to 4 000 tokens, wide, two a CU: 47 + 8 us; parts for one a CU: 62 + 6)
    const int64_t slots = kCus * (D == 128 ? 2 : (c.wide ? 3 : 4));
    // (a ragged batch has fewer row blocks than its longest request suggests)
    int64_t blocks = B * c.blocks;
    const int64_t packed = (T * G + rb - 1) / rb + B;
    if (packed < blocks) blocks = packed;
    c.grid = B * Hkv * c.blocks;
    // (find_share reads 64 requests at a time: 250 requests of 63 to 2047 tokens on one kv head take 53.9 us whole and 32.3 + 4.3 in
    // parts, 500 requests 64.2 and 64.8 + 4.5; lengths spread further than that were not measured: whole, the longest request is the
    // launch's time)
    if (blocks * Hkv >= 2 * slots || max_len <= 64 || B > 256) return c;
    c.slots = (int32_t)slots;
    // full parts, one more a unit that is not full, and what rounding adds
    const int64_t units = blocks * Hkv, full = (int64_t)full_parts((float)slots, (float)units, !c.wide);
    const int64_t rounding = c.blocks > 1 ? round_step((int32_t)Hkv) / 2 * units : 0;
    c.max_parts = (int32_t)(full + units + rounding + 16);
    c.grid = c.max_parts;
    c.part_bytes = c.max_parts * rb * (D + 4) * (int64_t)sizeof(float);
    c.bytes = c.part_bytes + T * Hq * 2 * (int64_t)sizeof(int32_t);
    return c;
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
// The same for a tree behind a prefix of P tokens: its tokens end with the last node that has a row, so key - P is a node of the request's
// own rows wherever it is used as one.
M355_HD ReqSpan tree_span(int64_t q0, int64_t q1, int64_t P, int64_t T, int64_t table_tokens) {
    const ReqSpan r = req_span(q0, q1, P, 0, T, table_tokens);
    return req_span(q0, q1, P, (int64_t)r.P + r.E, T, table_tokens);
}

}  // namespace m355
