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
    const int64_t* positions;                                 // trees: position of every node (read for slopes and windows)
    // the launch: row blocks of the longest request, and - where keys are split - the workgroups that fit the chip at once, the
    // parts there is room for, and the parts themselves
    int32_t blocks, slots, max_parts;                         // slots 0: no splits
    float* part;                                              // [max_parts][rows of a block][D + 4] unnormalised O, m, l
    int2* part_of;                                            // [T * Hq] {first row of the parts, how many}; 1 and fewer: the row is final
};

__device__ __forceinline__ ReqSpan load_span(const ScoredParams& p, int b) {
    const int64_t tokens = (int64_t)p.pt_cols * p.ps;
    if (!p.cu_q) {
        const int64_t L = p.seq_lens[b];
        return req_span(b, b + 1, L - 1, L, p.T, tokens);
    }
    const int64_t q0 = p.cu_q[b], q1 = p.cu_q[b + 1], P = p.prefix_lens[b];
    return p.seq_lens ? req_span(q0, q1, P, p.seq_lens[b], p.T, tokens) : tree_span(q0, q1, P, p.T, tokens);
}

__device__ __forceinline__ const int32_t* table_row(const ScoredParams& p, int b) {
    int64_t r = p.page_table_ids[b];
    r = r < 0 ? 0 : (r >= p.pt_rows ? p.pt_rows - 1 : r);
    return p.page_table + r * p.pt_stride;
}

// One workgroup's share of a call: row block rb of request b, kv head h, part sp of nsp, `chunk` keys each; its rows' results go to
// part slot part0 + sp.
struct Share {
    bool any;
    int32_t b, h, rb, sp, nsp, chunk, part0;
    ReqSpan r;
    const int32_t* pt_row;
};

// Inclusive sums over the lanes of a wave, in six vector instructions: inside rows of 16, then across them (the sum of lane 15 of
// each row to the next, of lane 31 to the upper half).
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T dpp_plus(T x) {
    return x + __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROWS, 0xF, false));
}
template <typename T>
__device__ __forceinline__ T wave_sums(T x) {
    x = dpp_plus<0x111, 0xF>(x);                       // row_shr:1
    x = dpp_plus<0x112, 0xF>(x);
    x = dpp_plus<0x114, 0xF>(x);
    x = dpp_plus<0x118, 0xF>(x);
    x = dpp_plus<0x142, 0xA>(x);                       // row_bcast:15
    return dpp_plus<0x143, 0xC>(x);                    // row_bcast:31
}
template <typename T>
__device__ __forceinline__ T lane_value(T x, int lane) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}

// Splits follow the batch, which the host does not know: every wave reads the requests' lengths (one per lane) and lays the work
// out for itself, the same way in all of them.
//   work  W = sum over requests of row blocks x keys x kv heads; a part holds at most size = W / full_parts keys (part_size)
//   parts nsp = ceil(keys / size) per request, all of one length: full_parts + units at most, and what rounding to whole rounds of the 8
//   XCDs adds (request_parts), which sizes grid and workspace
// Workgroups are numbered request by request, so those with nothing to do come last.  A workgroup that only finds out that it is idle
// still waits for a place and holds it for 2 us: with idle ones in between, the others started up to 40 us late.
template <int RB, bool FEW>
__device__ __forceinline__ Share find_share(const ScoredParams& p) {
    const int lane = threadIdx.x & 63;
    struct Req { ReqSpan r; int32_t blocks, keys, row; };
    auto load = [&](int b) {                           // everything a share needs of a request, in one round of loads
        Req q;
        const int at = imin(b, p.B - 1);
        const int64_t row = p.page_table_ids[at];
        q.r = load_span(p, at);
        q.row = (int32_t)(row < 0 ? 0 : (row >= p.pt_rows ? p.pt_rows - 1 : row));
        q.blocks = b < p.B ? row_blocks(q.r.E, p.G, RB, p.blocks) : 0;
        q.keys = p.window > 0 ? imin(q.r.L, imin(p.window, 0x3fffffff) + (p.mask ? q.r.E : RB)) : q.r.L;
        return q;
    };
    const Req first = load(lane);
    float work = 0.f, units = 0.f;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
        const Req q = b0 ? load(b0 + lane) : first;
        work += lane_value(wave_sums((float)q.blocks * (float)q.keys), 63);
        units += lane_value(wave_sums((float)q.blocks), 63);
    }
    work *= (float)p.Hkv;
    units *= (float)p.Hkv;
    const int32_t size = part_size(work, units, (float)p.slots, FEW);
    int32_t at = (int32_t)blockIdx.x, part0 = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
        const Req q = b0 ? load(b0 + lane) : first;
        const int32_t nsp = request_parts(q.keys, q.blocks, size, p.Hkv, FEW);
        const int32_t items = nsp * p.Hkv * q.blocks, items_to = wave_sums(items);       // (a workgroup a part)
        const unsigned long long past = __ballot(at < items_to);
        if (past) {
            const int k = __builtin_ctzll(past);       // the request of this workgroup, in lane k
            const int32_t i = at - lane_value(items_to - items, k), blocks = lane_value(q.blocks, k), n = lane_value(nsp, k);
            Share s;
            const PartItem it = part_item(i, blocks, n, p.Hkv);
            const int32_t u = it.u;
            s.rb = it.rb;
            s.any = true;
            // the kv head turns with part and request: an XCD should not read one head's column of the pools only (8 heads, 8 XCDs)
            s.sp = u / p.Hkv;
            s.b = b0 + k;
            s.h = blocks > 1 ? u % p.Hkv : (u + s.sp + s.b) % p.Hkv;
            s.nsp = n;
            s.chunk = ((lane_value(q.keys, k) + n - 1) / n + 63) & ~63;
            s.part0 = part0 + lane_value(items_to - items, k) + (s.rb * p.Hkv + s.h) * n;
            s.r = {lane_value(q.r.q0, k), lane_value(q.r.E, k), lane_value(q.r.P, k), lane_value(q.r.L, k)};
            s.pt_row = p.page_table + (int64_t)lane_value(q.row, k) * p.pt_stride;
            if (s.part0 + n > p.max_parts) s.any = false;              // (only cu_q that contradicts the call's bounds gets here)
            return s;
        }
        at -= lane_value(items_to, 63);
        part0 += lane_value(items_to, 63);
    }
    Share none = {};
    return none;
}

// Token range of a row block and of the rows' limits inside it: every row of the block sees [lo_max, hi_min), none sees a key
// outside [lo_min, hi_max).
struct BlockRange { int32_t lo_min, hi_max, lo_max, hi_min; };

// Rows j0 .. j1 of a request.  Without documents both limits grow with the row, so the first and the last row tell; a tree's
// rows all see the prefix and at most the whole tree.
__device__ __forceinline__ BlockRange block_range(const ScoredParams& p, const ReqSpan& r, int b, int j0, int j1) {
    if (p.mask) {                                      // positions P .. P + E - 1, in no order
        if (p.window == 0) return {0, r.L, 0, imin(r.P, r.L)};
        return {imax(r.P - p.window + 1, 0), r.L, imax(r.P + r.E - p.window, 0), imin(r.P, r.L)};
    }
    const int32_t bd = p.bidir ? p.bidir[b] : 0;
    const KeyRange a = visible_range(r.P + j0, r.L, p.window, 0, bd), z = visible_range(r.P + j1, r.L, p.window, 0, bd);
    return {a.lo, z.hi, z.lo, a.hi};
}

// the first token of a tree's prefix that a node at position pos sees; beyond P where the window ends inside the tree
__device__ __forceinline__ int32_t tree_lo(const ScoredParams& p, const ReqSpan& r, int32_t pos) {
    return p.window > 0 ? imax(imin(imax(pos, r.P), r.P + r.E - 1) - p.window + 1, 0) : 0;
}

// bits of the keys of a 32-key tile that a row sees
__device__ __forceinline__ uint32_t row_bits(const ScoredParams& p, const ReqSpan& r, int64_t t, int32_t lo, int32_t hi, int32_t base) {
    if (!p.mask) return range_bits(lo, hi, base);
    uint32_t bits = tree_bits(p.mask + t * p.words, p.words, r.P, hi, base) & ~low_bits(imin(lo, r.P) - base);
    if (lo > r.P)                                      // the window ends inside the tree: it counts positions, not nodes
        for (uint32_t left = bits; left; left &= left - 1) {
            const int k = __builtin_ctz(left);
            if (p.positions[r.q0 + (base + k - r.P)] < lo) bits &= ~(1u << k);
        }
    return bits;
}

// cap tanh(scale s / cap) log2(e) from the raw product s: tanh(x) = 1 - 2 / (1 + e^2x), exact at both ends (e^2x = 0 and inf);
// near 0 its absolute error is a unit or two of cap 2^-24, which is what counts in an exponent (hence no caps beyond 1024).
__device__ __forceinline__ float cap_score(const ScoredParams& p, float s) {
    return fmaf(-2.f * p.cap_log2, __builtin_amdgcn_rcpf(1.f + exp2_fast(s * p.cap_rate)), p.cap_log2);
}

// Infinities and NaN among the two 16-bit values of a dword: all exponent bits set.  Adding one to the exponent field then carries into
// the half's top bit, and only then - whole numbers without a compare, of which a tile needs hundreds at once.
template <bool F16>
__device__ __forceinline__ uint32_t exponent_carry(uint32_t w) {
    constexpr uint32_t field = F16 ? 0x7c007c00u : 0x7f807f80u, one = F16 ? 0x04000400u : 0x00800080u;
    return (w & field) + one;                          // bit 15 / 31: that half is not finite
}
template <bool F16>
__device__ __forceinline__ uint32_t nonfinite_halves(uint32_t w) { return ((exponent_carry<F16>(w) >> 15) & 0x00010001u) * 0xffffu; }
// Whether fragments hold any, at one instruction a dword: their greatest and least value, read as halves, in the order that NaN leads.  A
// bf16 infinity or NaN is a NaN as a half, and so are finite values from 2^121 up, for which the caller merely looks closer.
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
struct Extremes {
    f16x2 hi = {0, 0}, lo = {0, 0};
    __device__ __forceinline__ void add(bf16x8 f) {
        const u32x4 w = __builtin_bit_cast(u32x4, f);
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const uint32_t x = w[i], y = w[i + 1];     // (__builtin_bit_cast of w[i] itself would take element 0)
            const f16x2 a = __builtin_bit_cast(f16x2, x), b = __builtin_bit_cast(f16x2, y);
            hi = __builtin_elementwise_maximum(__builtin_elementwise_maximum(hi, a), b);
            lo = __builtin_elementwise_minimum(__builtin_elementwise_minimum(lo, a), b);
        }
    }
    __device__ __forceinline__ bool nonfinite() const {                  // in any lane of the wave
        return __any(((exponent_carry<true>(__builtin_bit_cast(uint32_t, hi)) | exponent_carry<true>(__builtin_bit_cast(uint32_t, lo))) & 0x80008000u) != 0);
    }
};
template <bool F16>
__device__ __forceinline__ bf16x8 frag_finite(bf16x8 f) {
    u32x4 w = __builtin_bit_cast(u32x4, f);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] &= ~nonfinite_halves<F16>(w[i]);
    return __builtin_bit_cast(bf16x8, w);
}
// the infinities and NaN of four consecutive values, 0 for the others
template <bool F16>
__device__ __forceinline__ f32x4 nonfinite4(uint2 w) {
    const uint32_t x = w.x & nonfinite_halves<F16>(w.x), y = w.y & nonfinite_halves<F16>(w.y);
    return f32x4{unpack16_lo<F16>(x), unpack16_hi<F16>(x), unpack16_lo<F16>(y), unpack16_hi<F16>(y)};
}

// s where bit `bit` of `seen` is set, -inf elsewhere
__device__ __forceinline__ float masked_score(float s, uint32_t seen, int bit) {
    const uint32_t keep = (uint32_t)((int32_t)(seen << (31 - bit)) >> 31);
    return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, s) & keep) | (0xff800000u & ~keep));
}

__device__ __forceinline__ int32_t slot_of(const ScoredParams& p, const int32_t* pt_row, int32_t tok) {
    const int32_t pg = p.ps_shift >= 0 ? tok >> p.ps_shift : tok / p.ps;
    return pool_slot(pt_row[pg], p.ps, tok - pg * p.ps, p.S);
}

}  // namespace m355
