// Attention over the paged KV pools with modified scores (no counterpart in the reference, whose backends run a plain causal
// softmax: torch_native_backend.py:25-193):
//
//     x[t, k] = scale q[t] . K[k];   x = cap tanh(x / cap) (cap > 0);   x -= slope[h] |pos(t) - pos(k)| (slopes)
//     out[t]  = sum_k softmax(x[t, .])_k V[k]  over the visible keys of row t;  zeros where the mask leaves nothing
//
// visible: an interval (causal, window, document start, bidirectional prefix: scored_rules.h visible_range) or, for a tree of
// drafted tokens, the prefix and the row's ancestors (tree_bits), inside a window of positions.
//
// A query row is a (token, q head of the group) pair, token-major, so the G heads that share a kv head share its loads.  Two
// kernels, by the rows a request brings: scored_few_kernel (single tokens: HBM-bound) and scored_wide_kernel (long
// extends, trees: bound by the vector unit's exponentials and the matrix unit, short ones by HBM).  Both walk [lo_min, hi_max) of their
// rows only, in one pass with the running maximum and sum of the softmax, and cut that range into splits when there are too few row
// blocks for 256 CUs; scored_merge_kernel then joins the splits.  Nothing is accumulated by atomics: results do not depend on
// an order of arrival.
//
// Masked keys.  A mask is one 32-bit word per (row, tile of 32 keys), whatever made it, and is looked at in tiles that some row
// sees in part only.  Scores of masked keys become -inf, so what K holds there cannot matter; the weight 0 times an infinity
// or NaN in V would be NaN, so in those tiles V is looked through and, where something is found, infinities and NaN are taken out
// of the matrix product and added to the rows that do see the key.
#include "prefill_common.h"
#include "scored_common.h"
#include "stream_plan.h"

namespace m355 {

// (request, kv head) unit u as one share, without splits
__device__ __forceinline__ Share whole_request(const ScoredParams& p, int u) {
    Share s = {};
    s.any = true;
    s.b = u / p.Hkv; s.h = u % p.Hkv; s.nsp = 1; s.chunk = 0x3fffffc0;
    s.r = load_span(p, s.b);
    s.pt_row = table_row(p, s.b);
    return s;
}

// the range of the rows of 16 neighbouring lanes, in all of them
template <int CTRL>
__device__ __forceinline__ BlockRange join_dpp(BlockRange a) {
    const int lo = __builtin_amdgcn_update_dpp(a.lo_min, a.lo_min, CTRL, 0xF, 0xF, true), hi = __builtin_amdgcn_update_dpp(a.hi_max, a.hi_max, CTRL, 0xF, 0xF, true);
    const int lx = __builtin_amdgcn_update_dpp(a.lo_max, a.lo_max, CTRL, 0xF, 0xF, true), hn = __builtin_amdgcn_update_dpp(a.hi_min, a.hi_min, CTRL, 0xF, 0xF, true);
    return {imin(a.lo_min, lo), imax(a.hi_max, hi), imax(a.lo_max, lx), imin(a.hi_min, hn)};
}
__device__ __forceinline__ BlockRange join16(BlockRange a) {
    return join_dpp<kDppMirror>(join_dpp<kDppHalfMirror>(join_dpp<kDppXor2>(join_dpp<kDppXor1>(a))));
}

// softmax(-inf everywhere so far): the difference of two -inf would be NaN
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }

// Weights go into the second product rounded to the element type.  Half precision keeps 11 bits of a weight down to 2^-14 and nothing
// below 2^-25, while 100 000 keys of that weight sum to 2^-8 of the best one's.  So in half precision all weights are 2^7 times as large,
// which drops out of the softmax; with the lazy maximum's 2^8 they end at 2^15.  A key then loses 2^-32 of the best one's weight at most.
template <bool F16>
constexpr float kLift = F16 ? 7.f : 0.f;

// ------------------------------------------------------------------------------------------------------------------------
// Up to 16 rows (single tokens): a workgroup takes the rows of one (request, kv head) and one split of the keys.  Its two waves
// walk tiles of 32 keys on their own (tile 2 i + wave), each with its own two-stage LDS ring filled by LDS-DMA: K and V are read once,
// no barrier sits in the loop, and the waves' results meet in LDS at the end.
//   S^T[key, row]  = K[32 x D] . Q^T[D x 16]   v_mfma_f32_16x16x32: a lane owns one row and 8 of the tile's keys
//   O^T[d, row]   += V^T[D x 32] . P^T[32 x 16]   P^T is the S^T accumulator rounded in place, V^T is read transposed
// Bound by HBM.  Two waves: the LDS then holds two workgroups a CU at head_dim 128 and four at 64, whose starts and ends overlap
// (16 requests of 20 000 to 32 768 tokens, 222 MB: 40.6 us, 5.5 TB/s; with four waves 49.8, with one 58.7).  More rows go to
// the other kernel: with 32 rows here, 16 requests of 2 250 tokens took 45 us against 29.
// ------------------------------------------------------------------------------------------------------------------------
constexpr int kFewWaves = 2;
constexpr int kFewSlots = 1024;                       // tokens whose pool slots are in LDS at a time

enum { kPlain, kCapped, kBiased };                         // what scores go through: the scale alone, a cap, distances (capped or not)

template <int D, bool MOD, bool F16>
__global__ __launch_bounds__(64 * kFewWaves) void scored_few_kernel(const ScoredParams p) {
    using M = MG<D>;
    constexpr int NW = kFewWaves, NT = 64 * NW, PITCH = D + 4;
    constexpr int RING = 2 * NW * M::STAGEB, JOIN = NW * kFewRows * (PITCH + 2) * 4;
    static_assert(JOIN <= RING, "the waves' results fit where the rings were");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[RING];
    __shared__ int32_t slots[kFewSlots];
    const int wid = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4;

    const int u = blockIdx.x;                         // (without splits the kv head turns with the request: see find_share)
    const Share sh = p.slots ? find_share<kFewRows, true>(p) : whole_request(p, u - u % p.Hkv + (u + u / p.Hkv) % p.Hkv);
    if (!sh.any || sh.rb) return;
    const int h = sh.h, b = sh.b, sp = sh.sp;
    const ReqSpan r = sh.r;
    const int rows = imin(r.E * p.G, kFewRows);       // (more than max_extend_len promised: left out)
    if (rows == 0) return;
    const int32_t* pt_row = sh.pt_row;
    const bool ok = n < rows;
    const int j = ok ? n / p.G : 0, g = ok ? n - j * p.G : 0;
    const int64_t t = r.q0 + j;
    int32_t lo = 0, hi = r.L, pos = r.P + j;
    BlockRange br;
    if (p.mask) {
        if ((MOD && p.slopes) || p.window) pos = (int32_t)p.positions[t];
        lo = tree_lo(p, r, pos);
    } else {
        const KeyRange v = visible_range(pos, r.L, p.window, p.doc_starts ? p.doc_starts[t] : 0, p.bidir ? p.bidir[b] : 0);
        lo = v.lo; hi = v.hi;
    }
    if (!p.doc_starts) {
        br = block_range(p, r, b, 0, r.E - 1);
    } else {
        const bool some = ok && lo < hi;
        br = join16({some ? lo : 0x7fffffff, some ? hi : 0, ok ? lo : 0, ok ? hi : 0x7fffffff});
    }
    const int lo_min = __builtin_amdgcn_readfirstlane(br.lo_min), hi_max = __builtin_amdgcn_readfirstlane(br.hi_max);
    const int lo_max = __builtin_amdgcn_readfirstlane(br.lo_max), hi_min = __builtin_amdgcn_readfirstlane(br.hi_min);
    const int first = lo_min & ~31, keys = lo_min < hi_max ? hi_max - first : 0;
    const int active = imax(1, imin(sh.nsp, (keys + sh.chunk - 1) / sh.chunk));
    if (sp >= active) return;
    const int t0 = first + sp * sh.chunk, t1 = keys ? (sp == active - 1 ? hi_max : t0 + sh.chunk) : t0;
    const float slope = MOD && p.slopes ? p.slopes[h * p.G + g] * kLog2e : 0.f;

    bf16x8 qf[M::KS];
#pragma unroll
    for (int s = 0; s < M::KS; ++s) {
        u32x4 w = {0u, 0u, 0u, 0u};
        if (ok) w = *reinterpret_cast<const u32x4*>(p.q + t * p.q_stride + (int64_t)(h * p.G + g) * D + 32 * s + 8 * kg);
        qf[s] = __builtin_bit_cast(bf16x8, w);
    }
    f32x4 O[M::DT];
#pragma unroll
    for (int dt = 0; dt < M::DT; ++dt) O[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;

    // ---- per-lane constants of the DMA and of the LDS reads (stream_plan.h MG: chunk ch of a row sits at ch ^ s(row))
    const int drow = lane / M::C, dch = lane % M::C;
    uint8_t* const ring = smem + wid * 2 * M::STAGEB;
    const uint32_t ring0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)ring);
    const uint8_t* kbase = reinterpret_cast<const uint8_t*>(p.k_pool) + (int64_t)h * M::ROWB;
    const uint8_t* vbase = reinterpret_cast<const uint8_t*>(p.v_pool) + (int64_t)h * M::ROWB;
    const uint64_t row_bytes = (uint64_t)p.row_elems * 2;
    int koff[M::NI], voff[M::NI];
#pragma unroll
    for (int i = 0; i < M::NI; ++i) {
        koff[i] = 16 * (dch ^ M::sK(i * M::RPI + drow));
        voff[i] = 16 * (dch ^ M::sV(i * M::RPI + drow));
    }
    const int ka0 = n * M::ROWB + 16 * (kg ^ M::sK(n));
    const int vrow = 4 * kg + (n >> 2);
    const int va0 = vrow * M::ROWB + 16 * (M::sV(vrow) | ((n & 3) >> 1)) + 8 * (n & 1);

    int w0 = t0, wn = 0;                              // the slot window: tokens w0 .. w0 + wn
    auto issue = [&](const int tile, const int st) {
        uint64_t ro[M::NI];
#pragma unroll
        for (int i = 0; i < M::NI; ++i) ro[i] = (uint64_t)(uint32_t)slots[imin(32 * tile + i * M::RPI + drow, wn - 1)] * row_bytes;
#pragma unroll
        for (int i = 0; i < M::NI; ++i) {
            glds16p<1>(kbase + ro[i] + koff[i], ring0 + st * M::STAGEB + 1024 * i);
            glds16p<1>(vbase + ro[i] + voff[i], ring0 + st * M::STAGEB + M::TILEB + 1024 * i);
        }
    };
    auto v_frag = [&](const uint8_t* st, const int dt) {
        const uint8_t* va = st + M::TILEB + (va0 ^ (32 * dt));
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(uintptr_t)(uint32_t)(uintptr_t)va);
        const s16x4 c = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(uintptr_t)(uint32_t)(uintptr_t)(va + 16 * M::ROWB));
        return __builtin_bit_cast(bf16x8, s16x8{a[0], a[1], a[2], a[3], c[0], c[1], c[2], c[3]});
    };
    auto consume = [&](const int base, const int stage) {
        const uint8_t* st = ring + stage * M::STAGEB;
        f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < M::KS; ++s) {
            const bf16x8 a0 = *reinterpret_cast<const bf16x8*>(st + (ka0 ^ (64 * s)));
            const bf16x8 a1 = *reinterpret_cast<const bf16x8*>(st + 16 * M::ROWB + (ka0 ^ (64 * s)));
            s0 = mfma_16x16x32<F16>(a0, qf[s], s0);
            s1 = mfma_16x16x32<F16>(a1, qf[s], s1);
        }
        // this lane: row n, keys base + 4 kg + i and base + 16 + 4 kg + i
        float s[8] = {s0[0], s0[1], s0[2], s0[3], s1[0], s1[1], s1[2], s1[3]};
        if constexpr (MOD) {
            if (p.cap_log2 > 0.f) {
#pragma unroll
                for (int i = 0; i < 8; ++i) s[i] = cap_score(p, s[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) s[i] *= p.scale_log2;
            }
            if (p.slopes) {
                if (p.mask && base + 32 > r.P) {          // some keys are nodes: their positions are their depths
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int tok = base + 16 * (i >> 2) + 4 * kg + (i & 3);
                        const int kp = tok < r.P ? tok : (int)p.positions[r.q0 + imin(tok - r.P, r.E - 1)];
                        s[i] = fmaf(-slope, fabsf((float)(pos - kp)), s[i]);
                    }
                } else {
                    const float d = (float)(pos - base - 4 * kg);
#pragma unroll
                    for (int i = 0; i < 8; ++i) s[i] = fmaf(-slope, fabsf(d - (float)(16 * (i >> 2) + (i & 3))), s[i]);
                }
            }
        }
        const bool part = base < lo_max || base + 32 > hi_min;             // wave-uniform
        uint32_t bits = 0;
        bool bad = false;
        if (part) {
            bits = row_bits(p, r, t, lo, hi, base);
            const uint32_t w = bits >> (4 * kg);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = masked_score(s[i], w, 16 * (i >> 2) + (i & 3));
            Extremes of;
#pragma unroll
            for (int dt = 0; dt < M::DT; ++dt) of.add(v_frag(st, dt));
            bad = of.nonfinite();
        }
        float mx = s[0], a, c;
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i]);
        lane_pair<16>(mx, a, c);
        mx = fmaxf(a, c);
        lane_pair<32>(mx, a, c);
        mx = fmaxf(a, c);
        if constexpr (!MOD) mx *= p.scale_log2;
        // the running maximum moves only when beaten by 2^kLazyMax: rescaling is rare, weights stay below
        // 2^(kLazyMax + kLift)
        const float m_new = mx > m_run + kLazyMax ? mx : m_run;
        const float alpha = m_new == m_run ? 1.f : exp2_fast(m_run - m_new);
        m_run = m_new;
        const float mu = finite_max(m_new) - kLift<F16>;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) { s[i] = exp2_fast(MOD ? s[i] - mu : fmaf(s[i], p.scale_log2, -mu)); sum += s[i]; }
        l_run = fmaf(l_run, alpha, sum);
        if (__any(alpha != 1.f)) {
#pragma unroll
            for (int dt = 0; dt < M::DT; ++dt) O[dt] *= alpha;
        }
        // the weights go into the second product rounded to the element type, as the matrix unit takes them; their sum does not
        const bf16x8 pf = __builtin_bit_cast(bf16x8, u32x4{pack16<F16>(s[0], s[1]), pack16<F16>(s[2], s[3]), pack16<F16>(s[4], s[5]), pack16<F16>(s[6], s[7])});
#pragma unroll
        for (int dt = 0; dt < M::DT; ++dt) {
            bf16x8 av = v_frag(st, dt);
            if (bad) av = frag_finite<F16>(av);
            O[dt] = mfma_16x16x32<F16>(av, pf, O[dt]);
        }
        if (bad) {                                                         // rare: infinities and NaN, for the rows that see them
            for (int tk = 0; tk < 32; ++tk) {
                if (!((bits >> tk) & 1u)) continue;
                const uint8_t* vr = st + M::TILEB + tk * M::ROWB + 8 * (kg & 1);
#pragma unroll
                for (int dt = 0; dt < M::DT; ++dt)
                    O[dt] += nonfinite4<F16>(*reinterpret_cast<const uint2*>(vr + 16 * ((2 * dt + (kg >> 1)) ^ M::sV(tk))));
            }
        }
    };

    for (; w0 < t1; w0 += kFewSlots) {
        wn = imin(kFewSlots, t1 - w0);
        __syncthreads();
        for (int i = threadIdx.x; i < wn; i += NT) slots[i] = slot_of(p, pt_row, w0 + i);
        __syncthreads();
        const int nt = (wn + 31) >> 5;
        if (wid < nt) issue(wid, 0);
        for (int k = wid; k < nt; k += 2 * NW) {
            if (k + NW < nt) { issue(k + NW, 1); wait_vmcnt<2 * M::NI>(); } else wait_vmcnt<0>();
            consume(w0 + 32 * k, 0);
            if (k + NW >= nt) break;
            if (k + 2 * NW < nt) { issue(k + 2 * NW, 0); wait_vmcnt<2 * M::NI>(); } else wait_vmcnt<0>();
            consume(w0 + 32 * (k + NW), 1);
        }
    }

    // ---- the waves' results meet in LDS
    float* const jo = reinterpret_cast<float*>(smem);
    float* const jm = jo + NW * kFewRows * PITCH;                           // (m, l) per wave and row
    float a, c;
    lane_pair<16>(l_run, a, c);
    float l_sum = a + c;
    lane_pair<32>(l_sum, a, c);
    l_sum = a + c;
    __syncthreads();
    if (kg == 0) *reinterpret_cast<float2*>(jm + 2 * (wid * kFewRows + n)) = make_float2(m_run, l_sum);
#pragma unroll
    for (int dt = 0; dt < M::DT; ++dt) *reinterpret_cast<f32x4*>(jo + (wid * kFewRows + n) * PITCH + 16 * dt + 4 * kg) = O[dt];
    __syncthreads();
    constexpr int CH = D / 4;
    for (int i = threadIdx.x; i < rows * CH; i += NT) {
        const int m = i / CH, ch = i % CH;
        float mw[NW], mx = -INFINITY, l = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) { mw[w] = jm[2 * (w * kFewRows + m)]; mx = fmaxf(mx, mw[w]); }
        const float mu = finite_max(mx);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float e = exp2_fast(mw[w] - mu);
            l = fmaf(e, jm[2 * (w * kFewRows + m) + 1], l);
            o += *reinterpret_cast<const f32x4*>(jo + (w * kFewRows + m) * PITCH + 4 * ch) * e;
        }
        const int row = m / p.G, head = h * p.G + m - row * p.G;
        const int64_t item = (int64_t)(r.q0 + row) * p.Hq + head;
        if (active > 1) {
            float* wo = p.part + ((int64_t)(sh.part0 + sp) * kFewRows + m) * (D + 4);
            *reinterpret_cast<f32x4*>(wo + 4 * ch) = o;
            if (ch == 0) *reinterpret_cast<float2*>(wo + D) = make_float2(mx, l);
        } else {
            const float inv = 1.f / l;
            uint2 w = {0u, 0u};
            if (l != 0.f) w = make_uint2(pack16<F16>(o[0] * inv, o[1] * inv), pack16<F16>(o[2] * inv, o[3] * inv));
            *reinterpret_cast<uint2*>(p.out + (int64_t)(r.q0 + row) * p.o_stride + (int64_t)head * D + 4 * ch) = w;
        }
        if (sp == 0 && ch == 0 && p.slots) p.part_of[item] = make_int2(sh.part0 * kFewRows + m, active);
    }
}

// ------------------------------------------------------------------------------------------------------------------------
// Many rows: the four waves of a workgroup own 32 consecutive rows each of one (request, kv head) and walk the keys together, a
// pair of 32-key tiles at a time, brought into LDS once per workgroup by LDS-DMA (two pairs deep).  The matrix products are
// those of prefill_attn.hip (v_mfma_f32_32x32x16, a lane owns one row and 16 of a tile's keys); what differs is the score
// stage between them and the range that is walked.
//
// Bound by vector issue: per score a multiply-add, an exponential, a sum, half a maximum and half a conversion stand beside
// 4 D matrix flops; a cap puts two more transcendentals and two plain instructions on top.  A prompt of 8192 tokens (32 / 8 heads of
// 128): 590 us plain, 930 TFLOP/s, 694 capped (capping one tile beside the other's matrix product in source order, forced or
// not: within 1%; the SIMD's other wave already fills the gaps).  16 capped turns of 384 to 640 tokens over 1024 cached: 273
// us, 640 TFLOP/s, in four rounds of workgroups the last of which is partly empty.  Documents of ~700 tokens at head_dim 64: 127 us,
// 475 TFLOP/s against 780 without documents: some nine key pairs a block, of which the first and last are masked, and the
// block's start.  Eight waves a workgroup (256 rows) gained nothing.  Capped scores have a kernel apart from biased ones: in one, the
// registers of both spill at head_dim 128 (16 capped turns 279 us, 4 trees of 64 nodes over 20 000 to 32 000 tokens 59 for 53).
// ------------------------------------------------------------------------------------------------------------------------
template <int D, int MOD, bool F16, bool SPLIT>
__global__ __launch_bounds__(256, 2) void scored_wide_kernel(const ScoredParams p) {
    using W = WgCfg<D>;
    constexpr int NW = 4, NBUF = 4;
    constexpr int NT = 64 * NW, ROWS = 32 * NW, IPW = 2 * W::NI / NW, HP = IPW / 2;
    constexpr int NP = NBUF / 2;                      // pairs the ring holds: NP - 1 are on their way while one is worked on
    static_assert(IPW % 2 == 0 && W::NI % NW == 0 && NP == 2 && NBUF * W::TILEB <= 65536 && ROWS == kWideRows, "ring geometry");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[NBUF * W::BUFB];      // NBUF K tiles, NBUF V tiles
    __shared__ int32_t slotw[kSlotWin];
    __shared__ int32_t wlim[NW][2];
    const int wid = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int l = threadIdx.x & 63, c = l & 31, hh = l >> 5;

    // ---- which rows and keys.  Without splits: all row blocks of one (request, kv head), which walk much the same keys, on one XCD,
    // the last (longest under a causal mask) first; pairs left over after the full rounds of 8 are spread over all XCDs
    Share sh;
    if constexpr (SPLIT) {
        sh = find_share<ROWS, false>(p);
        if (!sh.any) return;
    } else {
        const int n_bh = p.B * p.Hkv, mapped = (n_bh >> 3) * 8 * p.blocks;
        int tb, bh;
        if ((int)blockIdx.x < mapped) {
            const int item = blockIdx.x >> 3;
            tb = p.blocks - 1 - item % p.blocks; bh = (item / p.blocks) * 8 + (blockIdx.x & 7);
        } else {
            const int item = blockIdx.x - mapped;
            tb = p.blocks - 1 - item % p.blocks; bh = (n_bh & ~7) + item / p.blocks;
        }
        sh = whole_request(p, bh);
        sh.rb = tb;
    }
    const int h = sh.h, b = sh.b, sp = sh.sp, tb = sh.rb;
    const ReqSpan r = sh.r;
    const int32_t* pt_row = sh.pt_row;
    const int rows = r.E * p.G;
    if (ROWS * tb >= rows) return;                                 // whole workgroup: no barrier has been reached yet

    // ---- this lane's row and the limits of its wave and workgroup
    const int row0 = ROWS * tb + 32 * wid, mrow = row0 + c;
    const bool valid = mrow < rows;
    const int j = valid ? mrow / p.G : 0, g = valid ? mrow - j * p.G : 0;
    const int32_t t = r.q0 + j;
    int32_t pos = r.P + j, lo = 0, hi = r.L;
    BlockRange br = {0x7fffffff, 0, 0, 0x7fffffff};                // the wave's rows
    if (p.mask) {
        if (MOD == kBiased || p.window) pos = (int32_t)p.positions[t];
        lo = tree_lo(p, r, pos);
    } else {
        const KeyRange v = visible_range(pos, r.L, p.window, p.doc_starts ? p.doc_starts[t] : 0, p.bidir ? p.bidir[b] : 0);
        lo = v.lo; hi = v.hi;
    }
    if (!p.doc_starts) {
        if (row0 < rows) br = block_range(p, r, b, row0 / p.G, imin(r.E - 1, (row0 + 31) / p.G));
    } else {
        if (valid) {
            if (lo < hi) { br.lo_min = lo; br.hi_max = hi; }
            br.lo_max = lo; br.hi_min = hi;
        }
        br = join16(br);
        br.lo_min = imin(br.lo_min, __shfl_xor(br.lo_min, 16)); br.hi_max = imax(br.hi_max, __shfl_xor(br.hi_max, 16));
        br.lo_max = imax(br.lo_max, __shfl_xor(br.lo_max, 16)); br.hi_min = imin(br.hi_min, __shfl_xor(br.hi_min, 16));
    }
    if (br.lo_min >= br.hi_max) { br.lo_min = 0x7fffffff; br.hi_max = 0; }
    if (p.doc_starts && l == 0) { wlim[wid][0] = br.lo_min; wlim[wid][1] = br.hi_max; }
    const int w_lo_min = __builtin_amdgcn_readfirstlane(br.lo_min), w_hi_max = __builtin_amdgcn_readfirstlane(br.hi_max);
    const int w_lo_max = __builtin_amdgcn_readfirstlane(br.lo_max), w_hi_min = __builtin_amdgcn_readfirstlane(br.hi_min);

    bf16x8 qf[W::KS];
    f32x16 o[W::DT];
    {
        const uint16_t* qp = p.q + (int64_t)t * p.q_stride + (int64_t)(h * p.G + g) * D + hh * 8;
#pragma unroll
        for (int s = 0; s < W::KS; ++s) {
            u32x4 v = u32x4{0u, 0u, 0u, 0u};
            if (valid) v = *reinterpret_cast<const u32x4*>(qp + s * 16);
            qf[s] = __builtin_bit_cast(bf16x8, v);
        }
#pragma unroll
        for (int dt = 0; dt < W::DT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
    }
    // a score in log2 units is unit * s, s being what `modify` leaves: a capped one is kept as -1 / (1 + e^2x), which is its tanh but for
    // a factor and a constant; the constant drops out of the softmax and the factor into the exponent's multiply-add
    const float unit = MOD == kPlain ? p.scale_log2 : MOD == kCapped || p.cap_log2 > 0.f ? 2.f * p.cap_log2 : 1.f;
    const float slope = MOD == kBiased ? p.slopes[h * p.G + g] * kLog2e / unit : 0.f;
    int lo_wg, hi_wg;
    if (p.doc_starts) {
        __syncthreads();
        lo_wg = wlim[0][0]; hi_wg = wlim[0][1];
#pragma unroll
        for (int x = 1; x < NW; ++x) { lo_wg = imin(lo_wg, wlim[x][0]); hi_wg = imax(hi_wg, wlim[x][1]); }
    } else {                                                       // (no barrier, and no wait for the q fragments, where the rows' ends tell)
        const BlockRange w = block_range(p, r, b, ROWS * tb / p.G, imin(r.E - 1, (ROWS * tb + ROWS - 1) / p.G));
        lo_wg = w.lo_min; hi_wg = w.hi_max;
    }
    lo_wg = __builtin_amdgcn_readfirstlane(lo_wg); hi_wg = __builtin_amdgcn_readfirstlane(hi_wg);
    const bool none = lo_wg >= hi_wg;
    const int pair0 = none ? 0 : lo_wg >> 6, pairs_end = none ? 0 : (hi_wg + 63) >> 6, n_tiles = (hi_wg + 31) >> 5;
    const int per = sh.chunk >> 6;
    const int active = SPLIT ? imax(1, imin(sh.nsp, (pairs_end - pair0 + per - 1) / per)) : 1;
    if (sp >= active) return;
    const int p_begin = pair0 + sp * per, n_pairs = sp == active - 1 ? pairs_end : p_begin + per;   // exclusive end

    // ---- DMA duty of this wave (see prefill_attn.hip): pieces of 1 KiB of the pair's K and V tiles
    const int drow = l / W::C, dch = l % W::C;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)smem);
    const uint8_t* kbase = reinterpret_cast<const uint8_t*>(p.k_pool) + (int64_t)h * W::ROWB;
    const uint8_t* vbase = reinterpret_cast<const uint8_t*>(p.v_pool) + (int64_t)h * W::ROWB;
    const uint64_t row_bytes = (uint64_t)p.row_elems * 2;
    int cur_win = -1;
    auto fill_slots = [&](int win) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kSlotWin / NT; ++k) {
            const int i = (int)threadIdx.x + NT * k;
            slotw[i] = slot_of(p, pt_row, imin(win * kSlotWin + i, hi_wg - 1));
        }
        __syncthreads();
        cur_win = win;
    };
    // a pair past the end fetches the last one again (masked, into a vacated buffer): every pair costs every wave the same
    // number of DMA instructions and the counted waits are static
    auto pair_slots = [&](int pair, int32_t (&sl)[IPW]) {
        pair = pair < n_pairs ? pair : n_pairs - 1;
        if ((2 * pair) / (kSlotWin / 32) != cur_win) fill_slots((2 * pair) / (kSlotWin / 32));   // workgroup-uniform
#pragma unroll
        for (int x = 0; x < IPW; ++x) {
            const int tile = 2 * pair + x / HP < n_tiles ? 2 * pair + x / HP : n_tiles - 1;
            sl[x] = slotw[((tile * 32) & (kSlotWin - 1)) + (wid + NW * (x % HP)) * W::RPI + drow];
        }
    };
    uint32_t kch[HP], vch[HP];
#pragma unroll
    for (int y = 0; y < HP; ++y) {
        const int row = (wid + NW * y) * W::RPI + drow;
        kch[y] = 16 * (dch ^ W::sK(row));
        vch[y] = 16 * (dch ^ W::sV(row));
    }
    auto piece = [&](const bool is_v, const int x, const int32_t slot, const int buf0) {
        const uint64_t off = (uint64_t)(uint32_t)slot * row_bytes + (is_v ? vch[x % HP] : kch[x % HP]);
        glds16p<M355_PREFILL_POLICY>((is_v ? vbase : kbase) + off,
               lds0 + (is_v ? NBUF * W::TILEB : 0) + (buf0 + x / HP) * W::TILEB + 1024 * (wid + NW * (x % HP)));
    };

    uint32_t kaddr[W::KS], vaddr[W::DT];
    {
        const int ksw = W::sK(c);
#pragma unroll
        for (int s = 0; s < W::KS; ++s) kaddr[s] = lds0 + c * W::ROWB + 16 * ((2 * s + hh) ^ ksw);
        const int gidx = l >> 4, li = l & 15;
        const int vr = 4 * hh + (li >> 2), vcol = 2 * (gidx & 1) + ((li & 3) >> 1);
#pragma unroll
        for (int dt = 0; dt < W::DT; ++dt)
            vaddr[dt] = lds0 + NBUF * W::TILEB + vr * W::ROWB + 16 * ((4 * dt + vcol) ^ W::sV(vr)) + 8 * (li & 1);
    }
    auto rdk = [&](const int buf, const int s) {
        return *reinterpret_cast<const bf16x8 __attribute__((address_space(3)))*>((uintptr_t)(kaddr[s] + buf * W::TILEB));
    };
    auto rdv = [&](const int buf, const int f) {
        const uint32_t a0 = vaddr[f >> 1] + buf * W::TILEB + 16 * (f & 1) * W::ROWB;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(uintptr_t)a0);
        const s16x4 e = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(uintptr_t)(a0 + 8 * W::ROWB));
        return __builtin_bit_cast(bf16x8, s16x8{a[0], a[1], a[2], a[3], e[0], e[1], e[2], e[3]});
    };
    // lane: keys base + (i & 3) + 8 (i >> 2) + 4 hh
    auto modify = [&](f32x16& s, const int base) {
        if (MOD == kCapped || p.cap_log2 > 0.f) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_rcpf(-1.f - exp2_fast(s[i] * p.cap_rate));
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] *= p.scale_log2;
        }
        if constexpr (MOD == kBiased) {
            if (p.mask && base + 32 > r.P) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int tok = base + (i & 3) + 8 * (i >> 2) + 4 * hh;
                    const int node = imin(imax(tok - r.P, 0), r.E - 1);
                    const int kp = tok < r.P ? tok : (int)p.positions[r.q0 + node];
                    s[i] = fmaf(-slope, fabsf((float)(pos - kp)), s[i]);
                }
            } else {
                const float d = (float)(pos - base - 4 * hh);
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = fmaf(-slope, fabsf(d - (float)((i & 3) + 8 * (i >> 2))), s[i]);
            }
        }
    };
    auto mask = [&](f32x16& s, const uint32_t bits) {
        const uint32_t w = bits >> (4 * hh);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = masked_score(s[i], w, (i & 3) + 8 * (i >> 2));
    };
    float m_run = -INFINITY, l_run = 0.f;
    auto new_max = [&](float mx) {
        float a, e;
        lane_pair<32>(mx, a, e);
        mx = fmaxf(a, e) * unit;
        const float m_new = mx > m_run + kLazy ? mx : m_run;
        const float alpha = m_new == m_run ? 1.f : exp2_fast(m_run - m_new);
        m_run = m_new;
        if (__any(alpha != 1.f)) {
#pragma unroll
            for (int dt = 0; dt < W::DT; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[dt][i] *= alpha;
        }
        return alpha;
    };
    auto exp_pack = [&](f32x16& s, bf16x8 (&pf)[2]) {
        const float mu = finite_max(m_run) - kLift<F16>;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) { s[i] = exp2_fast(fmaf(s[i], unit, -mu)); sum += s[i]; }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            u32x4 w;
#pragma unroll
            for (int x = 0; x < 4; ++x) w[x] = pack16<F16>(s[8 * ks + 2 * x], s[8 * ks + 2 * x + 1]);
            pf[ks] = __builtin_bit_cast(bf16x8, w);
        }
        return sum;
    };
    auto tile_max = [&](const f32x16& s) {
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
        return mx;
    };
    // infinities and NaN of a tile's V fragments: out of the product, into the rows that see them
    auto clean = [&](bf16x8 (&f)[W::KS], const int buf, const uint32_t bits) {
        Extremes of;
#pragma unroll
        for (int s = 0; s < W::KS; ++s) of.add(f[s]);
        if (!of.nonfinite()) return;
#pragma unroll
        for (int s = 0; s < W::KS; ++s) f[s] = frag_finite<F16>(f[s]);
        for (int tk = 0; tk < 32; ++tk) {
            if (!((bits >> tk) & 1u)) continue;
            const uint8_t* vr = smem + (NBUF + buf) * W::TILEB + tk * W::ROWB + 8 * hh;
#pragma unroll
            for (int dt = 0; dt < W::DT; ++dt)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    const f32x4 e = nonfinite4<F16>(*reinterpret_cast<const uint2*>(vr + 16 * ((4 * dt + q4) ^ W::sV(tk))));
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[dt][4 * q4 + i] += e[i];
                }
        }
    };

    auto pair_step = [&](const int k, auto pb_const) {
        constexpr int pb = decltype(pb_const)::value, nb = 2 * ((pb + NP - 1) % NP);
        wait_vmcnt<(NP - 2) * 2 * IPW>();                          // pair k has landed; NP - 2 younger pairs stay in flight
        __syncthreads();                                           // ... everybody's part of it, and everyone left pair k - 1
        int32_t sl[IPW];
        const int base_a = 64 * k, base_b = 64 * k + 32;
        if (base_a >= w_hi_max || base_a + 64 <= w_lo_min) {       // wave-uniform: nothing here for this wave's rows
            pair_slots(k + NP - 1, sl);
#pragma unroll
            for (int x = 0; x < IPW; ++x) { piece(false, x, sl[x], nb); piece(true, x, sl[x], nb); }
            return;
        }
        bf16x8 fa[W::KS], fb[W::KS], pa[2], pbk[2];
        f32x16 sa, sb;
#pragma unroll
        for (int s = 0; s < W::KS; ++s) fa[s] = rdk(2 * pb, s);
        pair_slots(k + NP - 1, sl);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 16; ++i) { sa[i] = 0.f; sb[i] = 0.f; }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int s = 0; s < W::KS; ++s) {                          // S_a^T; tile b's K fragments fill in behind
            sa = mfma_32x32x16<F16>(fa[s], qf[s], sa);
            fb[s] = rdk(2 * pb + 1, s);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < W::KS; ++s) {                          // S_b^T; tile a's V^T fragments take tile a's K registers
            sb = mfma_32x32x16<F16>(fb[s], qf[s], sb);
            fa[s] = rdv(2 * pb, s);
        }
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < IPW; ++x) piece(false, x, sl[x], nb);
        if constexpr (MOD != kPlain) { modify(sa, base_a); modify(sb, base_b); }
        const bool part = base_a < w_lo_max || base_a + 64 > w_hi_min;      // wave-uniform
        uint32_t bits_a = 0, bits_b = 0;
        if (part) {
            bits_a = row_bits(p, r, t, lo, hi, base_a);
            bits_b = row_bits(p, r, t, lo, hi, base_b);
            mask(sa, bits_a);
            mask(sb, bits_b);
        }
        const float alpha = new_max(fmaxf(tile_max(sa), tile_max(sb)));
        if (part) clean(fa, 2 * pb, bits_a);
#pragma unroll
        for (int x = 0; x < IPW; ++x) piece(true, x, sl[x], nb);
        float sum = exp_pack(sa, pa);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int s = 0; s < W::KS; ++s) {                          // O^T += V_a^T P_a^T; tile b's V^T fragments fill in behind
            o[s >> 1] = mfma_32x32x16<F16>(fa[s], pa[s & 1], o[s >> 1]);
            fb[s] = rdv(2 * pb + 1, s);
        }
        sum += exp_pack(sb, pbk);                                  // independent of the MFMAs above: interleaved with them
        __builtin_amdgcn_sched_barrier(0);
        if (part) clean(fb, 2 * pb + 1, bits_b);
#pragma unroll
        for (int s = 0; s < W::KS; ++s) o[s >> 1] = mfma_32x32x16<F16>(fb[s], pbk[s & 1], o[s >> 1]);
        __builtin_amdgcn_s_setprio(0);
        l_run = fmaf(l_run, alpha, sum);
    };
    if (!none) {
        fill_slots((2 * p_begin) / (kSlotWin / 32));
        wait_vmcnt<0>();                                           // q fragments are in: the DMA count starts clean
#pragma unroll
        for (int y = 0; y < NP - 1; ++y) {
            int32_t sl[IPW];
            pair_slots(p_begin + y, sl);
#pragma unroll
            for (int x = 0; x < IPW; ++x) { piece(false, x, sl[x], 2 * y); piece(true, x, sl[x], 2 * y); }
        }
        for (int k0 = p_begin; k0 < n_pairs; k0 += NP) {
            pair_step(k0, IntC<0>{});
            if (k0 + 1 < n_pairs) pair_step(k0 + 1, IntC<1>{});
        }
        wait_vmcnt<0>();                                           // the repeated fetch of the last pair must not outlive the wave
    }

    float la, lb;
    lane_pair<32>(l_run, la, lb);
    const float lt = la + lb;
    const int64_t item = (int64_t)t * p.Hq + h * p.G + g;
    if (!valid) return;
    const int prow = 32 * wid + c;                                 // row inside the block
    if (SPLIT && sp == 0 && hh == 0) p.part_of[item] = make_int2(sh.part0 * ROWS + prow, active);
    if (active > 1) {                                              // unnormalised partial of this split: O^T, m, l
        float* wo = p.part + ((int64_t)(sh.part0 + sp) * ROWS + prow) * (D + 4);
#pragma unroll
        for (int dt = 0; dt < W::DT; ++dt)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                *reinterpret_cast<f32x4*>(wo + 32 * dt + 8 * q4 + 4 * hh) =
                    f32x4{o[dt][4 * q4 + 0], o[dt][4 * q4 + 1], o[dt][4 * q4 + 2], o[dt][4 * q4 + 3]};
        if (hh == 0) { wo[D] = m_run; wo[D + 1] = lt; }
        return;
    }
    const float inv = 1.f / lt;
    uint16_t* op = p.out + (int64_t)t * p.o_stride + (int64_t)(h * p.G + g) * D + 4 * hh;
#pragma unroll
    for (int dt = 0; dt < W::DT; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            uint2 w = {0u, 0u};
            if (lt != 0.f) w = make_uint2(pack16<F16>(o[dt][4 * q4 + 0] * inv, o[dt][4 * q4 + 1] * inv),
                                          pack16<F16>(o[dt][4 * q4 + 2] * inv, o[dt][4 * q4 + 3] * inv));
            *reinterpret_cast<uint2*>(op + 32 * dt + 8 * q4) = w;
        }
}

// out[row, head, :] = sum_s O_s 2^(m_s - M) / sum_s l_s 2^(m_s - M) over the parts of a row, RB part rows apart.  D/4 lanes hold a
// row, four floats each; GROUPS of them take every GROUPS-th part with eight parts' loads in flight per lane, and meet in LDS.
// One group where there are rows enough to fill the chip, eight where there are not and the launch is a chain of latencies (128
// rows of 32 parts: 4.7 us against 5.9 with one; 4096 rows: 4.3 with one, 9.3 with eight).
template <int D, int RB, int GROUPS, bool F16>
__global__ __launch_bounds__(256) void scored_merge_kernel(const ScoredParams p) {
    constexpr int LPI = D / 4, CH = 8, PER = 256 / (LPI * GROUPS);  // rows of a workgroup
    __shared__ f32x4 jo[GROUPS > 1 ? 256 : 1];
    __shared__ float2 jm[GROUPS > 1 ? PER * GROUPS : 1];
    const int li = threadIdx.x % LPI, gr = threadIdx.x / LPI % GROUPS, slot = threadIdx.x / (LPI * GROUPS);
    const int64_t item = (int64_t)blockIdx.x * PER + slot;
    const int64_t row = item / p.Hq, head = item - row * p.Hq;
    const int64_t r0 = p.cu_q ? imax(p.cu_q[0], 0) : 0, r1 = p.cu_q ? imin(p.cu_q[p.B], p.T) : imin(p.B, p.T);
    const bool mine = row >= r0 && row < r1;                        // (rows of no request: left as they were)
    const int2 of = mine ? p.part_of[item] : make_int2(0, 0);
    // 1: written by the attention kernel.  (A row that no share reached - lengths that contradict cu_q - has no entry: nothing out of
    // the parts is read for it.)
    const int n = of.x < 0 || of.y <= 1 || of.x / RB + (int64_t)of.y > p.max_parts ? 0 : of.y;
    if (GROUPS == 1 && n == 0) return;
    const float* base = p.part + (int64_t)of.x * (D + 4);
    float mx = -INFINITY, den = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = gr; s0 < n; s0 += CH * GROUPS) {
        float2 ml[CH];
        f32x4 o[CH];
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            const float* ps = base + (int64_t)imin(s0 + k * GROUPS, n - 1) * (RB * (D + 4));
            ml[k] = *reinterpret_cast<const float2*>(ps + D);
            o[k] = *reinterpret_cast<const f32x4*>(ps + 4 * li);
        }
        float mn = mx;
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            if (s0 + k * GROUPS >= n) { ml[k] = make_float2(-INFINITY, 0.f); o[k] = f32x4{0.f, 0.f, 0.f, 0.f}; }
            mn = fmaxf(mn, ml[k].x);
        }
        const float mu = finite_max(mn), rs = exp2_fast(mx - mu);
        den *= rs;
        acc *= rs;
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            const float w = exp2_fast(ml[k].x - mu);
            den = fmaf(w, ml[k].y, den);
            acc += o[k] * w;
        }
        mx = mn;
    }
    if constexpr (GROUPS > 1) {
        jo[threadIdx.x] = acc;
        if (li == 0) jm[slot * GROUPS + gr] = make_float2(mx, den);
        __syncthreads();
        if (gr || n == 0) return;
        float mn = -INFINITY;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) mn = fmaxf(mn, jm[slot * GROUPS + g].x);
        const float mu = finite_max(mn);
        den = 0.f;
        acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            const float w = exp2_fast(jm[slot * GROUPS + g].x - mu);
            den = fmaf(w, jm[slot * GROUPS + g].y, den);
            acc += jo[(slot * GROUPS + g) * LPI + li] * w;
        }
    }
    const float inv = 1.f / den;
    uint2 w = {0u, 0u};
    if (den != 0.f) w = make_uint2(pack16<F16>(acc[0] * inv, acc[1] * inv), pack16<F16>(acc[2] * inv, acc[3] * inv));
    *reinterpret_cast<uint2*>(p.out + row * p.o_stride + head * D + 4 * li) = w;
}

// ------------------------------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------------------------------
static int shift_of(int32_t x) {
    if (x <= 0 || (x & (x - 1))) return -1;
    int s = 0;
    while ((1 << s) < x) ++s;
    return s;
}

// what both entry points refuse
static int check_args(const M355ScoredArgs& a) {
    if (!a.q || !a.k_pool || !a.v_pool || !a.page_table || !a.page_table_ids || !a.out) return M355_ERR_INVALID_ARG;
    if (a.B < 0 || a.T < 0 || a.Hq <= 0 || a.Hkv <= 0 || a.Hq % a.Hkv || a.page_size <= 0 || a.pt_rows <= 0 || a.pt_cols <= 0) return M355_ERR_INVALID_ARG;
    if (a.pool_rows <= 0 || a.pool_rows > 0x7fffffffLL || a.pt_row_stride < a.pt_cols || (int64_t)a.pt_cols * a.page_size > 0x3fffffffLL) return M355_ERR_INVALID_ARG;
    if (a.max_extend_len <= 0 || a.max_seq_len_hint <= 0 || a.window < 0) return M355_ERR_INVALID_ARG;
    if (!(a.scale > 0.f) || !(a.scale < 1e15f)) return M355_ERR_INVALID_ARG;
    if (a.softcap != 0.f && !(a.softcap >= 1.f / 1024 && a.softcap <= 1024.f)) return M355_ERR_INVALID_ARG;     // (NaN too)
    if (a.dtype != M355_DTYPE_BF16 && a.dtype != M355_DTYPE_F16) return M355_ERR_UNSUPPORTED;
    if (a.D != 64 && a.D != 128) return M355_ERR_UNSUPPORTED;
    const int64_t W = (int64_t)a.Hq * a.D, row = a.pool_row_stride ? a.pool_row_stride : (int64_t)a.Hkv * a.D;
    if (row < (int64_t)a.Hkv * a.D || row % 8) return M355_ERR_INVALID_ARG;
    if (((uintptr_t)a.q | (uintptr_t)a.k_pool | (uintptr_t)a.v_pool | (uintptr_t)a.out) & 15) return M355_ERR_INVALID_ARG;
    if (a.q_row_stride % 8 || a.o_row_stride % 8 || a.q_row_stride < W || a.o_row_stride < W) return M355_ERR_INVALID_ARG;
    return M355_OK;
}

template <int D, int RB, bool F16>
static void launch_merge(const ScoredParams& p, int64_t rows, hipStream_t st) {
    constexpr int LPI = D / 4;
    if (rows * LPI < 256 * 256) hipLaunchKernelGGL((scored_merge_kernel<D, RB, 8, F16>), dim3((unsigned)((rows * LPI * 8 + 255) / 256)), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((scored_merge_kernel<D, RB, 1, F16>), dim3((unsigned)((rows * LPI + 255) / 256)), dim3(256), 0, st, p);
}

template <int D, int MOD, bool F16>
static void launch_kernels(const ScoredParams& p, const ScoredCut& c, hipStream_t st) {
    if (c.wide) {
        if (p.slots) hipLaunchKernelGGL((scored_wide_kernel<D, MOD, F16, true>), dim3((unsigned)c.grid), dim3(256), 0, st, p);
        else hipLaunchKernelGGL((scored_wide_kernel<D, MOD, F16, false>), dim3((unsigned)c.grid), dim3(256), 0, st, p);
    } else {
        hipLaunchKernelGGL((scored_few_kernel<D, MOD != kPlain, F16>), dim3((unsigned)c.grid), dim3(64 * kFewWaves), 0, st, p);
    }
    if (p.slots) {
        const int64_t rows = (int64_t)p.T * p.Hq;
        if (c.wide) launch_merge<D, kWideRows, F16>(p, rows, st);
        else launch_merge<D, kFewRows, F16>(p, rows, st);
    }
}

static int launch_scored(const M355ScoredArgs& a, void* stream) {
    if (const int e = check_args(a)) return e;
    const int32_t ext = a.cu_q ? a.max_extend_len : 1;
    const ScoredCut c = scored_cut(a.B, a.T, a.Hq, a.Hkv, a.D, ext, a.max_seq_len_hint);
    if (c.bytes && (!a.workspace || a.workspace_bytes < c.bytes || ((uintptr_t)a.workspace & 255))) return M355_ERR_WORKSPACE;
    if (c.grid > 0x3fffffffLL || (int64_t)a.T * a.Hq * (a.D / 4) / 256 > 0x3fffffffLL) return M355_ERR_INVALID_ARG;
    ScoredParams p = {};
    p.q = (const uint16_t*)a.q; p.k_pool = (const uint16_t*)a.k_pool; p.v_pool = (const uint16_t*)a.v_pool;
    p.page_table = a.page_table; p.page_table_ids = a.page_table_ids; p.seq_lens = a.seq_lens; p.prefix_lens = a.prefix_lens; p.cu_q = a.cu_q;
    p.out = (uint16_t*)a.out; p.q_stride = a.q_row_stride; p.o_stride = a.o_row_stride;
    p.row_elems = a.pool_row_stride ? a.pool_row_stride : (int64_t)a.Hkv * a.D;
    p.pt_stride = a.pt_row_stride; p.S = a.pool_rows; p.pt_rows = a.pt_rows; p.pt_cols = a.pt_cols;
    p.B = a.B; p.T = a.T; p.Hq = a.Hq; p.Hkv = a.Hkv; p.G = a.Hq / a.Hkv; p.ps = a.page_size; p.ps_shift = shift_of(a.page_size);
    p.scale_log2 = a.scale * kLog2e; p.cap_log2 = a.softcap * kLog2e; p.cap_rate = a.softcap > 0.f ? 2.f * a.scale * kLog2e / a.softcap : 0.f;
    p.slopes = a.slopes; p.window = a.window; p.doc_starts = a.doc_starts; p.bidir = a.bidir_lens;
    p.mask = a.tree_mask; p.words = a.mask_words; p.positions = a.positions;
    p.blocks = c.blocks; p.slots = c.slots; p.max_parts = c.max_parts;
    if (c.bytes) { p.part = (float*)a.workspace; p.part_of = (int2*)((uint8_t*)a.workspace + c.part_bytes); }
    hipStream_t st = (hipStream_t)stream;
    const int mod = a.slopes ? kBiased : a.softcap > 0.f ? kCapped : kPlain;
    const bool f16 = a.dtype == M355_DTYPE_F16;
#define M355_SCORED(DD, MM, FF) if (a.D == DD && mod == MM && f16 == FF) { launch_kernels<DD, MM, FF>(p, c, st); return check_launch(); }
    M355_SCORED(64, kPlain, false) M355_SCORED(64, kCapped, false) M355_SCORED(64, kBiased, false)
    M355_SCORED(64, kPlain, true) M355_SCORED(64, kCapped, true) M355_SCORED(64, kBiased, true)
    M355_SCORED(128, kPlain, false) M355_SCORED(128, kCapped, false) M355_SCORED(128, kBiased, false)
    M355_SCORED(128, kPlain, true) M355_SCORED(128, kCapped, true) M355_SCORED(128, kBiased, true)
#undef M355_SCORED
    return M355_ERR_UNSUPPORTED;
}

}  // namespace m355

using namespace m355;

extern "C" int64_t m355_scored_workspace_bytes(int32_t B, int32_t T, int32_t Hq, int32_t Hkv, int32_t D, int32_t max_extend_len,
                                               int32_t max_seq_len_hint) {
    if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || max_extend_len <= 0 || max_seq_len_hint <= 0) return 0;
    return scored_cut(B, T, Hq, Hkv, D, max_extend_len, max_seq_len_hint).bytes;
}

extern "C" int m355_scored_attn(const M355ScoredArgs* args, void* stream) {
    if (!args) return M355_ERR_INVALID_ARG;
    const M355ScoredArgs& a = *args;
    if (a.T == 0 || a.B == 0) return M355_OK;
    if (!a.seq_lens || a.tree_mask || a.mask_words || (a.prefix_lens == nullptr) != (a.cu_q == nullptr)) return M355_ERR_INVALID_ARG;
    if (!a.cu_q && a.T < a.B) return M355_ERR_INVALID_ARG;
    return launch_scored(a, stream);
}

extern "C" int m355_tree_attn(const M355ScoredArgs* args, void* stream) {
    if (!args) return M355_ERR_INVALID_ARG;
    const M355ScoredArgs& a = *args;
    if (a.T == 0 || a.B == 0) return M355_OK;
    if (!a.prefix_lens || !a.cu_q || !a.tree_mask || a.mask_words <= 0 || (int64_t)a.mask_words * 32 < a.max_extend_len) return M355_ERR_INVALID_ARG;
    if (a.seq_lens || a.doc_starts || a.bidir_lens || ((a.slopes || a.window) && !a.positions)) return M355_ERR_INVALID_ARG;
    return launch_scored(a, stream);
}
