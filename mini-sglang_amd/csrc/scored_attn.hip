// Attention over the paged KV pools with modified scores (no counterpart in the reference, whose backends run a plain causal
// softmax: torch_native_backend.py:25-193):
//
//     x[t, k] = scale q[t] . K[k];   x = cap tanh(x / cap) (cap > 0);   x -= slope[h] |pos(t) - pos(k)| (slopes)
//     out[t]  = sum_k softmax(x[t, .])_k V[k]  over the visible keys of row t;  zeros where the mask leaves nothing
//
// visible: an interval (causal, window, document start, bidirectional prefix: scored_rules.h visible_range) or, for a tree of
// drafted tokens, the prefix and the row's ancestors (tree_bits).
#include "scored_common.h"

namespace m355 {

// One wave per (query row, q head): lanes are keys in the score product and head-dim elements in the value sum.  Simple and
// right for every shape; each K/V row is read again by every row and head that sees it.
template <int D, bool F16>
__global__ __launch_bounds__(64) void scored_rows_kernel(const ScoredParams p) {
    __shared__ float qs[D], ps[64];
    __shared__ int32_t ss[64];
    const int lane = threadIdx.x, j = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const ReqSpan r = load_span(p, b);
    if (j >= r.E) return;
    const int64_t t = r.q0 + j;
    const int32_t* pt_row = table_row(p, b);
    const bool tree = p.mask != nullptr;
    int32_t pos = r.P + j;
    KeyRange v;
    if (tree) {
        v = {0, r.L};
        if (p.slopes) pos = (int32_t)p.positions[t];
    } else {
        v = visible_range(pos, r.L, p.window, p.doc_starts ? p.doc_starts[t] : 0, p.bidir ? p.bidir[b] : 0);
    }
    for (int d = lane; d < D; d += 64) {
        const uint32_t w = p.q[t * p.q_stride + (int64_t)h * D + d];
        qs[d] = unpack16_lo<F16>(w);
    }
    __syncthreads();
    const float slope = p.slopes ? p.slopes[h] : 0.f;
    const int64_t hoff = (int64_t)(h / p.G) * D;
    float m = -INFINITY, l = 0.f, o[D / 64];
    for (int x = 0; x < D / 64; ++x) o[x] = 0.f;
    for (int base = v.lo & ~31; base < v.hi; base += 64) {
        const int tok = base + lane;
        const int half = base + (lane & 32);
        const uint32_t bits = tree ? tree_bits(p.mask + t * p.words, p.words, r.P, v.hi, half) : range_bits(v.lo, v.hi, half);
        const bool seen = (bits >> (lane & 31)) & 1u;
        float s = -INFINITY;
        int32_t slot = 0;
        if (seen) {
            slot = slot_of(p, pt_row, tok);
            const uint16_t* kr = p.k_pool + (int64_t)slot * p.row_elems + hoff;
            float acc = 0.f;
            for (int c = 0; c < D / 8; ++c) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(kr + 8 * c);
                for (int y = 0; y < 4; ++y) acc += unpack16_lo<F16>(w[y]) * qs[8 * c + 2 * y] + unpack16_hi<F16>(w[y]) * qs[8 * c + 2 * y + 1];
            }
            s = acc * p.scale;
            if (p.cap > 0.f) s = p.cap * tanhf(s / p.cap);
            if (p.slopes) {
                const int32_t kp = tree && tok >= r.P ? (int32_t)p.positions[r.q0 + tok - r.P] : tok;
                s -= slope * fabsf((float)(pos - kp));
            }
        }
        float mt = s;
        for (int x = 32; x; x >>= 1) mt = fmaxf(mt, __shfl_xor(mt, x));
        const float mn = fmaxf(m, mt);
        const float mu = mn == -INFINITY ? 0.f : mn;
        const float alpha = exp2_fast((m - mu) * kLog2e);
        float e = exp2_fast((s - mu) * kLog2e);
        m = mn;
        ps[lane] = e;
        ss[lane] = seen ? slot : -1;
        for (int x = 32; x; x >>= 1) e += __shfl_xor(e, x);
        l = l * alpha + e;
        __syncthreads();
        for (int x = 0; x < D / 64; ++x) o[x] *= alpha;
        for (int k = 0; k < 64; ++k) {
            if (ss[k] < 0) continue;
            const uint16_t* vr = p.v_pool + (int64_t)ss[k] * p.row_elems + hoff;
            for (int x = 0; x < D / 64; ++x) o[x] += ps[k] * unpack16_lo<F16>((uint32_t)vr[lane + 64 * x]);
        }
        __syncthreads();
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    for (int x = 0; x < D / 64; ++x)
        p.out[t * p.o_stride + (int64_t)h * D + lane + 64 * x] = (uint16_t)(pack16<F16>(l == 0.f ? 0.f : o[x] * inv, 0.f) & 0xffffu);
}

static int shift_of(int32_t x) {
    if (x <= 0 || (x & (x - 1))) return -1;
    int s = 0;
    while ((1 << s) < x) ++s;
    return s;
}

// what both entry points refuse
static int check_common(const ScoredParams& p, int32_t max_extend_len, int32_t max_seq_len, int32_t D, int32_t dtype) {
    if (!p.q || !p.k_pool || !p.v_pool || !p.page_table || !p.page_table_ids || !p.out) return M355_ERR_INVALID_ARG;
    if (p.B < 0 || p.T < 0 || p.Hq <= 0 || p.Hkv <= 0 || p.Hq % p.Hkv || p.ps <= 0 || p.pt_rows <= 0 || p.pt_cols <= 0) return M355_ERR_INVALID_ARG;
    if (p.S <= 0 || p.S > 0x7fffffffLL || p.pt_stride < p.pt_cols || (int64_t)p.pt_cols * p.ps > 0x3fffffffLL) return M355_ERR_INVALID_ARG;
    if (max_extend_len <= 0 || max_seq_len <= 0 || p.window < 0) return M355_ERR_INVALID_ARG;
    if (!(p.scale > 0.f) || !(p.scale < 1e30f) || !(p.cap >= 0.f) || !(p.cap < 1e30f)) return M355_ERR_INVALID_ARG;
    if (dtype != M355_DTYPE_BF16 && dtype != M355_DTYPE_F16) return M355_ERR_UNSUPPORTED;
    if (D != 64 && D != 128) return M355_ERR_UNSUPPORTED;
    if (p.row_elems < (int64_t)p.Hkv * D || p.row_elems % 8) return M355_ERR_INVALID_ARG;
    if (((uintptr_t)p.q | (uintptr_t)p.k_pool | (uintptr_t)p.v_pool | (uintptr_t)p.out) & 15) return M355_ERR_INVALID_ARG;
    if (p.q_stride % 8 || p.o_stride % 8 || p.q_stride < (int64_t)p.Hq * D || p.o_stride < (int64_t)p.Hq * D) return M355_ERR_INVALID_ARG;
    return M355_OK;
}

static int launch_scored(const ScoredParams& p, int32_t max_extend_len, int32_t D, int32_t dtype, void* stream) {
    const dim3 grid((unsigned)max_extend_len, (unsigned)p.Hq, (unsigned)p.B);
    hipStream_t st = (hipStream_t)stream;
    const bool f16 = dtype == M355_DTYPE_F16;
    if (D == 64 && f16) hipLaunchKernelGGL((scored_rows_kernel<64, true>), grid, dim3(64), 0, st, p);
    else if (D == 64) hipLaunchKernelGGL((scored_rows_kernel<64, false>), grid, dim3(64), 0, st, p);
    else if (f16) hipLaunchKernelGGL((scored_rows_kernel<128, true>), grid, dim3(64), 0, st, p);
    else hipLaunchKernelGGL((scored_rows_kernel<128, false>), grid, dim3(64), 0, st, p);
    return check_launch();
}

}  // namespace m355

using namespace m355;

extern "C" int64_t m355_scored_workspace_bytes(int32_t B, int32_t T, int32_t Hq, int32_t Hkv, int32_t D, int32_t max_extend_len,
                                               int32_t max_seq_len_hint, int32_t window) {
    return 0;
}

extern "C" int m355_scored_attn(const void* q, int64_t q_row_stride, const void* k_pool, const void* v_pool, int64_t pool_row_stride,
                                int64_t S, const int32_t* page_table, int64_t pt_row_stride, int32_t pt_rows, int32_t pt_cols,
                                const int64_t* page_table_ids, const int64_t* seq_lens, const int64_t* prefix_lens,
                                const int32_t* cu_q, void* out, int64_t o_row_stride, int32_t B, int32_t T, int32_t max_extend_len,
                                int32_t max_seq_len_hint, int32_t Hq, int32_t Hkv, int32_t D, int32_t page_size, float scale,
                                float softcap, const float* slopes, int32_t window, const int32_t* doc_starts,
                                const int32_t* bidir_lens, void* workspace, int64_t workspace_bytes, int32_t dtype, void* stream) {
    if (T == 0 || B == 0) return M355_OK;
    if (!seq_lens || (prefix_lens == nullptr) != (cu_q == nullptr)) return M355_ERR_INVALID_ARG;
    ScoredParams p = {};
    p.q = (const uint16_t*)q; p.k_pool = (const uint16_t*)k_pool; p.v_pool = (const uint16_t*)v_pool;
    p.page_table = page_table; p.page_table_ids = page_table_ids; p.seq_lens = seq_lens; p.prefix_lens = prefix_lens; p.cu_q = cu_q;
    p.out = (uint16_t*)out; p.q_stride = q_row_stride; p.o_stride = o_row_stride;
    p.row_elems = pool_row_stride ? pool_row_stride : (int64_t)Hkv * D;
    p.pt_stride = pt_row_stride; p.S = S; p.pt_rows = pt_rows; p.pt_cols = pt_cols; p.B = B; p.T = T; p.Hq = Hq; p.Hkv = Hkv;
    p.ps = page_size; p.scale = scale; p.cap = softcap; p.slopes = slopes; p.window = window;
    p.doc_starts = doc_starts; p.bidir = bidir_lens;
    if (!cu_q && T < B) return M355_ERR_INVALID_ARG;
    if (const int e = check_common(p, max_extend_len, max_seq_len_hint, D, dtype)) return e;
    p.G = Hq / Hkv; p.ps_shift = shift_of(page_size);
    return launch_scored(p, cu_q ? max_extend_len : 1, D, dtype, stream);
}

extern "C" int m355_tree_attn(const void* q, int64_t q_row_stride, const void* k_pool, const void* v_pool, int64_t pool_row_stride,
                              int64_t S, const int32_t* page_table, int64_t pt_row_stride, int32_t pt_rows, int32_t pt_cols,
                              const int64_t* page_table_ids, const int64_t* prefix_lens, const int32_t* cu_q,
                              const uint32_t* tree_mask, int32_t mask_words, const int64_t* positions, void* out, int64_t o_row_stride,
                              int32_t B, int32_t T, int32_t max_nodes, int32_t max_seq_len_hint, int32_t Hq, int32_t Hkv, int32_t D,
                              int32_t page_size, float scale, float softcap, const float* slopes, void* workspace,
                              int64_t workspace_bytes, int32_t dtype, void* stream) {
    if (T == 0 || B == 0) return M355_OK;
    if (!prefix_lens || !cu_q || !tree_mask || mask_words <= 0 || (slopes && !positions)) return M355_ERR_INVALID_ARG;
    if ((int64_t)mask_words * 32 < max_nodes) return M355_ERR_INVALID_ARG;
    ScoredParams p = {};
    p.q = (const uint16_t*)q; p.k_pool = (const uint16_t*)k_pool; p.v_pool = (const uint16_t*)v_pool;
    p.page_table = page_table; p.page_table_ids = page_table_ids; p.prefix_lens = prefix_lens; p.cu_q = cu_q;
    p.out = (uint16_t*)out; p.q_stride = q_row_stride; p.o_stride = o_row_stride;
    p.row_elems = pool_row_stride ? pool_row_stride : (int64_t)Hkv * D;
    p.pt_stride = pt_row_stride; p.S = S; p.pt_rows = pt_rows; p.pt_cols = pt_cols; p.B = B; p.T = T; p.Hq = Hq; p.Hkv = Hkv;
    p.ps = page_size; p.scale = scale; p.cap = softcap; p.slopes = slopes;
    p.mask = tree_mask; p.words = mask_words; p.positions = positions;
    if (const int e = check_common(p, max_nodes, max_seq_len_hint, D, dtype)) return e;
    p.G = Hq / Hkv; p.ps_shift = shift_of(page_size);
    return launch_scored(p, max_nodes, D, dtype, stream);
}
