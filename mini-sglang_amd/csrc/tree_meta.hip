// Metadata of a batch of draft trees in one launch: the new pages enter the page table, every node gets its position
// (prefix + depth), its KV slot (the request's next slots in node order) and the mask of its ancestors.
//
// Whole numbers only; a few hundred nodes, so launch latency bounds it (1 tree of 8 nodes 2.8 us, 16 trees of 17 to 48 4.3, 4 of 64
// 4.8: three dependent trips to memory, then the climb in LDS).  One workgroup per request holds the parents in LDS;
// one thread per (node, mask word) climbs from the node towards the root - a parent is accepted only below its child, so
// every climb ends - and sets the bits that fall into its word.  No thread waits for another node's mask, which a
// row = parent's row | own bit recurrence would.
#include "scored_common.h"

namespace m355 {

constexpr int kMaxNodes = 1024;                       // M355_TREE_MAX_NODES

__global__ __launch_bounds__(256) void tree_prepare_kernel(int32_t* __restrict__ page_table, int64_t pt_stride, int32_t pt_rows, int32_t pt_cols,
                                                           const int64_t* __restrict__ page_table_ids, const int64_t* __restrict__ prefix_lens,
                                                           const int32_t* __restrict__ parents, const int32_t* __restrict__ cu_q,
                                                           const int32_t* __restrict__ new_pages, const int32_t* __restrict__ new_page_off,
                                                           int32_t new_page_count, int32_t T, int32_t ps, uint32_t* __restrict__ mask, int32_t words,
                                                           int64_t* __restrict__ positions, int64_t* __restrict__ out_cache_loc) {
    __shared__ int32_t par[kMaxNodes];
    const int b = blockIdx.x;
    // (length 0 stands in for the table's: the rows of the tree are what is wanted here)
    const ReqSpan r = req_span(cu_q[b], cu_q[b + 1], prefix_lens[b], 0, T, 0);
    const int n = imin(r.E, kMaxNodes), P = imax(r.P, 0);
    for (int j = threadIdx.x; j < n; j += 256) par[j] = parents[r.q0 + j];
    int64_t row = page_table_ids[b];
    const bool row_ok = row >= 0 && row < pt_rows;
    int32_t* const pt = page_table + (row_ok ? row : 0) * pt_stride;
    const int32_t first = (int32_t)(((int64_t)P + ps - 1) / ps);        // the first column the prefix does not use
    const int32_t off = new_pages ? imin(imax(new_page_off[b], 0), new_page_count) : 0;
    const int32_t* const fresh = new_pages + off;
    const int n_fresh = new_pages ? imin(imax(new_page_off[b + 1] - off, 0), new_page_count - off) : 0;
    if (row_ok)
        for (int i = threadIdx.x; i < n_fresh && first + i < pt_cols; i += 256) pt[first + i] = fresh[i];
    __syncthreads();
    for (int i = threadIdx.x; i < n * words; i += 256) {
        const int j = i / words, w = i - j * words;
        uint32_t bits = 0;
        int depth = 0;
        for (int a = j; a >= 0;) {
            if ((a >> 5) == w) bits |= 1u << (a & 31);
            const int up = par[a];
            if (up < 0 || up >= a) break;                                // the root, or not a parent
            ++depth;
            a = up;
            if (w && a < 32 * w) break;                                  // nothing further up falls into this word
        }
        mask[(int64_t)(r.q0 + j) * words + w] = bits;
        if (w == 0) {                                                    // (word 0 climbs the whole way)
            positions[r.q0 + j] = (int64_t)P + depth;
            const int32_t tok = P + j, col = tok / ps;
            int64_t loc = M355_NO_SLOT;
            if (row_ok && col < pt_cols) {
                const int32_t page = col >= first && col - first < n_fresh ? fresh[col - first] : pt[col];
                loc = (int64_t)page * ps + (tok - col * ps);
            }
            out_cache_loc[r.q0 + j] = loc;
        }
    }
}

}  // namespace m355

using namespace m355;

extern "C" int m355_tree_prepare(int32_t* page_table, int64_t pt_row_stride, int32_t pt_rows, int32_t pt_cols, const int64_t* page_table_ids,
                                 const int64_t* prefix_lens, const int32_t* parents, const int32_t* cu_q, const int32_t* new_pages,
                                 const int32_t* new_page_off, int32_t new_page_count, int32_t B, int32_t T, int32_t max_nodes, int32_t page_size,
                                 uint32_t* tree_mask, int32_t mask_words, int64_t* positions, int64_t* out_cache_loc, void* stream) {
    if (T == 0 || B == 0) return M355_OK;
    if (!page_table || !page_table_ids || !prefix_lens || !parents || !cu_q || !tree_mask || !positions || !out_cache_loc) return M355_ERR_INVALID_ARG;
    if (B < 0 || T < 0 || page_size <= 0 || pt_rows <= 0 || pt_cols <= 0 || pt_row_stride < pt_cols || max_nodes <= 0) return M355_ERR_INVALID_ARG;
    if ((new_pages == nullptr) != (new_page_off == nullptr) || new_page_count < 0) return M355_ERR_INVALID_ARG;
    if (mask_words <= 0 || (int64_t)mask_words * 32 < max_nodes) return M355_ERR_INVALID_ARG;
    if (max_nodes > kMaxNodes || mask_words > kMaxNodes / 32) return M355_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(tree_prepare_kernel, dim3((unsigned)B), dim3(256), 0, (hipStream_t)stream, page_table, pt_row_stride, pt_rows, pt_cols,
                       page_table_ids, prefix_lens, parents, cu_q, new_pages, new_page_off, new_page_count, T, page_size, tree_mask, mask_words, positions,
                       out_cache_loc);
    return check_launch();
}
