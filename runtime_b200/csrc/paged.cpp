// C-ABI entry points of the paged key/value cache and of sampling on device
// pointers: every argument the host can see is checked before any work.
#include <cuda_runtime.h>

#include <algorithm>
#include <new>
#include <vector>

#include "backend_internal.h"
#include "mf_common.cuh"
#include "packed_kernels.h"
#include "paged_checks.h"

using namespace mf;

extern "C" {

int32_t mfk_paged_append(void *key_pages, void *value_pages, int32_t page_dtype, uint64_t pages, uint32_t page_tokens,
                         const int32_t *page_table, uint32_t slots, uint32_t max_pages, const float *k, const float *v,
                         uint64_t tokens, const int32_t *starts, const int32_t *row_offsets, const int32_t *slot_ids,
                         uint32_t sequences, uint32_t kv_heads, uint32_t head_dim, void *stream) {
    PagedTable pt;
    pt.table = page_table, pt.slot_ids = slot_ids, pt.pages = pages, pt.slots = slots;
    pt.max_pages = max_pages, pt.page_tokens = page_tokens, pt.sequences = sequences;
    int32_t st = check_pages(page_dtype, pt, kv_heads, head_dim);
    if (st) return st;
    if (tokens > INT32_MAX) return fail(MF_OVERFLOW, "token rows exceed the 32-bit row offsets");
    if (!tokens || !sequences || !slots || !max_pages || !pages) return MF_OK;
    if (!key_pages || !value_pages || !page_table || !k || !v || !starts)
        return fail(MF_INVALID_ARGUMENT, "null device pointer");
    if (key_pages == value_pages) return fail(MF_INVALID_ARGUMENT, "key and value pages must have distinct storage");
    st = check_aligned({key_pages, value_pages, k, v}, 16);
    if (!st) st = check_aligned({page_table, starts, row_offsets, slot_ids}, 4);
    if (st) return st;
    return paged_append(key_pages, value_pages, page_dtype, pt, k, v, tokens, starts, row_offsets, kv_heads, head_dim,
                        (cudaStream_t)stream);
}

int32_t mfk_paged_gqa(float *out, const float *q, const void *key_pages, const void *value_pages, int32_t page_dtype,
                      uint64_t pages, uint32_t page_tokens, const int32_t *page_table, uint32_t slots,
                      uint32_t max_pages, const int32_t *lengths, const int32_t *slot_ids, uint32_t sequences,
                      uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, void *workspace, uint64_t workspace_bytes,
                      void *stream) {
    if (kv_heads == 0 || q_heads == 0 || q_heads % kv_heads)
        return fail(MF_INVALID_SHAPE, "query heads must be a nonzero multiple of key/value heads");
    PagedTable pt;
    pt.table = page_table, pt.slot_ids = slot_ids, pt.pages = pages, pt.slots = slots;
    pt.max_pages = max_pages, pt.page_tokens = page_tokens, pt.sequences = sequences;
    int32_t st = check_pages(page_dtype, pt, kv_heads, head_dim);
    if (st) return st;
    if ((uint64_t)sequences * q_heads > INT32_MAX / 128)
        return fail(MF_OVERFLOW, "query rows exceed the 32-bit work list");
    if (!sequences) return MF_OK;
    if (!out || !q || !lengths || !workspace || (slots && max_pages && pages && (!key_pages || !value_pages || !page_table)))
        return fail(MF_INVALID_ARGUMENT, "null device pointer");
    if (out == q) return fail(MF_INVALID_ARGUMENT, "paged attention output must not be its query");
    if (workspace_bytes < MF_PAGED_WORKSPACE_BYTES)
        return fail(MF_RESOURCE_LIMIT, "paged attention needs MF_PAGED_WORKSPACE_BYTES of workspace");
    st = check_aligned({out, q, key_pages, value_pages, workspace}, 16);
    if (!st) st = check_aligned({page_table, lengths, slot_ids}, 4);
    if (st) return st;
    if (!slots || !max_pages || !pages) pt.max_pages = 0;
    return paged_gqa(out, q, key_pages, value_pages, page_dtype, pt, lengths, q_heads, kv_heads, head_dim, workspace,
                     (cudaStream_t)stream);
}

int32_t mfk_copy_pages(void *const *pools, uint32_t n_pools, uint64_t pages, uint64_t page_bytes,
                       const uint32_t *sources, const uint32_t *destinations, uint64_t n, void *stream) {
    if (page_bytes == 0 || page_bytes % 16) return fail(MF_INVALID_LAYOUT, "a page must be a nonzero multiple of 16 bytes");
    if (pages > UINT64_MAX / page_bytes || pages > UINT32_MAX) return fail(MF_OVERFLOW, "pool size overflows");
    if (!n || !n_pools) return MF_OK;
    if (!pools || !sources || !destinations) return fail(MF_INVALID_ARGUMENT, "null argument");
    for (uint32_t p = 0; p < n_pools; ++p) {
        if (!pools[p]) return fail(MF_INVALID_ARGUMENT, "null device pointer");
        int32_t st = check_aligned({pools[p]}, 16);
        if (st) return st;
    }
    if (n > pages) return fail(MF_INVALID_ARGUMENT, "a page is the destination of two copies");
    for (uint64_t i = 0; i < n; ++i)
        if (sources[i] >= pages || destinations[i] >= pages)
            return fail(MF_OUT_OF_BOUNDS, "page id exceeds the pool's pages");
    try {
        bool twice = false, chained = false;
        if (n >= pages / 64) {
            std::vector<uint8_t> to(pages, 0);
            for (uint64_t i = 0; i < n; ++i) twice |= to[destinations[i]] != 0, to[destinations[i]] = 1;
            for (uint64_t i = 0; i < n; ++i) chained |= to[sources[i]] != 0;
        } else {  // few of many pages: no time for those that are not named
            std::vector<uint32_t> to(destinations, destinations + n);
            std::sort(to.begin(), to.end());
            twice = std::adjacent_find(to.begin(), to.end()) != to.end();
            for (uint64_t i = 0; i < n; ++i) chained |= std::binary_search(to.begin(), to.end(), sources[i]);
        }
        if (twice) return fail(MF_INVALID_ARGUMENT, "a page is the destination of two copies");
        if (chained) return fail(MF_INVALID_ARGUMENT, "a page is both source and destination");
    } catch (const std::bad_alloc &) {
        return fail(MF_RESOURCE_LIMIT, "host allocation failed");
    }
    return copy_pages(pools, n_pools, page_bytes, sources, destinations, n, (cudaStream_t)stream);
}

int32_t mfk_sample(float *out, const float *logits, uint64_t rows, uint64_t width, const float *temperature,
                   const int32_t *top_k, const float *top_p, const float *min_p, const float *uniform, void *stream) {
    if (!rows) return MF_OK;
    if (width == 0) return fail(MF_INVALID_SHAPE, "sampling needs a nonzero width");
    if (width > (1u << 24)) return fail(MF_OVERFLOW, "ids of more than 2^24 tokens are not exact in f32");
    if (rows >= INT32_MAX / 8) return fail(MF_OVERFLOW, "rows exceed the launch grid");
    if (!out || !logits || !temperature || !uniform) return fail(MF_INVALID_ARGUMENT, "null device pointer");
    int32_t st = check_aligned({out, logits, temperature, top_k, top_p, min_p, uniform}, 4);
    if (st) return st;
    // Rows are drawn in any order, and the order is found from every row's top_k and top_p.
    bool clash = overlap(out, rows * 4, logits, rows * width * 4) || overlap(out, rows * 4, top_k, rows * 4) ||
                 overlap(out, rows * 4, top_p, rows * 4);
    for (const float *own : {temperature, min_p, uniform}) clash |= own != out && overlap(out, rows * 4, own, rows * 4);
    if (clash) return fail(MF_INVALID_ARGUMENT, "sampling output overlaps an input");
    SampleSettings set;
    set.temperature = temperature, set.top_k = top_k, set.top_p = top_p, set.min_p = min_p, set.uniform = uniform;
    return sample(out, logits, rows, width, set, (cudaStream_t)stream);
}

}  // extern "C"
