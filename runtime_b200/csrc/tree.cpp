// C-ABI entry points of drafted trees on device pointers: every argument the
// host can see is checked before any work.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "backend_internal.h"
#include "mf_common.cuh"
#include "packed_kernels.h"
#include "paged_checks.h"

using namespace mf;

namespace {

PagedTable table_of(const int32_t *page_table, const int32_t *slot_ids, uint64_t pages, uint32_t slots, uint32_t max_pages,
                    uint32_t page_tokens, uint32_t sequences) {
    PagedTable pt;
    pt.table = page_table, pt.slot_ids = slot_ids, pt.pages = pages, pt.slots = slots;
    pt.max_pages = max_pages, pt.page_tokens = page_tokens, pt.sequences = sequences;
    return pt;
}

// An operand's bytes.
struct Span {
    const void *ptr;
    uint64_t bytes;
};

bool overlaps_any(Span out, std::initializer_list<Span> others) {
    for (const Span &s : others)
        if (overlap(out.ptr, out.bytes, s.ptr, s.bytes)) return true;
    return false;
}

int32_t check_convolution(uint32_t slots, uint64_t tokens, const int32_t *slot_ids, uint32_t sequences, uint32_t hidden,
                          uint32_t width) {
    if (hidden == 0 || width == 0)
        return fail(MF_INVALID_ARGUMENT, "short convolution hidden width and kernel width must be nonzero");
    if (width > 16) return fail(MF_UNSUPPORTED, "tree convolution takes kernel widths up to 16");
    if (hidden > (1u << 24)) return fail(MF_OVERFLOW, "short convolution hidden width exceeds its limit");
    if (tokens > INT32_MAX) return fail(MF_OVERFLOW, "token rows exceed the 32-bit row offsets");
    if (sequences > (1u << 20)) return fail(MF_RESOURCE_LIMIT, "more than 2^20 sequences in one call");
    if (!slot_ids && sequences > slots) return fail(MF_OUT_OF_BOUNDS, "more sequences than history slots");
    return MF_OK;
}

}  // namespace

extern "C" {

int32_t mfk_paged_append_rope(void *key_pages, void *value_pages, int32_t page_dtype, uint64_t pages,
                              uint32_t page_tokens, const int32_t *page_table, uint32_t slots, uint32_t max_pages,
                              float *q_out, const float *q, const float *k, const float *v, uint64_t tokens,
                              const float *q_weight, const float *k_weight, float epsilon, float theta,
                              const int32_t *positions, const int32_t *starts, const int32_t *row_offsets,
                              const int32_t *slot_ids, uint32_t sequences, uint32_t q_heads, uint32_t kv_heads,
                              uint32_t head_dim, void *stream) {
    PagedTable pt = table_of(page_table, slot_ids, pages, slots, max_pages, page_tokens, sequences);
    int32_t st = check_pages(page_dtype, pt, kv_heads, head_dim);
    if (st) return st;
    if (q_heads > 65536) return fail(MF_OVERFLOW, "page geometry exceeds its limits");
    if (!(theta > 0.0f) || std::isinf(theta)) return fail(MF_INVALID_ARGUMENT, "RoPE theta must be finite and positive");
    if ((q_weight || k_weight) && (!(epsilon > 0.0f) || std::isinf(epsilon)))
        return fail(MF_INVALID_ARGUMENT, "RMS epsilon must be finite and positive");
    if (tokens > INT32_MAX) return fail(MF_OVERFLOW, "token rows exceed the 32-bit row offsets");
    if (!tokens || !sequences) return MF_OK;
    const bool nowhere = !slots || !max_pages || !pages;  // no place exists
    if (!k || !v || !starts || (q_heads && (!q || !q_out)) || (!nowhere && (!key_pages || !value_pages || !page_table)))
        return fail(MF_INVALID_ARGUMENT, "null device pointer");
    if (!nowhere && key_pages == value_pages)
        return fail(MF_INVALID_ARGUMENT, "key and value pages must have distinct storage");
    st = check_aligned({key_pages, value_pages, q_out, q, k, v, q_weight, k_weight}, 16);
    if (!st) st = check_aligned({page_table, positions, starts, row_offsets, slot_ids}, 4);
    if (st) return st;
    const uint64_t q_bytes = tokens * q_heads * head_dim * 4, kv_bytes = tokens * kv_heads * head_dim * 4,
                   head_bytes = head_dim * 4ull;
    const uint64_t pool = pages * kv_heads * page_tokens * head_dim * (page_dtype == MF_PAGE_F32 ? 4 : 2);
    const Span out{q_heads ? q_out : nullptr, q_bytes};
    const std::initializer_list<Span> inputs = {{k, kv_bytes},           {v, kv_bytes},
                                                {q_weight, head_bytes},  {k_weight, head_bytes},
                                                {positions, tokens * 4}, {starts, sequences * 4ull},
                                                {row_offsets, sequences * 4ull + 4}, {slot_ids, sequences * 4ull},
                                                {page_table, (uint64_t)slots * max_pages * 4}};
    if (overlaps_any(out, inputs) || (q != q_out && overlap(out.ptr, q_bytes, q, q_bytes)) ||
        overlaps_any({key_pages, pool}, inputs) || overlaps_any({value_pages, pool}, inputs) ||
        overlaps_any({q_heads ? q : nullptr, q_bytes}, {{key_pages, pool}, {value_pages, pool}}) ||
        overlaps_any(out, {{key_pages, pool}, {value_pages, pool}}) || overlap(key_pages, pool, value_pages, pool))
        return fail(MF_INVALID_ARGUMENT, "an output of the rotated append overlaps another operand");
    if (nowhere) pt.max_pages = 0;
    return paged_append_rope(key_pages, value_pages, page_dtype, pt, q_out, q, k, v, tokens, q_weight, k_weight, epsilon,
                             theta, positions, starts, row_offsets, q_heads, kv_heads, head_dim, (cudaStream_t)stream);
}

int32_t mfk_paged_tree_gqa(float *out, const float *q, const void *key_pages, const void *value_pages,
                           int32_t page_dtype, uint64_t pages, uint32_t page_tokens, const int32_t *page_table,
                           uint32_t slots, uint32_t max_pages, uint64_t tokens, const int32_t *lengths,
                           const int32_t *row_offsets, const int32_t *parents, const int32_t *slot_ids,
                           uint32_t sequences, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, void *workspace,
                           uint64_t workspace_bytes, void *stream) {
    if (kv_heads == 0 || q_heads == 0 || q_heads % kv_heads)
        return fail(MF_INVALID_SHAPE, "query heads must be a nonzero multiple of key/value heads");
    PagedTable pt = table_of(page_table, slot_ids, pages, slots, max_pages, page_tokens, sequences);
    int32_t st = check_pages(page_dtype, pt, kv_heads, head_dim);
    if (st) return st;
    if (tokens > INT32_MAX || tokens * q_heads > INT32_MAX)
        return fail(MF_OVERFLOW, "query rows exceed the 32-bit work list");
    if (!tokens || !sequences) return MF_OK;
    const bool nowhere = !slots || !max_pages || !pages;
    if (!out || !q || !lengths || !workspace || (!nowhere && (!key_pages || !value_pages || !page_table)))
        return fail(MF_INVALID_ARGUMENT, "null device pointer");
    if (workspace_bytes < MF_PAGED_TREE_WORKSPACE_BYTES)
        return fail(MF_RESOURCE_LIMIT, "tree attention needs MF_PAGED_TREE_WORKSPACE_BYTES of workspace");
    st = check_aligned({out, q, key_pages, value_pages, workspace}, 16);
    if (!st) st = check_aligned({page_table, lengths, row_offsets, parents, slot_ids}, 4);
    if (st) return st;
    const uint64_t bytes = tokens * q_heads * head_dim * 4;
    const uint64_t pool = pages * kv_heads * page_tokens * head_dim * (page_dtype == MF_PAGE_F32 ? 4 : 2);
    const std::initializer_list<Span> inputs = {{q, bytes},
                                                {key_pages, pool},
                                                {value_pages, pool},
                                                {lengths, sequences * 4ull},
                                                {row_offsets, sequences * 4ull + 4},
                                                {parents, tokens * 4},
                                                {slot_ids, sequences * 4ull},
                                                {page_table, (uint64_t)slots * max_pages * 4}};
    if (overlaps_any({out, bytes}, inputs) || overlaps_any({workspace, workspace_bytes}, inputs) ||
        overlap(out, bytes, workspace, workspace_bytes))
        return fail(MF_INVALID_ARGUMENT, "tree attention output or workspace overlaps another operand");
    if (nowhere) pt.max_pages = 0;
    return paged_tree_gqa(out, q, key_pages, value_pages, page_dtype, pt, tokens, lengths, row_offsets, parents, q_heads,
                          kv_heads, head_dim, workspace, (cudaStream_t)stream);
}

int32_t mfk_tree_convolution(float *out, const float *projection, const float *kernel, const float *history,
                             uint32_t slots, uint64_t tokens, const int32_t *row_offsets, const int32_t *parents,
                             const int32_t *slot_ids, uint32_t sequences, uint32_t hidden, uint32_t width, void *stream) {
    int32_t st = check_convolution(slots, tokens, slot_ids, sequences, hidden, width);
    if (st) return st;
    if (!tokens || !sequences) return MF_OK;
    const uint64_t entries = (uint64_t)slots * (width - 1) * hidden;
    if (!out || !projection || !kernel || (entries && !history)) return fail(MF_INVALID_ARGUMENT, "null device pointer");
    st = check_aligned({out, projection, history}, hidden % 4 ? 4 : 16);
    if (!st) st = check_aligned({kernel, row_offsets, parents, slot_ids}, 4);
    if (st) return st;
    if (overlaps_any({out, tokens * hidden * 4}, {{projection, tokens * hidden * 12},
                                                  {kernel, (uint64_t)hidden * width * 4},
                                                  {history, entries * 4},
                                                  {row_offsets, sequences * 4ull + 4},
                                                  {parents, tokens * 4},
                                                  {slot_ids, sequences * 4ull}}))
        return fail(MF_INVALID_ARGUMENT, "tree convolution output overlaps an input");
    return tree_convolution(out, projection, kernel, history, slots, tokens, row_offsets, parents, slot_ids, sequences,
                            hidden, width, (cudaStream_t)stream);
}

int32_t mfk_tree_convolution_keep(float *history_out, const float *history, uint32_t slots, const float *projection,
                                  uint64_t tokens, const int32_t *paths, const int32_t *counts,
                                  const int32_t *row_offsets, const int32_t *slot_ids, uint32_t sequences,
                                  uint32_t hidden, uint32_t width, void *stream) {
    int32_t st = check_convolution(slots, tokens, slot_ids, sequences, hidden, width);
    if (st) return st;
    if (!sequences || !slots || width == 1) return MF_OK;
    if (!history_out || !history || !counts || (tokens && (!projection || !paths)))
        return fail(MF_INVALID_ARGUMENT, "null device pointer");
    st = check_aligned({history_out, history, projection, paths, counts, row_offsets, slot_ids}, 4);
    if (st) return st;
    const uint64_t bytes = (uint64_t)slots * (width - 1) * hidden * 4;
    if ((history_out != history && overlap(history_out, bytes, history, bytes)) ||
        overlaps_any({history_out, bytes}, {{projection, tokens * hidden * 12},
                                            {paths, tokens * 4},
                                            {counts, sequences * 4ull},
                                            {row_offsets, sequences * 4ull + 4},
                                            {slot_ids, sequences * 4ull}}))
        return fail(MF_INVALID_ARGUMENT, "tree convolution history overlaps another operand");
    return tree_convolution_keep(history_out, history, slots, projection, tokens, paths, counts, row_offsets, slot_ids,
                                 sequences, hidden, width, (cudaStream_t)stream);
}

int32_t mfk_paged_accept(int32_t *paths, int32_t *counts, float *next, void *const *pools, uint32_t n_pools,
                         int32_t page_dtype, uint64_t pages, uint32_t page_tokens, const int32_t *page_table,
                         uint32_t slots, uint32_t max_pages, const float *drafted, const float *sampled,
                         uint64_t tokens, const int32_t *starts, const int32_t *row_offsets, const int32_t *parents,
                         const int32_t *slot_ids, uint32_t sequences, uint32_t kv_heads, uint32_t head_dim,
                         void *stream) {
    PagedTable pt = table_of(page_table, slot_ids, pages, slots, max_pages, page_tokens, sequences);
    if (!n_pools) pt = table_of(nullptr, nullptr, 0, 0, 0, 1, sequences);  // nothing moves
    int32_t st = n_pools ? check_pages(page_dtype, pt, kv_heads, head_dim) : MF_OK;
    if (st) return st;
    if (tokens > INT32_MAX) return fail(MF_OVERFLOW, "token rows exceed the 32-bit row offsets");
    if (sequences > (1u << 20)) return fail(MF_RESOURCE_LIMIT, "more than 2^20 sequences in one call");
    if (!sequences) return MF_OK;
    const bool nowhere = !slots || !max_pages || !pages;
    if (!counts || !next || (tokens && (!paths || !drafted || !sampled)) ||
        (n_pools && (!pools || !starts || (!nowhere && !page_table))))
        return fail(MF_INVALID_ARGUMENT, "null device pointer");
    for (uint32_t p = 0; p < n_pools; ++p) {
        if (!nowhere && !pools[p]) return fail(MF_INVALID_ARGUMENT, "null device pointer");
        if ((st = check_aligned({pools[p]}, 16))) return st;
    }
    st = check_aligned({paths, counts, next, page_table, drafted, sampled, starts, row_offsets, parents, slot_ids}, 4);
    if (st) return st;
    const uint64_t rows = tokens * 4, seqs = sequences * 4ull;
    const std::initializer_list<Span> inputs = {{drafted, rows},
                                                {sampled, rows},
                                                {starts, seqs},
                                                {row_offsets, seqs + 4},
                                                {parents, rows},
                                                {slot_ids, seqs},
                                                {n_pools ? page_table : nullptr, (uint64_t)slots * max_pages * 4}};
    bool clash = overlaps_any({paths, rows}, inputs) || overlaps_any({counts, seqs}, inputs) ||
                 overlaps_any({next, seqs}, inputs) || overlaps_any({paths, rows}, {{counts, seqs}, {next, seqs}}) ||
                 overlap(counts, seqs, next, seqs);
    const uint64_t pool = pages * kv_heads * page_tokens * head_dim * (page_dtype == MF_PAGE_F32 ? 4 : 2);
    for (uint32_t p = 0; p < n_pools && !nowhere; ++p)
        clash |= overlaps_any({pools[p], pool}, inputs) || overlaps_any({pools[p], pool}, {{paths, rows}, {counts, seqs}, {next, seqs}});
    try {
        std::vector<uintptr_t> at(nowhere ? 0 : n_pools);  // (a pool named twice would move twice)
        for (size_t p = 0; p < at.size(); ++p) at[p] = reinterpret_cast<uintptr_t>(pools[p]);
        std::sort(at.begin(), at.end());
        for (size_t p = 1; p < at.size(); ++p) clash |= at[p] - at[p - 1] < pool;
    } catch (const std::bad_alloc &) {
        return fail(MF_RESOURCE_LIMIT, "host allocation failed");
    }
    if (clash) return fail(MF_INVALID_ARGUMENT, "an output of the acceptance overlaps another operand");
    if (nowhere) pt.max_pages = 0;
    return paged_accept(paths, counts, next, pools, n_pools, page_dtype, pt, drafted, sampled, tokens, starts,
                        row_offsets, parents, kv_heads ? kv_heads : 1, head_dim, (cudaStream_t)stream);
}

}  // extern "C"
