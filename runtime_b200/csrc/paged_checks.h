// Checks of the arguments that the entry points over paged caches share.
#pragma once

#include <initializer_list>

#include "mf_common.cuh"
#include "packed_kernels.h"

namespace mf {

inline int32_t check_pages(int32_t dtype, const PagedTable &pt, uint32_t kv_heads, uint32_t head_dim) {
    if (dtype < MF_PAGE_F32 || dtype > MF_PAGE_BF16) return fail(MF_INVALID_DTYPE, "unknown page dtype");
    if (kv_heads == 0 || head_dim == 0 || pt.page_tokens == 0)
        return fail(MF_INVALID_SHAPE, "page heads, head dimension and tokens must be nonzero");
    if (head_dim % 8 || head_dim > 128)
        return fail(MF_UNSUPPORTED, "paged attention takes head dimensions of 8 to 128 in steps of 8");
    if (kv_heads > 65536 || pt.page_tokens > (1u << 20))
        return fail(MF_OVERFLOW, "page geometry exceeds its limits");
    if ((uint64_t)pt.max_pages * pt.page_tokens > INT32_MAX || pt.pages > INT32_MAX)
        return fail(MF_OVERFLOW, "pages or positions exceed the 32-bit table");
    if (pt.pages * pt.page_tokens > (UINT32_MAX - 1) / kv_heads)
        return fail(MF_OVERFLOW, "rows of the pages exceed 32 bits");
    if (pt.sequences > (1u << 20)) return fail(MF_RESOURCE_LIMIT, "more than 2^20 sequences in one call");
    if (!pt.slot_ids && pt.sequences > pt.slots)
        return fail(MF_OUT_OF_BOUNDS, "more sequences than page-table slots");
    return MF_OK;
}

inline int32_t check_aligned(std::initializer_list<const void *> ptrs, uintptr_t bytes) {
    for (const void *p : ptrs)
        if (reinterpret_cast<uintptr_t>(p) % bytes)
            return fail(MF_INVALID_LAYOUT, bytes == 16 ? "device operands must be 16-byte aligned"
                                                       : "device operands must be 4-byte aligned");
    return MF_OK;
}

}  // namespace mf
