// What the kernels over paged caches share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "packed_kernels.h"

namespace mf {

// One value in the page's type, rounded to nearest even.
__device__ __forceinline__ void page_round(float &o, float v) { o = v; }
__device__ __forceinline__ void page_round(__half &o, float v) { o = __float2half_rn(v); }
__device__ __forceinline__ void page_round(__nv_bfloat16 &o, float v) { o = __float2bfloat16_rn(v); }

// The last of `n` offsets (the first is taken as at or before `row`) that is
// at or before `row`: 32 places at a time, by a whole warp.
__device__ __forceinline__ uint32_t last_offset_before(const int32_t *offsets, uint32_t n, int64_t row) {
    const uint32_t lane = threadIdx.x & 31;
    uint32_t lo = 0, hi = n;  // the answer lies in [lo, hi)
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 31) / 32, at = lo + lane * step;
        const bool before = at < hi && (lane == 0 || offsets[at] <= row);
        const uint32_t last = 31 - __clz(__ballot_sync(0xffffffffu, before));
        hi = min(hi, lo + (last + 1) * step);
        lo += last * step;
    }
    return lo;
}

// The rows of a sequence: [first, first + n).
struct SequenceRows {
    int64_t first;
    uint32_t n;
};
// Of offsets that are cut to [0, tokens).
__device__ __forceinline__ SequenceRows rows_between(int32_t begin, int32_t end, uint64_t tokens) {
    const int64_t first = min((int64_t)max(begin, 0), (int64_t)tokens);
    return {first, (uint32_t)max((int64_t)0, min((int64_t)end, (int64_t)tokens) - first)};
}
// Without offsets each sequence has one row.
__device__ __forceinline__ SequenceRows rows_of(const int32_t *offsets, uint32_t seq, uint64_t tokens) {
    if (!offsets) return {(int64_t)seq, seq < tokens};
    return rows_between(offsets[seq], offsets[seq + 1], tokens);
}
// The sequence that has `row`, and its rows; false where none has.  (By a whole warp.)
__device__ __forceinline__ bool sequence_of(const int32_t *offsets, uint32_t sequences, uint64_t tokens, int64_t row,
                                            uint32_t &seq, SequenceRows &rows) {
    seq = (uint32_t)row;
    if (offsets) {
        seq = last_offset_before(offsets, sequences, row);
        while (seq + 1 < sequences && offsets[seq + 1] <= row) ++seq;
    } else if (row >= (int64_t)sequences) {
        return false;
    }
    rows = rows_of(offsets, seq, tokens);
    return row >= rows.first && row - rows.first < (int64_t)rows.n;
}

// The row of token `pos` of a slot among the rows of head `head` of all pages,
// or -1 where it does not exist (a bad slot, position or page).
__device__ __forceinline__ int64_t page_row(const PagedTable &pt, int64_t slot, int64_t pos, uint32_t head, uint32_t kv_heads) {
    if (slot < 0 || slot >= (int64_t)pt.slots || pos < 0 || pos >= (int64_t)pt.max_pages * pt.page_tokens) return -1;
    const uint32_t nth = (uint32_t)pos / pt.page_tokens, off = (uint32_t)pos - nth * pt.page_tokens;
    const int64_t page = pt.table[slot * pt.max_pages + nth];
    if (page < 0 || page >= (int64_t)pt.pages) return -1;
    return (page * kv_heads + head) * pt.page_tokens + off;
}

}  // namespace mf
