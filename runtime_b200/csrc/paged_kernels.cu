// Paged key/value cache: rows into pages, copies of pages, entries of the
// table (attention over pages: paged_attention.cu).
//
// A cache is two arrays of pages, K and V, each [pages][kv_heads]
// [page_tokens][head_dim] in F32, F16 or BF16, and a table [slots][max_pages]
// of page ids: token p of slot s lies in row p % page_tokens of page
// table[s][p / page_tokens].  The rows of one KV head in a page are
// contiguous, so a head's keys are read in runs of page_tokens * head_dim.
#include <cuda_runtime.h>

#include <algorithm>

#include "mf_common.cuh"
#include "packed_kernels.h"
#include "paged_common.cuh"

namespace mf {

namespace {

// ---------------------------------------------------------------------
// Rows into pages
// ---------------------------------------------------------------------

// One thread per 8 values of a K row and the same 8 of the V row (head_dim is
// a multiple of 8, so both sides move in 16- or 32-byte pieces).  A warp finds
// the sequence of its first row, 32 offsets a step (a bisection's dependent
// reads cost 512 sequences 3 us); lanes in later rows walk on from there.  512
// rows of 512 values: 5 us, the latency of four dependent reads; 9386 rows F32:
// 16 us, 4.7 TB/s (16-bit pages 11.5, 5.0), bound by how many reads the threads resident have under way
// (32 registers: 48 cost 1.5 us).
template <typename T>
__global__ void __launch_bounds__(256, 6) paged_append_kernel(T *key_pages, T *value_pages, PagedTable pt, const float *k,
                                                           const float *v, uint64_t tokens, const int32_t *starts,
                                                           const int32_t *offsets, uint32_t kv_heads,
                                                           uint32_t head_dim) {
    pdl_wait();
    pdl_trigger();
    const uint32_t per_row = kv_heads * (head_dim / 8);
    const uint64_t total = tokens * per_row;
    const uint64_t whole = (total + 31) / 32 * 32;  // whole warps
    for (uint64_t e = blockIdx.x * (uint64_t)blockDim.x + threadIdx.x; e < whole;
         e += (uint64_t)gridDim.x * blockDim.x) {
        const uint64_t own = min(e, total - 1), row = own <= UINT32_MAX ? (uint32_t)own / per_row : own / per_row;
        const uint32_t piece = (uint32_t)(own - row * per_row), head = piece / (head_dim / 8),
                       d = (piece - head * (head_dim / 8)) * 8;
        uint32_t seq;
        int64_t pos;
        if (offsets) {
            seq = last_offset_before(offsets, pt.sequences, (int64_t)__shfl_sync(0xffffffffu, row, 0));
            while (seq + 1 < pt.sequences && offsets[seq + 1] <= (int64_t)row) ++seq;
            if ((int64_t)row < offsets[seq] || (int64_t)row >= offsets[seq + 1]) continue;
            pos = (int64_t)row - offsets[seq];
        } else {
            if (row >= pt.sequences) continue;
            seq = (uint32_t)row;
            pos = 0;
        }
        if (e >= total) continue;
        if (starts[seq] < 0) continue;
        pos += starts[seq];
        if (pos >= (int64_t)pt.max_pages * pt.page_tokens) continue;
        const int64_t slot = pt.slot_ids ? pt.slot_ids[seq] : (int64_t)seq;
        if (slot < 0 || slot >= (int64_t)pt.slots) continue;
        const uint32_t nth = (uint32_t)pos / pt.page_tokens, off = (uint32_t)pos - nth * pt.page_tokens;
        const int64_t page = pt.table[slot * pt.max_pages + nth];
        if (page < 0 || page >= (int64_t)pt.pages) continue;
        const uint64_t at = (((uint64_t)page * kv_heads + head) * pt.page_tokens + off) * head_dim + d;
        const uint64_t from = row * kv_heads * head_dim + piece * 8;
        const float *src[2] = {k + from, v + from};
        T *dst[2] = {key_pages + at, value_pages + at};
        float4 x[2][2];
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int i = 0; i < 2; ++i) x[w][i] = __ldcs(reinterpret_cast<const float4 *>(src[w]) + i);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const float4 a = x[w][0], b = x[w][1];
            alignas(16) T r[8];
            page_round(r[0], a.x), page_round(r[1], a.y), page_round(r[2], a.z), page_round(r[3], a.w);
            page_round(r[4], b.x), page_round(r[5], b.y), page_round(r[6], b.z), page_round(r[7], b.w);
#pragma unroll
            for (int i = 0; i < (int)sizeof(r) / 16; ++i)
                reinterpret_cast<uint4 *>(dst[w])[i] = reinterpret_cast<const uint4 *>(r)[i];
        }
    }
}

// ---------------------------------------------------------------------
// Copies of pages
// ---------------------------------------------------------------------

// The lists travel in the kernel's parameters (32764 bytes at most), so a call
// copies nothing to the device first and may return with the lists free.
template <uint32_t kPools, uint32_t kPairs>
struct PageCopies {
    void *pools[kPools];
    uint2 pairs[kPairs];  // source, destination
};

// One CTA per page and pool, eight loads ahead of their stores.  At 1900 pages
// of 16 KB in 12 pools it runs at the rate of a plain copy.
template <uint32_t kPools, uint32_t kPairs>
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ PageCopies<kPools, kPairs> c,
                                                         uint64_t page_vecs, uint32_t pools) {
    pdl_wait();
    pdl_trigger();
    constexpr int kAhead = 8;
    const uint32_t pair = blockIdx.x / pools, pool = blockIdx.x % pools;
    const uint4 *src = reinterpret_cast<const uint4 *>(c.pools[pool]) + c.pairs[pair].x * page_vecs;
    uint4 *dst = reinterpret_cast<uint4 *>(c.pools[pool]) + c.pairs[pair].y * page_vecs;
    for (uint64_t i0 = threadIdx.x; i0 < page_vecs; i0 += 256 * kAhead) {
        uint4 v[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (i0 + j * 256 < page_vecs) v[j] = src[i0 + j * 256];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (i0 + j * 256 < page_vecs) dst[i0 + j * 256] = v[j];
    }
}

template <uint32_t kPools, uint32_t kPairs>
int32_t copy_some(void *const *pools, uint32_t n_pools, uint64_t page_bytes, const uint32_t *sources,
                  const uint32_t *destinations, uint64_t n, cudaStream_t stream) {
    PageCopies<kPools, kPairs> c;
    std::copy(pools, pools + n_pools, c.pools);
    for (uint64_t i = 0; i < n; ++i) c.pairs[i] = make_uint2(sources[i], destinations[i]);
    return launch(copy_pages_kernel<kPools, kPairs>, dim3((unsigned)(n * n_pools)), dim3(256), 0, stream,
                  "copy_pages_kernel", c, page_bytes / 16, n_pools);
}

// ---------------------------------------------------------------------
// Entries of the table
// ---------------------------------------------------------------------

template <uint32_t kEntries>
struct TableChanges {
    uint2 changes[kEntries];  // entry, page id
};

template <uint32_t kEntries>
__global__ void __launch_bounds__(256) set_table_kernel(int32_t *table, const __grid_constant__ TableChanges<kEntries> c,
                                                        uint32_t n) {
    pdl_wait();
    pdl_trigger();
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) table[c.changes[i].x] = (int32_t)c.changes[i].y;
}

template <uint32_t kEntries>
int32_t set_some(int32_t *table, const uint32_t *entries, const uint32_t *ids, uint32_t n, cudaStream_t stream) {
    TableChanges<kEntries> c;
    for (uint32_t i = 0; i < n; ++i) c.changes[i] = make_uint2(entries[i], ids[i]);
    return launch(set_table_kernel<kEntries>, dim3((n + 255) / 256), dim3(256), 0, stream, "set_table_kernel", table, c, n);
}

}  // namespace

int32_t paged_set_table(int32_t *table, const uint32_t *entries, const uint32_t *ids, uint64_t n, cudaStream_t stream) {
    constexpr uint32_t kEntries = 4000;
    for (uint64_t i = 0; i < n; i += kEntries) {
        const uint32_t m = (uint32_t)std::min<uint64_t>(n - i, kEntries);
        // Few entries: fewer bytes of parameters, as for copies.
        const int32_t st = m <= 64 ? set_some<64>(table, entries + i, ids + i, m, stream)
                                   : set_some<kEntries>(table, entries + i, ids + i, m, stream);
        if (st) return st;
    }
    return MF_OK;
}

int32_t paged_append(void *key_pages, void *value_pages, int32_t dtype, const PagedTable &pt, const float *k,
                     const float *v, uint64_t tokens, const int32_t *starts, const int32_t *offsets, uint32_t kv_heads,
                     uint32_t head_dim, cudaStream_t stream) {
    if (!tokens || !pt.sequences) return MF_OK;
    const uint64_t pieces = tokens * kv_heads * (head_dim / 8);
    const dim3 grid((unsigned)std::min<uint64_t>((pieces + 255) / 256, (uint64_t)sm_count() * 32)), block(256);
    if (dtype == MF_PAGE_F32)
        return launch(paged_append_kernel<float>, grid, block, 0, stream, "paged_append_kernel", (float *)key_pages,
                      (float *)value_pages, pt, k, v, tokens, starts, offsets, kv_heads, head_dim);
    if (dtype == MF_PAGE_F16)
        return launch(paged_append_kernel<__half>, grid, block, 0, stream, "paged_append_kernel", (__half *)key_pages,
                      (__half *)value_pages, pt, k, v, tokens, starts, offsets, kv_heads, head_dim);
    return launch(paged_append_kernel<__nv_bfloat16>, grid, block, 0, stream, "paged_append_kernel",
                  (__nv_bfloat16 *)key_pages, (__nv_bfloat16 *)value_pages, pt, k, v, tokens, starts, offsets, kv_heads,
                  head_dim);
}

int32_t copy_pages(void *const *pools, uint32_t n_pools, uint64_t page_bytes, const uint32_t *sources,
                   const uint32_t *destinations, uint64_t n, cudaStream_t stream) {
    constexpr uint32_t kPools = 64, kPairs = 4000;
    for (uint32_t p = 0; p < n_pools; p += kPools)
        for (uint64_t i = 0; i < n; i += kPairs) {
            const uint32_t np = std::min(n_pools - p, kPools);
            const uint64_t m = std::min<uint64_t>(n - i, kPairs);
            // Few pages: fewer bytes of parameters (12 pages: 9 us a call with the large list, 6 with the small).
            const int32_t st =
                np <= 16 && m <= 48
                    ? copy_some<16, 48>(pools + p, np, page_bytes, sources + i, destinations + i, m, stream)
                    : copy_some<kPools, kPairs>(pools + p, np, page_bytes, sources + i, destinations + i, m, stream);
            if (st) return st;
        }
    return MF_OK;
}

}  // namespace mf
