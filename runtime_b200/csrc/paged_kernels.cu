// Paged key/value cache: rows into pages, copies of pages (attention over
// pages: paged_attention.cu).
//
// A cache is two arrays of pages, K and V, each [pages][kv_heads]
// [page_tokens][head_dim] in F32, F16 or BF16, and a table [slots][max_pages]
// of page ids: token p of slot s lies in row p % page_tokens of page
// table[s][p / page_tokens].  The rows of one KV head in a page are
// contiguous, so a head's keys are read in runs of page_tokens * head_dim.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "mf_common.cuh"
#include "packed_kernels.h"

namespace mf {

namespace {

// One value in the page's type, rounded to nearest even.
__device__ __forceinline__ void page_round(float &o, float v) { o = v; }
__device__ __forceinline__ void page_round(__half &o, float v) { o = __float2half_rn(v); }
__device__ __forceinline__ void page_round(__nv_bfloat16 &o, float v) { o = __float2bfloat16_rn(v); }

// ---------------------------------------------------------------------
// Rows into pages
// ---------------------------------------------------------------------

// One thread per 8 values of a K row and the same 8 of the V row (head_dim is
// a multiple of 8, so both sides move in 16- or 32-byte pieces).  The row's
// sequence is found by bisection in the row offsets.
template <typename T>
__global__ void __launch_bounds__(256) paged_append_kernel(T *key_pages, T *value_pages, PagedTable pt, const float *k,
                                                           const float *v, uint64_t tokens, const int32_t *starts,
                                                           const int32_t *offsets, uint32_t kv_heads,
                                                           uint32_t head_dim) {
    pdl_wait();
    pdl_trigger();
    const uint32_t per_row = kv_heads * (head_dim / 8);
    const uint64_t total = tokens * per_row;
    for (uint64_t e = blockIdx.x * (uint64_t)blockDim.x + threadIdx.x; e < total;
         e += (uint64_t)gridDim.x * blockDim.x) {
        const uint64_t row = e / per_row;
        const uint32_t piece = (uint32_t)(e - row * per_row), head = piece / (head_dim / 8),
                       d = (piece - head * (head_dim / 8)) * 8;
        uint32_t seq;
        int64_t pos;
        if (offsets) {
            // The last sequence whose first row is at or before this one.
            uint32_t lo = 0, hi = pt.sequences;
            while (hi - lo > 1) {
                const uint32_t mid = lo + (hi - lo) / 2;
                if ((int64_t)offsets[mid] <= (int64_t)row) lo = mid; else hi = mid;
            }
            seq = lo;
            if ((int64_t)row < offsets[seq] || (int64_t)row >= offsets[seq + 1]) continue;
            pos = (int64_t)row - offsets[seq];
        } else {
            if (row >= pt.sequences) continue;
            seq = (uint32_t)row;
            pos = 0;
        }
        if (starts[seq] < 0) continue;
        pos += starts[seq];
        if (pos >= (int64_t)pt.max_pages * pt.page_tokens) continue;
        const int64_t slot = pt.slot_ids ? pt.slot_ids[seq] : (int64_t)seq;
        if (slot < 0 || slot >= (int64_t)pt.slots) continue;
        const int64_t page = pt.table[slot * pt.max_pages + pos / pt.page_tokens];
        if (page < 0 || page >= (int64_t)pt.pages) continue;
        const uint64_t at = (((uint64_t)page * kv_heads + head) * pt.page_tokens + pos % pt.page_tokens) * head_dim + d;
        const float *src[2] = {k + row * kv_heads * head_dim + piece * 8, v + row * kv_heads * head_dim + piece * 8};
        T *dst[2] = {key_pages + at, value_pages + at};
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const float4 a = reinterpret_cast<const float4 *>(src[w])[0], b = reinterpret_cast<const float4 *>(src[w])[1];
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

__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ PageCopies c, uint64_t page_vecs,
                                                         uint32_t pools) {
    pdl_wait();
    pdl_trigger();
    const uint32_t pair = blockIdx.x / pools, pool = blockIdx.x % pools;
    const uint4 *src = reinterpret_cast<const uint4 *>(c.pools[pool]) + c.pairs[pair].x * page_vecs;
    uint4 *dst = reinterpret_cast<uint4 *>(c.pools[pool]) + c.pairs[pair].y * page_vecs;
    for (uint64_t i = threadIdx.x; i < page_vecs; i += blockDim.x) dst[i] = src[i];
}

}  // namespace

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
    for (uint32_t p0 = 0; p0 < n_pools; p0 += kCopyPools) {
        PageCopies c;
        const uint32_t np = std::min<uint32_t>(n_pools - p0, kCopyPools);
        for (uint32_t p = 0; p < np; ++p) c.pools[p] = pools[p0 + p];
        for (uint64_t i0 = 0; i0 < n; i0 += kCopyPairs) {
            const uint64_t m = std::min<uint64_t>(n - i0, kCopyPairs);
            for (uint64_t i = 0; i < m; ++i) c.pairs[i] = make_uint2(sources[i0 + i], destinations[i0 + i]);
            if (int32_t st = launch(copy_pages_kernel, dim3((unsigned)(m * np)), dim3(256), 0, stream,
                                    "copy_pages_kernel", c, page_bytes / 16, np))
                return st;
        }
    }
    return MF_OK;
}

}  // namespace mf
