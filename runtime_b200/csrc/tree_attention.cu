// Attention of several rows per sequence over a paged cache: drafted trees,
// and prompts that go on in chunks (layout: paged_kernels.cu; trees:
// tree_kernels.cu).
//
// Row r of a sequence's n rows is its token L - n + r.  It sees the tokens
// before the rows, its ancestors and itself:
// out = sum_j p_j v_j / sum_j p_j, p_j = exp(q . k_j / sqrt(D) - m).
#include <cuda_runtime.h>

#include <algorithm>

#include "mf_common.cuh"
#include "packed_kernels.h"
#include "paged_common.cuh"

namespace mf {

namespace {

struct TreeGqaArgs {
    float *out;
    const float *q;
    const void *keys, *values;
    PagedTable pt;
    uint64_t tokens;
    const int32_t *lengths, *offsets, *parents;
    uint32_t q_heads, kv_heads, head_dim;
};

__device__ __forceinline__ float page_value(float v) { return v; }
__device__ __forceinline__ float page_value(__half v) { return __half2float(v); }
__device__ __forceinline__ float page_value(__nv_bfloat16 v) { return __bfloat162float(v); }

// A warp for each row and query head; 32 tokens a step, a lane to each for the
// scores and dimensions dealt to the lanes for the weighted sum.
template <typename T>
__global__ void __launch_bounds__(128) tree_gqa_simple_kernel(const TreeGqaArgs a) {
    __shared__ float s_q[4][128];
    pdl_wait();
    pdl_trigger();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint64_t item = (uint64_t)blockIdx.x * 4 + warp;
    if (item >= a.tokens * a.q_heads) return;
    const int64_t row = (int64_t)(item / a.q_heads);
    const uint32_t head = (uint32_t)(item % a.q_heads), kvh = head / (a.q_heads / a.kv_heads), D = a.head_dim;
    uint32_t seq = a.offsets ? last_offset_before(a.offsets, a.pt.sequences, row) : (uint32_t)row;
    if (a.offsets)
        while (seq + 1 < a.pt.sequences && a.offsets[seq + 1] <= row) ++seq;
    if (seq >= a.pt.sequences) return;
    const int64_t first = a.offsets ? a.offsets[seq] : row, end = a.offsets ? a.offsets[seq + 1] : row + 1;
    if (first < 0 || row < first || row >= end) return;
    const int64_t n = min(end, (int64_t)a.tokens) - first, start = (int64_t)a.lengths[seq] - n;
    const int64_t slot = a.pt.slot_ids ? a.pt.slot_ids[seq] : (int64_t)seq;
    const float *q = a.q + item * D;
    for (uint32_t d = lane; d < D; d += 32) s_q[warp][d] = q[d] * rsqrtf((float)D);
    __syncwarp();
    float m = -INFINITY, l = 0.0f, o[4] = {}, far_l = 0.0f, far[4] = {};  // (far: what is summed less often)
    const T *keys = static_cast<const T *>(a.keys), *values = static_cast<const T *>(a.values);
    for (int64_t p0 = 0; p0 <= start + (row - first); p0 += 32) {
        const int64_t pos = p0 + lane;
        bool seen = pos <= start + (row - first);
        if (seen && pos >= start && a.parents) {
            int64_t at = row - first;
            while (at > pos - start) {
                const int64_t up = a.parents[first + at];
                at = up < at ? up : -1;
            }
            seen = at == pos - start;
        }
        const int64_t at = seen ? page_row(a.pt, slot, pos, kvh, a.kv_heads) : -1;
        float s = -INFINITY;
        if (at >= 0) {
            float c[8] = {};  // sums of eight kinds: fewer roundings one after another
            for (uint32_t d = 0; d < D; d += 8)
                for (int i = 0; i < 8; ++i) c[i] = fmaf(s_q[warp][d + i], page_value(keys[at * D + d + i]), c[i]);
            s = ((c[0] + c[1]) + (c[2] + c[3])) + ((c[4] + c[5]) + (c[6] + c[7]));
        }
        const float now = fmaxf(m, warp_max(s));
        const float base = now == -INFINITY ? 0.0f : now, keep = expf(m - base), p = at >= 0 ? expf(s - base) : 0.0f;
        m = now;
        l = l * keep + warp_sum(p), far_l *= keep;
        float c[4] = {};
        for (int j = 0; j < 32; ++j) {
            const int64_t from = __shfl_sync(0xffffffffu, at, j);
            const float w = __shfl_sync(0xffffffffu, p, j);
            if (from < 0) continue;
            for (int i = 0; i < 4; ++i)
                if (lane + 32 * i < D) c[i] = fmaf(w, page_value(values[from * D + lane + 32 * i]), c[i]);
        }
        const bool add = p0 % 2048 == 0;
        if (add) far_l += l, l = 0.0f;
        for (int i = 0; i < 4; ++i) {
            o[i] = fmaf(o[i], keep, c[i]), far[i] *= keep;
            if (add) far[i] += o[i], o[i] = 0.0f;
        }
    }
    l += far_l;
    for (int i = 0; i < 4; ++i) o[i] += far[i];
    for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < D) a.out[item * D + lane + 32 * i] = l == 0.0f ? 0.0f : o[i] / l;
}

}  // namespace

int32_t paged_tree_gqa(float *out, const float *q, const void *key_pages, const void *value_pages, int32_t dtype,
                       const PagedTable &pt, uint64_t tokens, const int32_t *lengths, const int32_t *offsets,
                       const int32_t *parents, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, void *,
                       cudaStream_t stream) {
    if (!pt.sequences || !tokens) return MF_OK;
    TreeGqaArgs a;
    a.out = out, a.q = q, a.keys = key_pages, a.values = value_pages, a.pt = pt, a.tokens = tokens;
    a.lengths = lengths, a.offsets = offsets, a.parents = parents;
    a.q_heads = q_heads, a.kv_heads = kv_heads, a.head_dim = head_dim;
    const dim3 grid((unsigned)((tokens * q_heads + 3) / 4)), block(128);
    return launch(dtype == MF_PAGE_F32   ? tree_gqa_simple_kernel<float>
                  : dtype == MF_PAGE_F16 ? tree_gqa_simple_kernel<__half>
                                         : tree_gqa_simple_kernel<__nv_bfloat16>,
                  grid, block, 0, stream, "tree_gqa_simple_kernel", a);
}

}  // namespace mf
