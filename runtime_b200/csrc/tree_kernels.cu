// Drafted trees over paged caches: rotated appends, the short convolution along
// a tree's branches, acceptance (attention of a tree: tree_attention.cu).
//
// A draft gives every sequence some rows, its tokens to be verified.  Row 0 is
// the last token that is certain, and a row's parent is an earlier row of the
// same sequence; a row whose parent is not one (-1, as a rule) continues the
// sequence's past, and without parents every row continues the row before it.
#include <cuda_runtime.h>

#include <algorithm>

#include "mf_common.cuh"
#include "packed_kernels.h"
#include "paged_common.cuh"

namespace mf {

namespace {

// ---------------------------------------------------------------------
// Rotated rows into pages
// ---------------------------------------------------------------------

constexpr int kRopeRows = 4;   // of a CTA at most
constexpr int kRopeAhead = 2;  // heads of a thread whose loads are under way at once

struct RopeArgs {
    void *key_pages, *value_pages;
    PagedTable pt;
    float *q_out;
    const float *q, *k, *v, *q_weight, *k_weight;
    const int32_t *positions, *starts, *offsets;
    uint64_t tokens;
    uint32_t q_heads, kv_heads, head_dim, rows;
    float epsilon, theta;
};

// x' = x / sqrt(mean x^2 + epsilon) * weight (heads of q and k), then each pair
// (x'[c], x'[c + D/2]) turned by the row's position times theta^(-2c/D),
// frequency and angle rounded to F32 as everywhere in this library.
//
// A thread holds four pairs of a head (two 16-byte loads), so pairs never cross
// threads, and the sum of squares adds in the order of head_norm_rope where
// head_dim is 64: a cache may be written by either, bit for bit.  Sines and
// cosines (in 64 bits, as there) are made once for a row and shared by its heads.
//
// Bound by the reads and writes of q, k and v where rows are many, else by the
// chain offsets - table - row.  7,931 rows of 32/8 heads of 64 into F32 pages
// (195 MB) take 41.0 us a call among others, 4.8 TB/s, and 45.1 alone after L2 was
// flushed, with four rows a CTA; with eight 45.3 and 49.2, whose CTAs come in 1.3
// waves, and with two 47.0 and 51.2, whose angles take longer than their rows.  Two
// heads' loads are under way at once: with one 43.4, with three 42.6.  Few rows are
// split by heads until two CTAs per SM have some: 8 rows 3.6 us a call in a graph.
template <typename T>
__global__ void __launch_bounds__(256) append_rope_kernel(const RopeArgs a) {
    __shared__ float2 s_turn[kRopeRows * 64];  // (cosine, sine)
    __shared__ float s_frequency[64];
    __shared__ int64_t s_at[kRopeRows];  // the row in the pages; -1: none, -2: of no sequence
    __shared__ float s_position[kRopeRows];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, half = a.head_dim / 2;
    for (uint32_t c = tid; c < half; c += 256)
        s_frequency[c] = (float)pow((double)a.theta, -2.0 * (double)c / (double)a.head_dim);
    pdl_wait();
    pdl_trigger();
    const uint64_t row0 = (uint64_t)blockIdx.x * a.rows;
    const uint32_t rows = (uint32_t)min((uint64_t)a.rows, a.tokens - row0);
    for (uint32_t r = warp; r < rows; r += 8) {
        const int64_t row = (int64_t)(row0 + r);
        int64_t at = -2, pos = 0;
        uint32_t s;
        SequenceRows own;
        if (sequence_of(a.offsets, a.pt.sequences, a.tokens, row, s, own)) {
            const int64_t start = a.starts[s];
            pos = start + (row - own.first);
            at = start < 0 ? -1 : page_row(a.pt, a.pt.slot_ids ? a.pt.slot_ids[s] : (int64_t)s, pos, 0, a.kv_heads);
            if (a.positions) pos = a.positions[row];
        }
        if ((tid & 31) == 0) s_at[r] = at, s_position[r] = (float)pos;
    }
    __syncthreads();
    for (uint32_t e = tid; e < rows * half; e += 256) {
        const float angle = __fmul_rn(s_position[e / half], s_frequency[e % half]);
        double sine, cosine;
        sincos((double)angle, &sine, &cosine);
        s_turn[e] = make_float2((float)cosine, (float)sine);
    }
    __syncthreads();

    uint32_t lanes = 1;  // of a head
    while (lanes < half / 4) lanes *= 2;
    const uint32_t t = tid & (lanes - 1), groups = 256 / lanes, heads = a.q_heads + 2 * a.kv_heads, c = 4 * t;
    const uint32_t total = rows * heads, step = groups * gridDim.y;
    const bool active = c < half;
    struct Head {
        float4 x, y;
        uint32_t row, head;  // row of the CTA
        bool use;
    };
    auto load = [&](uint32_t e0) {
        Head it;
        const uint32_t e = min(e0 + tid / lanes, total - 1);
        it.row = e / heads, it.head = e - it.row * heads;
        it.use = active && e0 + tid / lanes < total && s_at[it.row] != -2;
        it.x = it.y = make_float4(0, 0, 0, 0);
        if (it.use) {
            const uint64_t row = row0 + it.row;
            const float *src = it.head < a.q_heads ? a.q + (row * a.q_heads + it.head) * a.head_dim
                               : it.head < a.q_heads + a.kv_heads
                                   ? a.k + (row * a.kv_heads + it.head - a.q_heads) * a.head_dim
                                   : a.v + (row * a.kv_heads + it.head - a.q_heads - a.kv_heads) * a.head_dim;
            it.x = __ldcs(reinterpret_cast<const float4 *>(src + c));
            it.y = __ldcs(reinterpret_cast<const float4 *>(src + half + c));
        }
        return it;
    };
    auto finish = [&](const Head &it) {
        float4 x = it.x, y = it.y;
        const uint32_t r = it.row, h = it.head;
        const int64_t at = s_at[r];
        const bool is_q = h < a.q_heads, is_k = !is_q && h < a.q_heads + a.kv_heads;
        const uint32_t kvh = is_q ? 0 : h - a.q_heads - (is_k ? 0 : a.kv_heads);
        const float *weight = is_q ? a.q_weight : is_k ? a.k_weight : nullptr;
        // (The lanes of a warp may hold heads of all kinds: all take part in the sum.)
        float4 ss = make_float4(fmaf(y.x, y.x, x.x * x.x), fmaf(y.y, y.y, x.y * x.y), fmaf(y.z, y.z, x.z * x.z),
                                fmaf(y.w, y.w, x.w * x.w));
        for (uint32_t o = lanes / 2; o > 0; o /= 2) {
            ss.x += __shfl_xor_sync(0xffffffffu, ss.x, o), ss.y += __shfl_xor_sync(0xffffffffu, ss.y, o);
            ss.z += __shfl_xor_sync(0xffffffffu, ss.z, o), ss.w += __shfl_xor_sync(0xffffffffu, ss.w, o);
        }
        if (!it.use) return;
        if (weight) {
            const float sum = (ss.x + ss.z) + (ss.y + ss.w);
            const float rec = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sum, (float)a.head_dim), a.epsilon)));
            const float4 w = *reinterpret_cast<const float4 *>(weight + c), z = *reinterpret_cast<const float4 *>(weight + half + c);
            x.x = __fmul_rn(__fmul_rn(x.x, rec), w.x), x.y = __fmul_rn(__fmul_rn(x.y, rec), w.y);
            x.z = __fmul_rn(__fmul_rn(x.z, rec), w.z), x.w = __fmul_rn(__fmul_rn(x.w, rec), w.w);
            y.x = __fmul_rn(__fmul_rn(y.x, rec), z.x), y.y = __fmul_rn(__fmul_rn(y.y, rec), z.y);
            y.z = __fmul_rn(__fmul_rn(y.z, rec), z.z), y.w = __fmul_rn(__fmul_rn(y.w, rec), z.w);
        }
        if (is_q || is_k) {
            const float2 *turn = s_turn + r * half + c;
            auto rotate = [](float &u, float &v, float2 cs) {
                const float first = u, second = v;
                u = __fsub_rn(__fmul_rn(first, cs.x), __fmul_rn(second, cs.y));
                v = __fadd_rn(__fmul_rn(second, cs.x), __fmul_rn(first, cs.y));
            };
            rotate(x.x, y.x, turn[0]), rotate(x.y, y.y, turn[1]), rotate(x.z, y.z, turn[2]), rotate(x.w, y.w, turn[3]);
        }
        if (is_q) {
            float *dst = a.q_out + ((row0 + r) * a.q_heads + h) * a.head_dim;
            *reinterpret_cast<float4 *>(dst + c) = x;
            *reinterpret_cast<float4 *>(dst + half + c) = y;
        } else if (at >= 0) {
            T *dst = static_cast<T *>(is_k ? a.key_pages : a.value_pages) +
                     (uint64_t)(at + (int64_t)kvh * a.pt.page_tokens) * a.head_dim;
            struct alignas(4 * sizeof(T)) Four {
                T v[4];
            } u, w;
            page_round(u.v[0], x.x), page_round(u.v[1], x.y), page_round(u.v[2], x.z), page_round(u.v[3], x.w);
            page_round(w.v[0], y.x), page_round(w.v[1], y.y), page_round(w.v[2], y.z), page_round(w.v[3], y.w);
            *reinterpret_cast<Four *>(dst + c) = u;
            *reinterpret_cast<Four *>(dst + half + c) = w;
        }
    };
    for (uint32_t e0 = blockIdx.y * groups; e0 < total; e0 += kRopeAhead * step) {
        Head it[kRopeAhead];
#pragma unroll
        for (int i = 0; i < kRopeAhead; ++i) it[i] = load(e0 + i * step);
#pragma unroll
        for (int i = 0; i < kRopeAhead; ++i) finish(it[i]);
    }
}

// ---------------------------------------------------------------------
// Short convolution along branches
// ---------------------------------------------------------------------

constexpr int kConvRows = 8;       // rows of a CTA at most
constexpr int kConvMaxWidth = 16;  // taps
constexpr int kConvThreads = 128;

struct TreeConvArgs {
    float *out;
    const float *projection, *kernel, *history;
    const int32_t *offsets, *parents, *slot_ids;
    uint64_t tokens;
    uint32_t slots, sequences, hidden, width, rows;
};

// out[r] = C[r] * sum_j kernel[j] * u[a_j], u = B * V, a_{width-1} = r and each
// a_j the parent of a_{j+1}; past the first row, the sequence's history.  Taps
// add in order, each product and sum rounded, as in the convolution of single
// sequences: on a chain the results are the same bits.
//
// Bound by the projections (each row's three parts once): a thread has all loads
// of a row (seven at width 3) under way at once, a CTA takes up to eight rows,
// whose ancestors are near ones and mostly found in L1 or L2.  1,792 rows of
// 2,048 channels (59 MB): 16 us from cold memory, 3.7 TB/s.
template <int V, int W>
__global__ void __launch_bounds__(kConvThreads) tree_conv_kernel(const TreeConvArgs a) {
    // Of every row and tap: the row whose u it takes, or -1 - the history's entry
    // (of all slots), or kNothing.
    constexpr int64_t kNothing = INT64_MIN;
    __shared__ int64_t s_tap[kConvRows][kConvMaxWidth];
    __shared__ bool s_in[kConvRows];
    pdl_wait();
    pdl_trigger();
    const uint32_t hist = (W ? W : a.width) - 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint64_t row0 = (uint64_t)blockIdx.x * a.rows;
    const uint32_t rows = (uint32_t)min((uint64_t)a.rows, a.tokens - row0);
    for (uint32_t r = warp; r < rows; r += kConvThreads / 32) {
        const int64_t row = (int64_t)(row0 + r);
        uint32_t seq;
        SequenceRows own;
        const bool in = sequence_of(a.offsets, a.sequences, a.tokens, row, seq, own);
        if (lane) continue;
        s_in[r] = in;
        if (!in) continue;
        const int64_t slot = a.slot_ids ? a.slot_ids[seq] : (int64_t)seq, first = own.first;
        int64_t at = row - first;
        for (int j = (int)hist; j >= 0; --j) {
            s_tap[r][j] = at >= 0                                  ? first + at
                          : slot >= 0 && slot < (int64_t)a.slots ? -1 - (slot * hist + hist + at)
                                                                   : kNothing;
            if (at <= 0) {
                --at;
                continue;
            }
            const int64_t up = a.parents ? (int64_t)a.parents[first + at] : at - 1;
            at = up >= 0 && up < at ? up : -1;
        }
    }
    __syncthreads();
    const uint32_t c = (blockIdx.y * kConvThreads + threadIdx.x) * V;
    if (c >= a.hidden) return;
    const uint64_t pitch = 3ull * a.hidden;
    struct alignas(4 * V) Vec {
        float v[V];
    };
    auto load = [](const float *p) { return *reinterpret_cast<const Vec *>(p); };
    float weight[W ? W : 1][V];
    if constexpr (W > 0) {
#pragma unroll
        for (int j = 0; j < W; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) weight[j][i] = a.kernel[(uint64_t)(c + i) * W + j];
    }
    for (uint32_t r = 0; r < rows; ++r) {
        if (!s_in[r]) continue;
        const Vec gate = load(a.projection + (row0 + r) * pitch + a.hidden + c);
        Vec total = {};
        if constexpr (W > 0) {
            Vec b[W], v[W];
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const int64_t at = s_tap[r][j];
                b[j] = v[j] = Vec{};
                if (at >= 0) {
                    b[j] = load(a.projection + at * pitch + c), v[j] = load(a.projection + at * pitch + 2ull * a.hidden + c);
                } else if (at != kNothing) {
                    b[j] = load(a.history + (uint64_t)(-1 - at) * a.hidden + c);
#pragma unroll
                    for (int i = 0; i < V; ++i) v[j].v[i] = 1.0f;
                }
            }
#pragma unroll
            for (int j = 0; j < W; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i)
                    total.v[i] = __fadd_rn(total.v[i], __fmul_rn(weight[j][i], __fmul_rn(b[j].v[i], v[j].v[i])));
        } else {
            for (uint32_t j = 0; j <= hist; ++j) {
                const int64_t at = s_tap[r][j];
                Vec u = {};
                if (at >= 0) {
                    const Vec b = load(a.projection + at * pitch + c), v = load(a.projection + at * pitch + 2ull * a.hidden + c);
#pragma unroll
                    for (int i = 0; i < V; ++i) u.v[i] = __fmul_rn(b.v[i], v.v[i]);
                } else if (at != kNothing) {
                    u = load(a.history + (uint64_t)(-1 - at) * a.hidden + c);
                }
#pragma unroll
                for (int i = 0; i < V; ++i)
                    total.v[i] = __fadd_rn(total.v[i], __fmul_rn(a.kernel[(uint64_t)(c + i) * a.width + j], u.v[i]));
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) total.v[i] = __fmul_rn(total.v[i], gate.v[i]);
        *reinterpret_cast<Vec *>(a.out + (row0 + r) * a.hidden + c) = total;
    }
}

struct ConvKeepArgs {
    float *history_out;
    const float *history, *projection;
    const int32_t *paths, *counts, *offsets, *slot_ids;
    uint64_t tokens;
    uint32_t slots, sequences, hidden, width;
};

// The history after the accepted rows: the last width - 1 of its entries and
// theirs.  A thread owns a channel of a sequence and reads all before it writes.
// Bound by the chain counts - path - rows: 64 sequences of 2,048 channels 2.7 us a
// call in a graph, 6 from cold memory.
template <int W>
__global__ void __launch_bounds__(128) tree_conv_keep_kernel(const ConvKeepArgs a) {
    pdl_wait();
    pdl_trigger();
    const uint32_t c = blockIdx.x * 128 + threadIdx.x;
    if (c >= a.hidden) return;
    constexpr int kMost = W > 0 ? W - 1 : kConvMaxWidth - 1;
    const uint32_t hist = W > 0 ? W - 1 : a.width - 1;
    for (uint32_t seq = blockIdx.y; seq < a.sequences; seq += gridDim.y) {
        const int64_t slot = a.slot_ids ? a.slot_ids[seq] : (int64_t)seq;
        if (slot < 0 || slot >= (int64_t)a.slots) continue;
        const SequenceRows own = rows_of(a.offsets, seq, a.tokens);
        const int64_t first = own.first;
        const uint32_t n = own.n;
        const uint32_t count = (uint32_t)min((int64_t)n, max((int64_t)0, (int64_t)a.counts[seq]));
        const uint64_t base = (uint64_t)slot * hist * a.hidden + c;
        float entry[kMost > 0 ? kMost : 1];
#pragma unroll
        for (int j = 0; j < kMost; ++j) {
            if (j >= (int)hist) break;
            const int64_t at = (int64_t)count - hist + j;  // of the accepted rows
            if (at < 0) {
                entry[j] = a.history[base + (uint64_t)(j + count) * a.hidden];
            } else {
                const int64_t place = a.paths[first + at];
                const float *p = a.projection + (uint64_t)(first + place) * 3 * a.hidden + c;
                entry[j] = place >= 0 && place < (int64_t)n ? __fmul_rn(p[0], p[2ull * a.hidden]) : 0.0f;
            }
        }
#pragma unroll
        for (int j = 0; j < kMost; ++j)
            if (j < (int)hist) a.history_out[base + (uint64_t)j * a.hidden] = entry[j];
    }
}

// ---------------------------------------------------------------------
// Acceptance
// ---------------------------------------------------------------------

constexpr uint32_t kAcceptPools = 64;
constexpr int kAcceptThreads = 256;

struct AcceptArgs {
    void *pools[kAcceptPools];
    PagedTable pt;
    const float *drafted, *sampled;
    const int32_t *starts, *offsets, *parents;
    int32_t *paths, *counts;  // null: another launch writes them
    float *next;
    uint64_t tokens;
    uint32_t n_pools, kv_heads, row_bytes;  // row_bytes: of one KV head
};

// A CTA owns a sequence (and, where there are few, some of the pools).  One warp
// walks from row 0: a row's next is its first child whose drafted id is the
// row's own draw, 32 rows a step; up to 128 rows are held in registers, so that
// a step costs a few shuffles (reading each from memory 512 sequences took 27
// us).  Up to 32 rows of the path are then moved: row path[j] to place j, a
// thread for each 16 bytes, four loads ahead of their stores, ascending, so that
// no place is written before it is read (j <= path[j] < path[j + 1]).  Bound by
// the walk, a step after the other: 512 sequences of 16 rows take 9.3 us a call in a
// graph with 12 pools of BF16 pages, 14 from cold memory, of which the moves (25 MB)
// would take 4 at DRAM's rate.  Past 128 rows a step reads memory: a chunk of 500 rows
// that are all accepted takes 102 us, of 2,500 502 (with parents 161 and 798).
__global__ void __launch_bounds__(kAcceptThreads) accept_kernel(const __grid_constant__ AcceptArgs a) {
    constexpr int kHeld = 4;  // rows of a lane
    __shared__ int64_t s_from[32], s_to[32];
    __shared__ uint32_t s_count, s_done;
    pdl_wait();
    pdl_trigger();
    const uint32_t seq = blockIdx.x, lane = threadIdx.x & 31;
    const SequenceRows own = rows_of(a.offsets, seq, a.tokens);
    const int64_t first = own.first;
    const uint32_t n = own.n;
    const bool tells = a.counts && blockIdx.y == 0, held = n <= 32 * kHeld;
    const int64_t slot = a.pt.slot_ids ? a.pt.slot_ids[seq] : (int64_t)seq;
    const int64_t start = a.starts ? a.starts[seq] : -1;
    const float *drafted = a.drafted + first, *sampled = a.sampled + first;
    const uint32_t vecs = a.row_bytes / 16, heads_vecs = vecs * a.kv_heads;
    float held_drafted[kHeld], held_sampled[kHeld];
    int32_t held_parent[kHeld];
    if (threadIdx.x < 32 && held)
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
            const uint32_t i = 32 * k + lane;
            held_drafted[k] = i < n ? drafted[i] : 0.0f, held_sampled[k] = i < n ? sampled[i] : 0.0f;
            held_parent[k] = i >= n ? -1 : a.parents ? a.parents[first + i] : (int32_t)i - 1;
        }
    // The first child of row `at`, from at + 1 on, whose id is drawn there; n: none.
    auto child = [&](uint32_t at) -> uint32_t {
        if (held) {
            float want = 0.0f;
#pragma unroll
            for (uint32_t k = 0; k < kHeld; ++k)
                if (at / 32 == k) want = __shfl_sync(0xffffffffu, held_sampled[k], at % 32);
#pragma unroll
            for (uint32_t k = 0; k < kHeld; ++k) {
                if (32 * k >= n) break;
                const uint32_t i = 32 * k + lane;
                const uint32_t hits = __ballot_sync(0xffffffffu, i > at && i < n && held_parent[k] == (int32_t)at && held_drafted[k] == want);
                if (hits) return 32 * k + __ffs(hits) - 1;
            }
            return n;
        }
        const float want = sampled[at];
        if (!a.parents) return at + 1 < n && drafted[at + 1] == want ? at + 1 : n;
        for (uint32_t i0 = at + 1; i0 < n; i0 += 32) {
            const uint32_t i = i0 + lane;
            const uint32_t hits = __ballot_sync(0xffffffffu, i < n && a.parents[first + i] == (int32_t)at && drafted[i] == want);
            if (hits) return i0 + __ffs(hits) - 1;
        }
        return n;
    };
    uint32_t path = 0, at = 0;  // rows on the path; the last of them
    for (bool more = n > 0; more;) {
        __syncthreads();  // (the lists below have been read)
        if (threadIdx.x < 32) {
            const uint32_t begin = path;
            uint32_t mine = 0;  // the row of place begin + lane
            bool ended = false;
            while (path - begin < 32) {
                const uint32_t next = path ? child(at) : 0;
                if (next == n) {
                    ended = true;
                    break;
                }
                at = next;
                if (lane == path - begin) mine = at;
                ++path;
            }
            const uint32_t place = begin + lane;
            if (place < path) {
                const bool moves = mine != place && start >= 0 && a.n_pools;
                s_from[lane] = moves ? page_row(a.pt, slot, start + mine, 0, a.kv_heads) : -1;
                s_to[lane] = moves ? page_row(a.pt, slot, start + place, 0, a.kv_heads) : -1;
                if (tells) a.paths[first + place] = (int32_t)mine;
            }
            if (lane == 0) s_count = path - begin, s_done = ended;
        }
        __syncthreads();
        const uint32_t count = s_count;
        more = !s_done;
        const uint32_t pools = (a.n_pools + gridDim.y - 1 - blockIdx.y) / gridDim.y;  // this CTA's: blockIdx.y and on
        for (uint32_t e = threadIdx.x; e < pools * heads_vecs; e += kAcceptThreads) {
            const uint32_t p = e / heads_vecs, in = e - p * heads_vecs, h = in / vecs;
            char *pool = static_cast<char *>(a.pools[blockIdx.y + p * gridDim.y]) + (uint64_t)(in - h * vecs) * 16;
            const int64_t shift = (int64_t)h * a.pt.page_tokens;
            for (uint32_t j0 = 0; j0 < count; j0 += 4) {
                uint4 x[4];
                bool moves[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    moves[k] = j0 + k < count && s_from[j0 + k] >= 0 && s_to[j0 + k] >= 0;
                    if (moves[k]) x[k] = *reinterpret_cast<const uint4 *>(pool + (s_from[j0 + k] + shift) * a.row_bytes);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (moves[k]) *reinterpret_cast<uint4 *>(pool + (s_to[j0 + k] + shift) * a.row_bytes) = x[k];
            }
        }
    }
    if (tells && threadIdx.x < 32) {
        for (uint32_t i = path + lane; i < n; i += 32) a.paths[first + i] = -1;
        if (lane == 0) {
            a.counts[seq] = (int32_t)path;
            a.next[seq] = n ? sampled[at] : __int_as_float(0x7fc00000);
        }
    }
}

}  // namespace

int32_t paged_append_rope(void *key_pages, void *value_pages, int32_t dtype, const PagedTable &pt, float *q_out,
                          const float *q, const float *k, const float *v, uint64_t tokens, const float *q_weight,
                          const float *k_weight, float epsilon, float theta, const int32_t *positions,
                          const int32_t *starts, const int32_t *offsets, uint32_t q_heads, uint32_t kv_heads,
                          uint32_t head_dim, cudaStream_t stream) {
    if (!tokens || !pt.sequences) return MF_OK;
    RopeArgs a;
    a.key_pages = key_pages, a.value_pages = value_pages, a.pt = pt, a.q_out = q_out, a.q = q, a.k = k, a.v = v;
    a.q_weight = q_weight, a.k_weight = k_weight, a.positions = positions, a.starts = starts, a.offsets = offsets;
    a.tokens = tokens, a.q_heads = q_heads, a.kv_heads = kv_heads, a.head_dim = head_dim;
    a.epsilon = epsilon, a.theta = theta;
    const uint64_t sms = sm_count();
    a.rows = (uint32_t)std::min<uint64_t>(kRopeRows, std::max<uint64_t>(1, tokens / (sms * 4)));
    const uint64_t ctas = (tokens + a.rows - 1) / a.rows;
    if (ctas > INT32_MAX) return fail(MF_OVERFLOW, "token rows exceed the launch grid");
    uint32_t lanes = 1;
    while (lanes < head_dim / 8) lanes *= 2;
    const uint32_t passes = (a.rows * (q_heads + 2 * kv_heads) + 256 / lanes - 1) / (256 / lanes);
    const uint32_t split = (uint32_t)std::min<uint64_t>(passes, std::max<uint64_t>(1, 2 * sms / ctas));
    const dim3 grid((unsigned)ctas, split), block(256);
    if (dtype == MF_PAGE_F32)
        return launch(append_rope_kernel<float>, grid, block, 0, stream, "append_rope_kernel", a);
    if (dtype == MF_PAGE_F16)
        return launch(append_rope_kernel<__half>, grid, block, 0, stream, "append_rope_kernel", a);
    return launch(append_rope_kernel<__nv_bfloat16>, grid, block, 0, stream, "append_rope_kernel", a);
}

int32_t tree_convolution(float *out, const float *projection, const float *kernel, const float *history, uint32_t slots,
                         uint64_t tokens, const int32_t *offsets, const int32_t *parents, const int32_t *slot_ids,
                         uint32_t sequences, uint32_t hidden, uint32_t width, cudaStream_t stream) {
    if (!tokens || !sequences || !hidden) return MF_OK;
    TreeConvArgs a;
    a.out = out, a.projection = projection, a.kernel = kernel, a.history = history, a.offsets = offsets;
    a.parents = parents, a.slot_ids = slot_ids, a.tokens = tokens, a.slots = slots, a.sequences = sequences;
    a.hidden = hidden, a.width = width;
    const int v = hidden % 4 == 0 ? 4 : 1;
    const uint32_t parts = (hidden + kConvThreads * v - 1) / (kConvThreads * v);
    if (parts > 65535) return fail(MF_OVERFLOW, "short convolution hidden width exceeds its limit");
    // Rows of a CTA: one where a wave holds all (8 rows of 1024 values and their keep
    // 10.2 us after L2 was flushed, for 16.4 with eight), eight where CTAs come in waves
    // (1792 of 2048 and their keep 14.4 us among others, for 20.0 with one).
    a.rows = (uint32_t)std::min<uint64_t>(kConvRows, std::max<uint64_t>(1, tokens * parts / ((uint64_t)sm_count() * 6)));
    const dim3 grid((unsigned)((tokens + a.rows - 1) / a.rows), parts), block(kConvThreads);
    return launch(v == 4   ? width == 3 ? tree_conv_kernel<4, 3> : tree_conv_kernel<4, 0>
                  : width == 3 ? tree_conv_kernel<1, 3> : tree_conv_kernel<1, 0>,
                  grid, block, 0, stream, "tree_conv_kernel", a);
}

int32_t tree_convolution_keep(float *history_out, const float *history, uint32_t slots, const float *projection,
                              uint64_t tokens, const int32_t *paths, const int32_t *counts, const int32_t *offsets,
                              const int32_t *slot_ids, uint32_t sequences, uint32_t hidden, uint32_t width,
                              cudaStream_t stream) {
    if (!sequences || !hidden || width < 2) return MF_OK;
    ConvKeepArgs a;
    a.history_out = history_out, a.history = history, a.projection = projection, a.paths = paths, a.counts = counts;
    a.offsets = offsets, a.slot_ids = slot_ids, a.tokens = tokens, a.slots = slots, a.sequences = sequences;
    a.hidden = hidden, a.width = width;
    const dim3 grid((hidden + 127) / 128, std::min(sequences, 65535u)), block(128);
    return launch(width == 3 ? tree_conv_keep_kernel<3> : tree_conv_keep_kernel<0>, grid, block, 0, stream,
                  "tree_conv_keep_kernel", a);
}

int32_t paged_accept(int32_t *paths, int32_t *counts, float *next, void *const *pools, uint32_t n_pools, int32_t dtype,
                     const PagedTable &pt, const float *drafted, const float *sampled, uint64_t tokens,
                     const int32_t *starts, const int32_t *offsets, const int32_t *parents, uint32_t kv_heads,
                     uint32_t head_dim, cudaStream_t stream) {
    if (!pt.sequences) return MF_OK;
    for (uint32_t p = 0; p == 0 || p < n_pools; p += kAcceptPools) {
        AcceptArgs a;
        a.n_pools = std::min(n_pools - p, kAcceptPools);
        std::copy(pools + p, pools + p + a.n_pools, a.pools);
        a.pt = pt, a.drafted = drafted, a.sampled = sampled, a.starts = starts, a.offsets = offsets;
        a.parents = parents, a.paths = paths, a.counts = p ? nullptr : counts, a.next = next, a.tokens = tokens;
        a.kv_heads = kv_heads, a.row_bytes = head_dim * (dtype == MF_PAGE_F32 ? 4 : 2);
        const uint32_t split = std::max(1u, std::min(a.n_pools, 4 * (uint32_t)sm_count() / pt.sequences));
        if (int32_t st = launch(accept_kernel, dim3(pt.sequences, split), dim3(kAcceptThreads), 0, stream,
                                "accept_kernel", a))
            return st;
    }
    return MF_OK;
}

}  // namespace mf
