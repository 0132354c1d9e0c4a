// One-token attention over a paged key/value cache (layout: paged_kernels.cu).
//
// out = sum_j p_j v_j / sum_j p_j, p_j = exp(q . k_j / sqrt(D) - m), one pass
// over the tokens with the running maximum m and sum (held in F32).  Bound by
// the bytes of K and V, each read once: everything below keeps the loads
// going and the arithmetic out of their way.
//
// Split.  The work is a list of units of 128, 64 or 32 tokens, sequence by sequence
// and KV head by KV head, and the CTAs of one wave take equal runs of it,
// whatever the lengths are: the list is built on the device from `lengths`,
// so a captured call follows them.  A run that ends inside a sequence leaves
// its maximum, sum and weighted values in the workspace; the last CTA to
// arrive joins them in one order, so repeats are equal bit for bit.  (Two runs
// for each place in the wave even out the CTAs' ends but cost a join more: 32
// ragged sequences 42 us against 36, 512 sequences 122 against 113.)
//
// Loads.  A warp owns 32, 16 or 8 tokens of every unit and a ring of cp.async stages
// of its own (no block barrier in the loop); the page lookup of a token is
// done by one lane, a stage ahead, and handed over by shuffles.
//
// Arithmetic.  Eight query heads of a KV head are the rows of mma.sync tiles
// (tcgen05 wants 64 or 128 rows; at 8 the tensor pipe is not the bound, the
// loads are), tokens the columns, so the score tile's accumulator is, lane by
// lane, the operand of P V.  Every 8 heads take a pass over K and V of their own
// (96 sequences of 1000-5000, one KV head of 128, BF16: 8 heads 41 us, 16 65, 32
// 113).  F32 accuracy comes from splitting the F32 operand (q, then p) in parts of the page's type whose products are summed
// in F32: rows 0-7 hold the high parts and rows 8-15 the next ones, so two
// parts cost one MMA.  F16 pages: two parts of 11 bits (q scaled to [2^14,
// 2^15) by a power of two per head and p by 2^14, so that low parts stay
// above F16's smallest step).  BF16 pages: three parts of 8 bits (two would leave
// 2^-16 of each operand out).  F32 pages: TF32 parts of 11 bits of both
// operands, four products.  Against 64 bits the output is off by 2e-7 to 5e-7
// of its norm, less than a plain F32 form's 6e-7 to 1.1e-6.
//
// Measured (B200, calls back to back): 512 sequences of 513-640 tokens, 32/8
// heads of 64, BF16, 613 MB: 113 us, 5.4 TB/s, 0.83 of a plain copy's rate; 123
// us where each call follows other work.  In its steady part (94 us) it runs at
// that rate; the rest is the 4 us before the first rows arrive (lengths, table,
// rows: three dependent reads), CTAs that end apart, and the joins.  One sequence of 131071 tokens F16 52 us (5.2 TB/s).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "mf_common.cuh"
#include "packed_kernels.h"
#include "tc_sm100.cuh"

namespace mf {

namespace {

using sm100::smem_u32;

constexpr int kPgWarps = 4;
constexpr int kPgHeads = 8;                // query heads of one pass over a KV head

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ float4 lds4(uint32_t at) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

// d = a b + c; c is d or zero (the constant needs no registers).
#define MF_PG_MMA(name, shape, type)                                                                       \
    __device__ __forceinline__ void name(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, \
                                         uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3) { \
        asm("mma.sync.aligned." shape ".row.col.f32." type "." type ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, " \
            "{%10,%11,%12,%13};"                                                                           \
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])                                               \
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));   \
    }
MF_PG_MMA(mma_f16, "m16n8k16", "f16")
MF_PG_MMA(mma_bf16, "m16n8k16", "bf16")
MF_PG_MMA(mma_tf32, "m16n8k8", "tf32")
#undef MF_PG_MMA

// d (+)= the products of an F32 operand's parts (rows 0-7 high, rows 8-15 next,
// and for BF16 a third in a second MMA, summed first) with a page's values.
template <int kParts>
__device__ __forceinline__ void mma_parts(float (&d)[4], const uint32_t (&x0)[kParts], const uint32_t (&x1)[kParts],
                                          uint32_t b0, uint32_t b1, bool add) {
    const float c0 = add ? d[0] : 0.0f, c1 = add ? d[1] : 0.0f, c2 = add ? d[2] : 0.0f, c3 = add ? d[3] : 0.0f;
    if constexpr (kParts == 2) {
        mma_f16(d, x0[0], x0[1], x1[0], x1[1], b0, b1, c0, c1, c2, c3);
    } else {
        mma_bf16(d, x0[2], 0, x1[2], 0, b0, b1, c0, c1, c2, c3);
        mma_bf16(d, x0[0], x0[1], x1[0], x1[1], b0, b1, d[0], d[1], d[2], d[3]);
    }
}

// 2^x, 0 for -infinity (the hardware's exponential, 2 units in the last place).
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// x in parts: 11 bits rounded, and the rest (the MMA reads its first 11 bits).
// Two integer operations where the conversion instruction takes several.
__device__ __forceinline__ void split_tf32(float x, uint32_t &hi, uint32_t &lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}
// The parts of a pair, packed as an MMA operand register each (x in the low half).
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&part)[2], __half) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    part[0] = *reinterpret_cast<const uint32_t *>(&h);
    part[1] = *reinterpret_cast<const uint32_t *>(&l);
}
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&part)[3], __nv_bfloat16) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        part[i] = *reinterpret_cast<const uint32_t *>(&h);
        x -= __uint_as_float(part[i] << 16);
        y -= __uint_as_float(part[i] & 0xffff0000u);
    }
}

template <typename T>
struct PageType;
template <>
struct PageType<float> {
    static constexpr int kParts = 2;
    static constexpr float kShift = 0.0f;  // exponent added to every weight
};
template <>
struct PageType<__half> {
    static constexpr int kParts = 2;
    static constexpr float kShift = 14.0f;
};
template <>
struct PageType<__nv_bfloat16> {
    static constexpr int kParts = 3;
    static constexpr float kShift = 0.0f;
};

template <typename T, int D>
struct PagedShape {
    static constexpr bool kF32 = sizeof(T) == 4;
    static constexpr int kPitch = D * (int)sizeof(T);
    static constexpr int kChunks = kPitch / 16;  // 16-byte chunks of a row
    // Tokens of a warp's tile: 32 where a stage stays at 8 KB (fewer steps per
    // token), else 16, and 8 for F32 rows of 128, of which two CTAs then fit an
    // SM (233 sequences of 256 tokens, 4 heads: 57 us for 76; one of 32768 39 for 57).
    static constexpr int kTile = kPitch <= 128 ? 32 : kPitch <= 256 ? 16 : 8;
    // Stages of a warp's ring and CTAs per SM, by registers and shared memory.
    // 512 sequences of 513-640 BF16 tokens: 3 CTAs of 2 stages 113 us, 2 of 3
    // stages 132 us (a step's arithmetic hides behind the other warps' loads);
    // 32 ragged F32 sequences 37 and 41 us; 16-bit rows of 128 spill registers
    // with 3 (47 and 42 us).
    static constexpr bool kThree = kPitch <= 128 || (kF32 && kPitch <= 256);
    static constexpr int kStages = kThree ? 2 : 3;
    static constexpr int kCtas = kThree ? 3 : 2;
    static constexpr int kUnit = kTile * kPgWarps;
    static constexpr uint32_t kFull = 0xffffffffu >> (32 - kTile);
    static constexpr int kStageBytes = 2 * kTile * kPitch;  // K, then V
    static constexpr int kPart = kPgHeads * (D + 2);  // a run's partial: weighted values [8][D], maxima [8], sums [8]
    static constexpr size_t kSmem = (size_t)kPgWarps * kStages * kStageBytes;
    static_assert(kPart * 4 <= kStageBytes, "the warps are joined in the stage that they used last");
    // The swizzle of a row's chunks: ldmatrix reads 8 rows of a chunk, the F32
    // fragments 2 rows x 4 chunks (K) or 4 even or odd rows x 2 chunks (V).
    static __device__ __forceinline__ int k_chunk(int row, int c) { return kF32 ? c ^ ((row & 1) << 2) : c ^ (row & 7); }
    static __device__ __forceinline__ int v_chunk(int row, int c) { return kF32 ? c ^ (row & 6) : c ^ (row & 7); }
};

// Runs that end inside an item.
struct PagedWork {
    unsigned *arrived;  // [CTAs], zero between calls
    float *partial;     // [2 * CTAs][kPart]
};

struct PagedArgs {
    float *out;
    const float *q;
    const void *keys, *values;
    PagedTable pt;
    const int32_t *lengths;
    uint32_t q_heads, kv_heads, head_dim, passes;  // passes: groups of 8 query heads per KV head
    uint32_t page_magic, page_shift;  // pos / page_tokens = mulhi(pos, magic) >> shift for pos < 2^31; 0: one token a page
    uint32_t aligned;                 // pages of 16 tokens or a multiple, rows without padding
    PagedWork work;
};

// A sequence's tokens as far as the table reaches; none for a bad slot.
__device__ __forceinline__ int seq_length(const PagedArgs &a, uint32_t seq) {
    const int64_t slot = a.pt.slot_ids ? a.pt.slot_ids[seq] : (int64_t)seq;
    if (slot < 0 || slot >= (int64_t)a.pt.slots) return 0;
    return max(0, (int)min((int64_t)a.lengths[seq], (int64_t)a.pt.max_pages * a.pt.page_tokens));
}

// Units of a sequence.  (Unsigned: a length may be as large as 2^31 - 1.)
template <int kUnit>
__device__ __forceinline__ int units_of(int len) {
    return (int)(((uint32_t)len + kUnit - 1) / kUnit);
}

// A place in the list of units: item = (sequence, KV head, pass).  Each item
// has a place more than units, its first, in which nothing is done: beginning
// and ending an item (its queries, the join) costs about a unit's time, so
// runs of equally many places take equally long.
template <int kUnit>
struct PagedCursor {
    uint32_t seq, item;  // item: KV head * passes + pass
    int unit, units, len;
    int at;  // places from the run's first

    // Moves on by a unit, which is a place further, or two into the next item.
    __device__ __forceinline__ void next(const PagedArgs &a, uint32_t items) {
        ++at;
        if (++unit < units) return;
        ++at;
        unit = 0;
        if (++item < items) return;
        item = 0;
        do {
            if (++seq >= a.pt.sequences) {
                units = len = 0;
                return;
            }
            len = seq_length(a, seq);
            units = units_of<kUnit>(len);
        } while (!units);
    }
};
// Places of an item with this many units.
__device__ __forceinline__ int item_places(int units) { return units ? units + 1 : 0; }

// Joins the warps' partials (`pitch` floats apart): to the output (weighted
// mean, 0 where no weight is) or as the partial of a run.
template <int D>
__device__ __forceinline__ void join_warps(const float *join, uint32_t pitch, uint32_t heads, uint32_t head_dim, float *out,
                                           float *part) {
    for (uint32_t e = threadIdx.x; e < heads * D; e += kPgWarps * 32) {
        const uint32_t h = e / D, d = e % D;
        float most = -INFINITY, sum = 0.0f, acc = 0.0f;
#pragma unroll
        for (int w = 0; w < kPgWarps; ++w) most = fmaxf(most, join[w * pitch + kPgHeads * D + h]);
        const float base = most == -INFINITY ? 0.0f : most;
#pragma unroll
        for (int w = 0; w < kPgWarps; ++w) {
            const float f = exp2_fast(join[w * pitch + kPgHeads * D + h] - base);
            sum = fmaf(join[w * pitch + kPgHeads * (D + 1) + h], f, sum);
            acc = fmaf(join[w * pitch + e], f, acc);
        }
        if (part) {
            part[e] = acc;
            if (d == 0) part[kPgHeads * D + h] = most, part[kPgHeads * (D + 1) + h] = sum;
        } else if (d < head_dim) {
            out[h * head_dim + d] = sum == 0.0f ? 0.0f : acc / sum;
        }
    }
}

// Warp w's share of an item's runs (w, w + 4, ...; the first run's partial
// lies in slot 1 of its CTA, the others' in slot 0) as a partial in `to`.  A
// lane takes four values of every 128 with 16-byte loads, two runs in flight
// (with four the main loop spills registers).
template <int D>
__device__ __forceinline__ void gather_runs(const float *partial, int runs, uint32_t heads, float *to) {
    constexpr int kPart = kPgHeads * (D + 2), kVecs = kPgHeads * D / 128, kAtOnce = 2;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto slot = [&](int k) { return partial + (uint64_t)(k ? 2 * k : 1) * kPart; };
    float most = -INFINITY;  // of head lane % 8
#pragma unroll 8
    for (int k = warp + kPgWarps * (lane >> 3); k < runs; k += kPgWarps * 4)
        most = fmaxf(most, __ldcg(slot(k) + kPgHeads * D + (lane & 7)));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
    const float base = most == -INFINITY ? 0.0f : most;
    float sum = 0.0f;
    float4 acc[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) acc[i] = make_float4(0, 0, 0, 0);
    for (int k0 = warp; k0 < runs; k0 += kPgWarps * kAtOnce) {
        float f[kAtOnce], part[kAtOnce];
        float4 v[kAtOnce][kVecs];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            const int k = k0 + j * kPgWarps;
            const float *from = slot(min(k, runs - 1));
            f[j] = __ldcg(from + kPgHeads * D + (lane & 7));
            part[j] = __ldcg(from + kPgHeads * (D + 1) + (lane & 7));
#pragma unroll
            for (int i = 0; i < kVecs; ++i)
                v[j][i] = (i * 128 + lane * 4) / D < (int)heads
                              ? __ldcg(reinterpret_cast<const float4 *>(from + i * 128 + lane * 4))
                              : make_float4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            f[j] = k0 + j * kPgWarps < runs ? exp2_fast(f[j] - base) : 0.0f;
            sum = fmaf(part[j], f[j], sum);
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                const int h = (i * 128 + lane * 4) / D;
                const float fh = __shfl_sync(0xffffffffu, f[j], h);
                acc[i].x = fmaf(v[j][i].x, fh, acc[i].x), acc[i].y = fmaf(v[j][i].y, fh, acc[i].y);
                acc[i].z = fmaf(v[j][i].z, fh, acc[i].z), acc[i].w = fmaf(v[j][i].w, fh, acc[i].w);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kVecs; ++i) *reinterpret_cast<float4 *>(to + i * 128 + lane * 4) = acc[i];
    if (lane < kPgHeads) to[kPgHeads * D + lane] = most, to[kPgHeads * (D + 1) + lane] = sum;
}

// Sequences without tokens: rows of zeros.
__device__ __forceinline__ void zero_rows(const PagedArgs &a) {
    for (uint32_t s = blockIdx.x; s < a.pt.sequences; s += gridDim.x) {
        if (seq_length(a, s)) continue;
        for (uint32_t e = threadIdx.x; e < a.q_heads * a.head_dim; e += kPgWarps * 32)
            a.out[(uint64_t)s * a.q_heads * a.head_dim + e] = 0.0f;
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(kPgWarps * 32, PagedShape<T, D>::kCtas) paged_gqa_kernel(const PagedArgs a) {
    using S = PagedShape<T, D>;
    using Type = PageType<T>;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ long long s_scan[kPgWarps];
    __shared__ PagedCursor<S::kUnit> s_start;
    __shared__ uint32_t s_mask[kPgWarps][S::kStages];
    __shared__ unsigned s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_trigger();

    // The list: places before each thread's sequences, and their total.
    const uint32_t items = a.kv_heads * a.passes, sequences = a.pt.sequences;
    const uint32_t per = (sequences + kPgWarps * 32 - 1) / (kPgWarps * 32);
    const uint32_t seq0 = min(sequences, tid * per), seq1 = min(sequences, seq0 + per);
    long long mine = 0;
    for (uint32_t s = seq0; s < seq1; ++s) mine += (long long)item_places(units_of<S::kUnit>(seq_length(a, s))) * items;
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) s_scan[warp] = upto;
    __syncthreads();
    long long before = upto - mine, total = 0;
    for (int w = 0; w < kPgWarps; ++w) {
        if (w < warp) before += s_scan[w];
        total += s_scan[w];
    }
    const long long ctas = min((long long)gridDim.x, total);
    if ((long long)blockIdx.x >= ctas) {
        zero_rows(a);
        return;
    }
    const long long first = total * blockIdx.x / ctas, end = total * (blockIdx.x + 1) / ctas;
    if (first >= before && first < before + mine) {
        long long left = first - before;
        PagedCursor<S::kUnit> c;
        for (c.seq = seq0;; ++c.seq) {  // (bounded whatever another stream does to the lengths)
            c.len = seq_length(a, c.seq);
            c.units = units_of<S::kUnit>(c.len);
            const long long n = (long long)item_places(c.units) * items;
            if (left < n || c.seq + 1 >= seq1) break;
            left -= n;
        }
        c.item = (uint32_t)(left / (c.units + 1));
        const int place = (int)(left - (long long)c.item * (c.units + 1));
        c.unit = max(place - 1, 0), c.at = place == 0;
        s_start = c;
    }
    __syncthreads();

    const uint32_t ring = smem_u32(smem) + warp * S::kStages * S::kStageBytes;
    const uint32_t row_bytes = a.head_dim * (uint32_t)sizeof(T);
    const int my_chunk = lane % S::kChunks, my_row = lane / S::kChunks;  // of each load below
    const unsigned char *keys = static_cast<const unsigned char *>(a.keys) + my_chunk * 16;
    const unsigned char *values = static_cast<const unsigned char *>(a.values) + my_chunk * 16;
    const bool in_row = (uint32_t)my_chunk * 16 < row_bytes;
    const uint32_t group = a.q_heads / a.kv_heads;
    PagedCursor<S::kUnit> load = s_start, use = s_start;
    const int count = (int)(end - first);  // places

    // Lane r (modulo the tile) finds token r of the warp's tile at the cursor:
    // its row among all rows of the pages, or kNone.
    constexpr uint32_t kNone = 0xffffffffu;
    auto find = [&](const PagedCursor<S::kUnit> &c) -> uint32_t {
        const uint32_t pos = (uint32_t)c.unit * S::kUnit + warp * S::kTile + lane % S::kTile;
        if (pos >= (uint32_t)c.len) return kNone;
        const uint32_t slot = a.pt.slot_ids ? (uint32_t)a.pt.slot_ids[c.seq] : c.seq;
        const uint32_t p = a.page_magic ? __umulhi(pos, a.page_magic) >> a.page_shift : pos, off = pos - p * a.pt.page_tokens;
        const int page = a.pt.table[(uint64_t)slot * a.pt.max_pages + p];
        if (page < 0 || (uint64_t)page >= a.pt.pages) return kNone;
        return ((uint32_t)page * a.kv_heads + c.item / a.passes) * a.pt.page_tokens + off;
    };
    uint32_t row_at = load.at < count ? find(load) : kNone;
    // Starts the loads of the next tile into `stage`, then looks the tile
    // after it up (and, where a new item begins, touches its queries, so that
    // they wait in L1 when the item's turn comes).
    auto issue = [&](int stage) {
        if (load.at < count) {
            const uint32_t to = ring + stage * S::kStageBytes;
            const unsigned seen = __ballot_sync(0xffffffffu, row_at != kNone) & S::kFull;
            if (lane == 0) s_mask[warp][stage] = seen;
            constexpr int kSteps = S::kTile * S::kChunks / 32, kRows = 32 / S::kChunks;  // loads of a lane; rows of each
            if (a.aligned && seen == S::kFull) {
                // Whole rows, and 16 tokens to a page at least: one address for each 16.
                constexpr int kRun = S::kTile < 16 ? S::kTile : 16;
#pragma unroll
                for (int u = 0; u < S::kTile / kRun; ++u) {
                    const uint64_t from = (uint64_t)(__shfl_sync(0xffffffffu, row_at, u * kRun) + my_row) * S::kPitch;
                    const unsigned char *k = keys + from, *v = values + from;
#pragma unroll
                    for (int i = 0; i < kSteps * kRun / S::kTile; ++i) {
                        const int row = u * kRun + i * kRows + my_row;
                        cp_async16(to + row * S::kPitch + S::k_chunk(row, my_chunk) * 16, k + i * kRows * S::kPitch);
                        cp_async16(to + (S::kTile + row) * S::kPitch + S::v_chunk(row, my_chunk) * 16,
                                   v + i * kRows * S::kPitch);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    const int row = i * kRows + my_row;
                    const uint32_t at = __shfl_sync(0xffffffffu, row_at, row);
                    const bool there = at != kNone && in_row;
                    const uint64_t from = (uint64_t)(there ? at : 0) * row_bytes;
                    cp_async16(to + row * S::kPitch + S::k_chunk(row, my_chunk) * 16, keys + from, there ? 16 : 0);
                    cp_async16(to + (S::kTile + row) * S::kPitch + S::v_chunk(row, my_chunk) * 16, values + from,
                               there ? 16 : 0);
                }
            }
            load.next(a, items);
            if (load.at < count) {
                row_at = find(load);
                if (load.unit == 0) {
                    const uint32_t pass = load.item % a.passes, heads = min((uint32_t)kPgHeads, group - pass * kPgHeads);
                    const uint32_t e = lane * (kPgHeads * D / 32);
                    if (e < heads * a.head_dim) {
                        float touched;
                        asm volatile("ld.global.ca.f32 %0, [%1];" : "=f"(touched) : "l"(
                            a.q + ((uint64_t)load.seq * a.q_heads + load.item / a.passes * group + pass * kPgHeads) * a.head_dim + e));
                    }
                }
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < S::kStages - 1; ++s) issue(s);
    zero_rows(a);  // (while the first loads are under way)

    // Per-item state: query parts, scale of a raw score to base 2, running
    // maximum and sum of head g (this lane's tokens), weighted values.  MMA
    // accumulators start from zero and are added by FMA: the tensor core cuts
    // its sums where an FMA rounds, and over a long run the cuts add up (1.4e-6
    // of an F32 output against 0.3e-6).
    constexpr int kParts = Type::kParts, kQBlocks = S::kF32 ? D / 4 : D / 8, kSub = S::kTile / 16, kOct = S::kTile / 8;
    uint32_t qr[kQBlocks][kParts];
    float unit_scale = 1.0f, m = -INFINITY, l = 0.0f, o[D / 8][2];
    int stage = 0, begun = 0;
    bool fresh = true;

    while (use.at < count) {
        cp_async_wait<S::kStages - 2>();
        __syncwarp();
        issue(stage == 0 ? S::kStages - 1 : stage - 1);
        const uint32_t pass = use.item % a.passes, kvh = use.item / a.passes;
        const uint32_t heads = min((uint32_t)kPgHeads, group - pass * kPgHeads);
        const uint64_t head0 = (uint64_t)use.seq * a.q_heads + kvh * group + pass * kPgHeads;
        if (fresh) {
            fresh = false;
            begun = use.at;
            m = -INFINITY, l = 0.0f;
#pragma unroll
            for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = 0.0f;
            const float *qh = a.q + (head0 + g) * a.head_dim;
            const float to_base2 = 1.4426950408889634f / sqrtf((float)a.head_dim);
            if constexpr (S::kF32) {
#pragma unroll
                for (int b = 0; b < D / 16; ++b) {
                    float4 v = make_float4(0, 0, 0, 0);
                    const uint32_t d = b * 16 + t * 4;
                    if (g < (int)heads && d < a.head_dim) v = *reinterpret_cast<const float4 *>(qh + d);
                    split_tf32(v.x * to_base2, qr[b * 4 + 0][0], qr[b * 4 + 0][1]);
                    split_tf32(v.y * to_base2, qr[b * 4 + 1][0], qr[b * 4 + 1][1]);
                    split_tf32(v.z * to_base2, qr[b * 4 + 2][0], qr[b * 4 + 2][1]);
                    split_tf32(v.w * to_base2, qr[b * 4 + 3][0], qr[b * 4 + 3][1]);
                }
            } else {
                float2 v[D / 8];
                float most = 0.0f;
#pragma unroll
                for (int b = 0; b < D / 8; ++b) {
                    const uint32_t d = b * 8 + t * 2;
                    v[b] = make_float2(0, 0);
                    if (g < (int)heads && d < a.head_dim) v[b] = *reinterpret_cast<const float2 *>(qh + d);
                    v[b].x *= to_base2, v[b].y *= to_base2;
                    most = fmaxf(most, fmaxf(fabsf(v[b].x), fabsf(v[b].y)));
                }
                float up = 1.0f;
                if constexpr (Type::kShift > 0) {
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                    unit_scale = 1.0f;
                    if (most > 0.0f && most < INFINITY) {
                        const int e = min(max(14 - ilogbf(most), -100), 100);
                        up = ldexpf(1.0f, e), unit_scale = ldexpf(1.0f, -e);
                    }
                }
#pragma unroll
                for (int b = 0; b < D / 8; ++b) split_pair(v[b].x * up, v[b].y * up, qr[b], T{});
            }
        }

        const uint32_t seen = s_mask[warp][stage];
        const uint32_t kt = ring + stage * S::kStageBytes, vt = kt + S::kTile * S::kPitch;
        if (seen) {
            // Scores.  This lane: head g, tokens 2t and 2t + 1 of each 8.
            float s[kOct * 2];
            if constexpr (S::kF32) {
#pragma unroll
                for (int nt = 0; nt < kOct; ++nt) s[2 * nt] = s[2 * nt + 1] = 0.0f;
#pragma unroll
                for (int u = 0; u < kOct; u += 2) {
#pragma unroll
                    for (int b = 0; b < D / 16; ++b) {
#pragma unroll
                        for (int nt = u; nt < u + 2 && nt < kOct; ++nt) {
                            const int row = nt * 8 + g;
                            const float4 k = lds4(kt + row * S::kPitch + S::k_chunk(row, b * 4 + t) * 16);
                            uint32_t hx, lx, hy, ly, hz, lz, hw, lw;
                            split_tf32(k.x, hx, lx), split_tf32(k.y, hy, ly);
                            split_tf32(k.z, hz, lz), split_tf32(k.w, hw, lw);
                            const uint32_t(*qb)[kParts] = qr + b * 4;
                            float c[4];
                            mma_tf32(c, qb[0][0], qb[0][1], qb[1][0], qb[1][1], lx, ly, 0.0f, 0.0f, 0.0f, 0.0f);
                            mma_tf32(c, qb[2][0], qb[2][1], qb[3][0], qb[3][1], lz, lw, c[0], c[1], c[2], c[3]);
                            mma_tf32(c, qb[0][0], qb[0][1], qb[1][0], qb[1][1], hx, hy, c[0], c[1], c[2], c[3]);
                            mma_tf32(c, qb[2][0], qb[2][1], qb[3][0], qb[3][1], hz, hw, c[0], c[1], c[2], c[3]);
                            s[nt * 2] += c[0] + c[2], s[nt * 2 + 1] += c[1] + c[3];
                        }
                    }
                }
            } else {
#pragma unroll
                for (int u = 0; u < kSub; ++u) {  // 16 tokens at a time
                    float *su = s + u * 4;
                    su[0] = su[1] = su[2] = su[3] = 0.0f;
#pragma unroll
                    for (int b2 = 0; b2 < D / 32; ++b2) {
                        float c[2][4];
#pragma unroll
                        for (int b = 2 * b2; b < 2 * b2 + 2; ++b) {
                            const int i = lane >> 3, row = u * 16 + (i >> 1) * 8 + (lane & 7), chunk = 2 * b + (i & 1);
                            uint32_t k[4];
                            ldsm4(k, kt + row * S::kPitch + S::k_chunk(row, chunk) * 16);
#pragma unroll
                            for (int nt = 0; nt < 2; ++nt)
                                mma_parts<kParts>(c[nt], qr[2 * b], qr[2 * b + 1], k[2 * nt], k[2 * nt + 1], b > 2 * b2);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) su[i] += c[i / 2][i % 2] + c[i / 2][i % 2 + 2];
                    }
                }
            }
            if constexpr (Type::kShift > 0) {
#pragma unroll
                for (int i = 0; i < kOct * 2; ++i) s[i] *= unit_scale;
            }
            if (seen != S::kFull) {
#pragma unroll
                for (int i = 0; i < kOct * 2; ++i) {
                    const int token = i / 2 * 8 + i % 2;
                    s[i] = seen >> (token + 2 * t) & 1 ? s[i] : -INFINITY;
                }
            }
            float top = s[0];
#pragma unroll
            for (int i = 1; i < kOct * 2; ++i) top = fmaxf(top, s[i]);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float now = fmaxf(top, m), base = now == -INFINITY ? 0.0f : now;
            const float keep = exp2_fast(m - base);
            m = now;
            l *= keep;
            float p[kOct * 2];
#pragma unroll
            for (int i = 0; i < kOct * 2; ++i) p[i] = exp2_fast(s[i] - (base - Type::kShift)), l += p[i];
            // Weighted values.
            if constexpr (S::kF32) {
                uint32_t h[kOct * 2], r[kOct * 2];
#pragma unroll
                for (int i = 0; i < kOct * 2; ++i) split_tf32(p[i], h[i], r[i]);
#pragma unroll
                for (int b = 0; b < D / 32; ++b) {
                    float c[4][4] = {};
#pragma unroll
                    for (int nt = 0; nt < kOct; ++nt) {
                        const int r0 = nt * 8 + 2 * t, r1 = r0 + 1;
                        const float4 v0 = lds4(vt + r0 * S::kPitch + S::v_chunk(r0, b * 8 + g) * 16);
                        const float4 v1 = lds4(vt + r1 * S::kPitch + S::v_chunk(r1, b * 8 + g) * 16);
                        const float x0[4] = {v0.x, v0.y, v0.z, v0.w}, x1[4] = {v1.x, v1.y, v1.z, v1.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t a0, b0, a1, b1;
                            split_tf32(x0[j], a0, b0), split_tf32(x1[j], a1, b1);
                            mma_tf32(c[j], h[2 * nt], r[2 * nt], h[2 * nt + 1], r[2 * nt + 1], b0, b1, c[j][0], c[j][1],
                                     c[j][2], c[j][3]);
                            mma_tf32(c[j], h[2 * nt], r[2 * nt], h[2 * nt + 1], r[2 * nt + 1], a0, a1, c[j][0], c[j][1],
                                     c[j][2], c[j][3]);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int i = 0; i < 2; ++i) o[b * 4 + j][i] = fmaf(o[b * 4 + j][i], keep, c[j][i] + c[j][i + 2]);
                }
            } else {
                uint32_t pp[kSub * 2][kParts];
#pragma unroll
                for (int i = 0; i < kSub * 2; ++i) split_pair(p[2 * i], p[2 * i + 1], pp[i], T{});
#pragma unroll
                for (int b = 0; b < D / 16; ++b) {
                    float c[2][4];
#pragma unroll
                    for (int u = 0; u < kSub; ++u) {
                        const int i = lane >> 3, row = u * 16 + (i & 1) * 8 + (lane & 7), chunk = 2 * b + (i >> 1);
                        uint32_t v[4];
                        ldsm4_trans(v, vt + row * S::kPitch + S::v_chunk(row, chunk) * 16);
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            mma_parts<kParts>(c[j], pp[2 * u], pp[2 * u + 1], v[2 * j], v[2 * j + 1], u > 0);
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int i = 0; i < 2; ++i) o[2 * b + j][i] = fmaf(o[2 * b + j][i], keep, c[j][i] + c[j][i + 2]);
                }
            }
        }
        // The run's last unit of this item: join the warps.
        if (use.unit + 1 == use.units || use.at + 1 == count) {
            fresh = true;
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            // In the stage just used, which the next step's loads fill again.
            constexpr uint32_t kJoinPitch = S::kStages * S::kStageBytes / 4;
            float *join = reinterpret_cast<float *>(smem + stage * S::kStageBytes), *mine_o = join + warp * kJoinPitch;
            __syncwarp();
            if (t == 0) mine_o[kPgHeads * D + g] = m, mine_o[kPgHeads * (D + 1) + g] = l;
#pragma unroll
            for (int j = 0; j < D / 8; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    // Column 2t + i of tile j: the F32 tiles interleave four dimensions.
                    const int d = S::kF32 ? j / 4 * 32 + 4 * (2 * t + i) + j % 4 : j * 8 + 2 * t + i;
                    mine_o[g * D + d] = o[j][i];
                }
            __syncthreads();
            float *out = a.out + head0 * a.head_dim;
            const bool starts = use.unit == use.at - begun;  // this run has the item's first unit
            if (starts && use.unit + 1 == use.units) {
                join_warps<D>(join, kJoinPitch, heads, a.head_dim, out, nullptr);
            } else {
                // A run that starts the item writes slot 1 of its CTA, one that goes on with it slot 0.
                join_warps<D>(join, kJoinPitch, heads, a.head_dim, nullptr,
                              a.work.partial + (uint64_t)(2 * blockIdx.x + starts) * S::kPart);
                // The places [u0, u1) of the item's units and the CTAs that own its ends.
                const long long u0 = first + use.at - use.unit, u1 = u0 + use.units;
                const int c0 = (int)(((u0 + 1) * ctas - 1) / total), runs = (int)((u1 * ctas - 1) / total) - c0 + 1;
                __syncthreads();
                if (tid == 0) {
                    __threadfence();  // the block's partial, then its arrival
                    s_last = atomicAdd(&a.work.arrived[c0], 1u) + 1 == (unsigned)runs;
                    if (s_last) a.work.arrived[c0] = 0;
                    __threadfence();  // and the others' before what the block reads next
                }
                __syncthreads();
                if (s_last) {
                    gather_runs<D>(a.work.partial + (uint64_t)2 * c0 * S::kPart, runs, heads, mine_o);
                    __syncthreads();
                    join_warps<D>(join, kJoinPitch, heads, a.head_dim, out, nullptr);
                }
            }
            __syncthreads();
        }
        stage = stage + 1 == S::kStages ? 0 : stage + 1;
        use.next(a, items);
    }
    cp_async_wait<0>();
}

template <typename T, int D>
int32_t paged_gqa_run(const PagedArgs &a0, void *workspace, cudaStream_t stream) {
    using S = PagedShape<T, D>;
    PagedArgs a = a0;
    a.aligned = a.pt.page_tokens % 16 == 0 && a.head_dim == D;
    const int64_t wave = (int64_t)sm_count() * S::kCtas;
    a.work.arrived = static_cast<unsigned *>(workspace);
    a.work.partial = reinterpret_cast<float *>(static_cast<char *>(workspace) + 16384);
    // As many CTAs as the workspace has slots for, whatever the device.
    const int64_t slots = (MF_PAGED_WORKSPACE_BYTES - 16384) / (sizeof(float) * 2 * S::kPart);
    const int64_t most = (int64_t)a.pt.sequences * a.kv_heads * a.passes *
                         (1 + ((int64_t)a.pt.max_pages * a.pt.page_tokens + S::kUnit - 1) / S::kUnit);
    const int64_t grid = std::min({wave, slots, most, (int64_t)4096});
    if (most / grid >= INT32_MAX) return fail(MF_OVERFLOW, "the page table's capacity exceeds the 32-bit work list");
    const uint64_t row_bytes = (uint64_t)a.pt.sequences * a.q_heads * a.head_dim * sizeof(float);
    if (overlap(a.out, row_bytes, a.q, row_bytes))
        return fail(MF_INVALID_ARGUMENT, "paged attention output must not overlap its query");
    static std::atomic<uint64_t> ready{0};
    if (int32_t st = allow_smem(paged_gqa_kernel<T, D>, S::kSmem, ready)) return st;
    return launch(paged_gqa_kernel<T, D>, dim3((unsigned)grid), dim3(kPgWarps * 32), S::kSmem, stream,
                  "paged_gqa_kernel", a);
}

}  // namespace

int32_t paged_gqa(float *out, const float *q, const void *key_pages, const void *value_pages, int32_t dtype,
                  const PagedTable &pt, const int32_t *lengths, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim,
                  void *workspace, cudaStream_t stream) {
    if (!pt.sequences) return MF_OK;
    PagedArgs a;
    a.out = out, a.q = q, a.keys = key_pages, a.values = value_pages, a.pt = pt, a.lengths = lengths;
    a.q_heads = q_heads, a.kv_heads = kv_heads, a.head_dim = head_dim;
    a.passes = (q_heads / kv_heads + kPgHeads - 1) / kPgHeads;
    a.work = PagedWork{};
    // ceil(2^(32 + shift) / page_tokens) with shift = ceil(log2) - 1: exact for
    // positions below 2^31.
    a.page_shift = 0;
    while ((2u << a.page_shift) < pt.page_tokens) ++a.page_shift;
    a.page_magic = pt.page_tokens == 1 ? 0 : (uint32_t)(((1ull << (32 + a.page_shift)) + pt.page_tokens - 1) / pt.page_tokens);
    if (head_dim <= 64)
        return dtype == MF_PAGE_F32   ? paged_gqa_run<float, 64>(a, workspace, stream)
               : dtype == MF_PAGE_F16 ? paged_gqa_run<__half, 64>(a, workspace, stream)
                                      : paged_gqa_run<__nv_bfloat16, 64>(a, workspace, stream);
    return dtype == MF_PAGE_F32   ? paged_gqa_run<float, 128>(a, workspace, stream)
           : dtype == MF_PAGE_F16 ? paged_gqa_run<__half, 128>(a, workspace, stream)
                                  : paged_gqa_run<__nv_bfloat16, 128>(a, workspace, stream);
}

}  // namespace mf
