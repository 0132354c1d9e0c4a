// Sampling a token id per row of logits.
//
// With w_i = exp((l_i - max) / T) and the order "larger logit first, equal
// logits by index", a row keeps the first top_k tokens (their mass M), of
// those each whose mass before it is below top_p * M, of those each with
// w_i >= min_p; the id is the first kept token, in index order, whose running
// kept mass exceeds u times the kept mass.  Both cuts are prefixes of the
// same order, so they come down to one place in it: the last token that
// stays, as (logit, index).
//
// Weights are integers, round(w * 2^shift), and every sum is exact: a result
// does not depend on how the row was split or in which order atomics arrived,
// and a running mass near a border is not moved by rounding (F32 sums over
// 65536 tokens would move borders by 1e-3 of a token's weight).  shift is 46,
// less where the width would let a sum pass 2^62.
//
// The work.  A cluster of CTAs holds a row in shared memory, so DRAM is read
// once, and shares maxima, masses and lists through distributed shared memory
// (rows past 360448 tokens are read again from L2).  The first pass takes the
// maximum (and each thread's); with top-k, the threads' maxima bound the
// top_k-th logit from below so closely that the tokens above the bound, hardly
// more than top_k, are listed in one CTA, ranked against one another and drawn
// from without another pass.  A cut by mass alone first tries the tokens within
// exp(-8) of the largest the same way.  Rows that this does not settle (a flat
// row with top-p) get a histogram of (max - l) / T, then a list of the bin
// that the cut falls in.
//
// Measured (B200): 512 rows of 65536 with mixed settings 109 us, where reading
// them takes 20.  What bounds it is each row's chain (load, maximum, bound,
// list, rank, draw, each ended by a barrier of the CTA or the cluster: 59 us
// for 512 greedy rows, 78 with top-k 50, 87 without a filter, 112 with top-p
// 0.9 at temperature 0.6, 264 with top-p 0.95 at 1.3), which two CTAs per SM
// overlap only in part.  One row 9 to 13 us, all latency (22 where it is flat).
// With all but 100 logits of a row at -infinity a CTA may have too few finite
// maxima to bound top-k 50, and the row goes to the histogram: 512 rows 86-90 us.
// Rows past 360448 tokens spill 8 bytes.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <float.h>

#include <algorithm>

#include "mf_common.cuh"
#include "packed_kernels.h"
#include "tc_sm100.cuh"

namespace mf {

namespace {

namespace cg = cooperative_groups;

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kChunk = 128;  // tokens of a warp's step: four a lane
constexpr int kBins = 4096;
constexpr float kBinScale = 124.0f;  // bins of (max - l) / T of 1/124: the last one's weights round to 0
constexpr int kSortBins = 256;
constexpr int kList = 512;
constexpr float kNear = 8.0f;  // a cut by mass alone: (max - l) / T of the tokens listed
constexpr int kMaxCluster = 8;
constexpr uint64_t kStageFloats = 44 * 1024;  // of a CTA at most
constexpr size_t kMostSmem = 227 * 1024;
constexpr int kPowers = 64, kCopies = 16;
constexpr unsigned kPairs = 64;

using u64 = unsigned long long;
static_assert(kBins * 4 >= 2 * kList * 8, "the ranking's scratch fits the histogram");

// 2^(j / 64).
__device__ const double kPowerTable[kPowers] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0};

// Logits as unsigned integers of the same order, and back.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v == 0.0f ? 0.0f : v);  // -0 equals +0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// A token's place in a row's order: larger is earlier.
__device__ __forceinline__ u64 order_of(float v, uint64_t index) {
    return (u64)order_key(v) << 32 | (0xffffffffu - (uint32_t)index);
}

struct Row {
    float top, half_top;  // largest logit, and half of it
    float floor;    // no weight below: (max - l) / T > 34
    float inverse;  // 2 / T in F32, for the bins
    double rate;    // log2(e) / T
    double unit;    // 1.5 * 2^(52 - shift): adding it rounds to steps of 2^-shift
};

// What a row asks for, in the units of its weights.
struct Wanted {
    bool by_count, by_mass;
    u64 count, least;  // top_k; min_p's weight
    float p, u;
};

// What the CTAs of a cluster tell one another, and scratch.
struct alignas(16) Shared {
    double powers[kPowers * kCopies];  // a half-warp's reads hit 16 banks of 8 bytes
    // Of the histograms, and where those are done with, scratch of the ranking
    // (beside one another they would leave rows of 145000 to 160000 one CTA per
    // SM: 256 rows of 151936 205 us for 131).
    alignas(8) unsigned count[kBins];
    __device__ __forceinline__ u64 *sorted() { return reinterpret_cast<u64 *>(count); }
    __device__ __forceinline__ u64 *by_rank() { return sorted() + kList; }
    u64 mass[256];  // of the digits of a bin that is too full
    // Listed tokens: key and place, the halves of their order.
    uint32_t keys[kList], places[kList];
    unsigned sort_count[2][kSortBins];  // zero before use
    float top[kMaxCluster], near[kMaxCluster];
    int bad[kMaxCluster];
    u64 kept[kMaxCluster], weight[kMaxCluster];
    u64 cut, cut_mass;  // the last token that stays and the mass up to it
    unsigned listed;
    int settled;
    u64 listed_mass;
    int cross_first, cross_last;  // of the histogram's bins
    u64 cross_before;
    int full;  // the list has overflowed: nothing more goes into it
    // Within the CTA.
    u64 part[kSampleWarps];
    float part_top[kSampleWarps], part_low[kSampleWarps];
    unsigned part_count[kSampleWarps];
    unsigned last_rank;
    unsigned row;
};

// bits(w + unit) for w = exp((v - top) / T) rounded to a step: subtracting
// bits(unit) leaves the weight, and sums may subtract once.  2^y for y = n +
// j / 64 + f, |f| <= 1/128: 2^(n + j / 64) from the table, 2^f by its Taylor
// series to f^3 (the rest is below 2^-34 of the weight: over 65536 equal
// tokens it moves a border by 1e-9 of the mass).
__device__ __forceinline__ u64 weight_bits(float v, const Row &r, const Shared &s) {
    constexpr double kMagic = 6755399441055744.0 / kPowers;  // 1.5 * 2^52 / 64: sums round to 1/64
    constexpr double kLn2 = 0.69314718055994530942;
    const double d = (double)v - (double)r.top;
    const double t = fma(d, r.rate, kMagic);
    const double f = fma(d, r.rate, kMagic - t);
    const int k = __double2loint(t);
    double power = s.powers[(k & (kPowers - 1)) * kCopies + (threadIdx.x & (kCopies - 1))];
    power = __hiloint2double(__double2hiint(power) + (int)((unsigned)k << 14 & 0xfff00000u), __double2loint(power));
    const double q = fma(f, fma(f, kLn2 * kLn2 * kLn2 / 6, kLn2 * kLn2 / 2), kLn2);
    return (u64)__double_as_longlong(v < r.floor ? r.unit : fma(power * f, q, power) + r.unit);
}
__device__ __forceinline__ u64 weight_of(float v, const Row &r, const Shared &s) {
    return weight_bits(v, r, s) - (u64)__double_as_longlong(r.unit);
}

// Half of max - l, whose whole can pass F32's range.
__device__ __forceinline__ float half_gap(float v, const Row &r) { return fmaf(-0.5f, v, r.half_top); }

__device__ __forceinline__ int bin_of(float v, const Row &r) {
    return (int)fminf(half_gap(v, r) * r.inverse * kBinScale, (float)(kBins - 1));
}

// Sum over a warp of values up to 2^48.
__device__ __forceinline__ u64 warp_sum48(u64 v) {
    const unsigned lo = __reduce_add_sync(0xffffffffu, (unsigned)v & 0xffffffu);
    const unsigned hi = __reduce_add_sync(0xffffffffu, (unsigned)(v >> 24));
    return ((u64)hi << 24) + lo;
}

__device__ __forceinline__ u64 warp_upto(u64 v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    return v;
}

__device__ __forceinline__ unsigned warp_upto(unsigned v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    return v;
}

__device__ __forceinline__ u64 block_sum(u64 v, u64 *part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < kSampleWarps; ++w) v += part[w];
    return v;
}

__device__ __forceinline__ u64 mass_limit(float p, u64 mass) { return max((u64)ceil((double)p * (double)mass), 1ull); }

__device__ __forceinline__ u64 mass_target(float u, u64 total) {
    const u64 t = u > 0.0f ? (u64)floor((double)fminf(u, 1.0f) * (double)total) : 0;
    return min(t, total - 1);
}

// A CTA's share of a row: `size` tokens from index `first`, in shared memory
// or in global memory (rows too wide for a cluster).
template <bool kStaged>
struct Slice {
    const float *x;
    uint64_t first, row_chunks;
    int size, chunks, most_chunks;  // most: of any CTA of the row
    bool aligned;       // to 16 bytes
    float index_scale;  // bins of a counting sort per token of the row

    // Tokens 4 lane .. 4 lane + 3 of a chunk; -infinity past the end.
    __device__ __forceinline__ float4 four(int chunk) const {
        const int at = chunk * kChunk + (threadIdx.x & 31) * 4;
        if constexpr (kStaged) return *reinterpret_cast<const float4 *>(x + at);
        if (aligned && at + 4 <= size) return __ldg(reinterpret_cast<const float4 *>(x + at));
        float4 v;
        v.x = at + 0 < size ? x[at + 0] : -INFINITY;
        v.y = at + 1 < size ? x[at + 1] : -INFINITY;
        v.z = at + 2 < size ? x[at + 2] : -INFINITY;
        v.w = at + 3 < size ? x[at + 3] : -INFINITY;
        return v;
    }

    // Calls f(chunk, four tokens) for this warp's chunks, kLoads of them loaded
    // at a time where they come from global memory.
    template <int kLoads, typename F>
    __device__ __forceinline__ void each(F f) const {
        constexpr int kAhead = kStaged ? 1 : kLoads;
        const int warp = threadIdx.x >> 5;
        for (int c0 = warp; c0 < chunks; c0 += kSampleWarps * kAhead) {
            float4 v[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (c0 + i * kSampleWarps < chunks) v[i] = four(c0 + i * kSampleWarps);
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (c0 + i * kSampleWarps < chunks) f(c0 + i * kSampleWarps, v[i]);
        }
    }
};

// The CTA's share of the bound from below on the top_k-th logit: a value that k
// = ceil(top_k / ranks) of its threads' maxima reach, and few more (the lower
// edge of the bin, of 256 from the largest to the smallest maximum, in which
// the k-th lies, with a hundredth of a bin for F32's rounding); -infinity where
// it has fewer maxima.
__device__ __forceinline__ float near_bound(Shared &s, float mine, float hi, float lo, int k, float temperature) {
    const int lane = threadIdx.x & 31;
    lo = fmaxf(lo, hi - 34.0f * temperature);
    const float scale = hi > lo ? 255.0f / (hi - lo) : 0.0f;
    const int bin = mine == -INFINITY ? 256 : (int)fminf((hi - mine) * scale, 255.0f);
    if (bin < 256) atomicAdd(&s.count[bin], 1u);
    __syncthreads();
    if (threadIdx.x < 32) {
        unsigned n[8], sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += n[i] = s.count[lane * 8 + i];
        unsigned before = warp_upto(sum) - sum;
        if (lane == 0) s.cross_last = 256;  // fewer maxima than that
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (before < (unsigned)k && before + n[i] >= (unsigned)k) s.cross_last = lane * 8 + i;
            before += n[i];
        }
    }
    __syncthreads();
    const int last = s.cross_last;  // (the last bin also holds what lies below its edge)
    return last >= 255 ? -INFINITY : scale > 0.0f ? hi - (last + 1.01f) / scale : hi;
}

__device__ __forceinline__ void add_to_list(Shared &s, Shared *lead, float v, uint64_t index) {
    if (*static_cast<volatile int *>(&s.full)) return;
    const unsigned n = atomicAdd(&lead->listed, 1u);
    if (n >= kList) {
        s.full = 1;
        return;
    }
    lead->keys[n] = order_key(v), lead->places[n] = 0xffffffffu - (uint32_t)index;
}

// The rank, larger first, of this thread's `order` (unlike all others) among
// the first n threads'.  `bin` (0 .. kSortBins - 1) does not decrease with it:
// a counting sort by bins leaves a few others to compare with.
__device__ __forceinline__ unsigned rank_of(Shared &s, unsigned *sort_count, unsigned n, u64 order, int bin) {
    const int tid = threadIdx.x, lane = tid & 31;
    unsigned slot = 0;
    if (tid < n) slot = atomicAdd(&sort_count[bin], 1u);
    __syncthreads();
    if (tid < 32) {  // each count becomes the sum up to it
        constexpr int kPer = kSortBins / 32;
        unsigned c[kPer], sum = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) sum += c[i] = sort_count[lane * kPer + i];
        unsigned upto = warp_upto(sum) - sum;
#pragma unroll
        for (int i = 0; i < kPer; ++i) sort_count[lane * kPer + i] = upto += c[i];
    }
    __syncthreads();
    unsigned first = 0, last = 0;
    if (tid < n) {
        first = bin ? sort_count[bin - 1] : 0, last = sort_count[bin];
        s.sorted()[first + slot] = order;
    }
    __syncthreads();
    unsigned rank = first;
    for (unsigned i = first; i < last; ++i) rank += s.sorted()[i] > order;
    return rank;
}

// The sum of the values of lower rank (each of the n threads with a token has
// a rank of its own below n), and of all.
__device__ __forceinline__ u64 ranked_before(Shared &s, unsigned n, unsigned rank, u64 value, u64 &total) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid < n) s.by_rank()[rank] = value;
    __syncthreads();
    const u64 v = tid < n ? s.by_rank()[tid] : 0, upto = warp_upto(v);
    if (lane == 31) s.part[warp] = upto;
    __syncthreads();
    u64 before = upto - v;
    total = 0;
    for (int w = 0; w < kSampleWarps; ++w) {
        if (w < warp) before += s.part[w];
        total += s.part[w];
    }
    if (tid < n) s.by_rank()[tid] = before;
    __syncthreads();
    return tid < n ? s.by_rank()[rank] : 0;
}

// Bins of logits from the largest down to `low`, and of indexes.
__device__ __forceinline__ int sort_bin(const Row &row, float v, float low) {
    return (int)fminf(fmaxf((row.top - v) * ((kSortBins - 1) / (row.top - low)), 0.0f), (float)(kSortBins - 1));
}
template <bool kStaged>
__device__ __forceinline__ int index_bin(const Slice<kStaged> &slice, uint32_t place) {
    return (int)fminf((float)(0xffffffffu - place) * slice.index_scale, (float)(kSortBins - 1));
}

// Cut and draw from a list of up to kPairs tokens: eight threads a token
// compare it with all others, adding up the weights before it in the row's
// order, then the kept weights before it in index order.  Three barriers, where
// sorting takes some fourteen: one row 12.5 us for 13.4, 512 rows 115 for 117
// (greedy 60 for 65, top-p 0.9 at temperature 0.6 104 for 113); four threads a
// token, up to 128, 116.
// False where the list does not reach the cut.
__device__ __forceinline__ bool draw_pairs(Shared &s, const Row &row, const Wanted &want, unsigned n, bool whole,
                                           u64 mass, float *out) {
    const unsigned tid = threadIdx.x, log_per = 3, per = 1u << log_per;
    static_assert(kPairs << 3 <= kSampleThreads, "eight threads a token");
    if (tid < n) {
        const uint32_t key = s.keys[tid];
        s.sorted()[tid] = (u64)key << 32 | s.places[tid];
        s.by_rank()[tid] = weight_of(key_value(key), row, s);
    }
    __syncthreads();
    const unsigned mine = tid >> log_per, part = tid & (per - 1);
    const u64 order = mine < n ? s.sorted()[mine] : 0, weight = mine < n ? s.by_rank()[mine] : 0;
    unsigned ahead = 0;
    u64 before = 0;
    for (unsigned j = part; j < n; j += per)
        if (s.sorted()[j] > order) ++ahead, before += s.by_rank()[j];
    for (unsigned o = 1; o < per; o <<= 1) {
        ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    bool stay = mine < n && (!want.by_count || ahead < want.count);
    if (want.by_mass) {
        if (mine < n && ahead == (want.by_count ? (unsigned)want.count : n) - 1) s.listed_mass = before + weight;
        __syncthreads();
        const u64 listed_mass = s.listed_mass, limit = mass_limit(want.p, whole ? mass : listed_mass);
        if (listed_mass < limit) return false;
        stay = stay && before < limit;
    }
    const u64 kept = stay && weight >= want.least ? weight : 0;
    if (part == 0 && mine < n) s.mass[mine] = kept;
    __syncthreads();
    u64 run = 0, total = 0;
    const uint32_t place = (uint32_t)order;
    for (unsigned j = part; j < n; j += per) {
        const u64 w = s.mass[j];
        total += w;
        if (s.places[j] > place) run += w;
    }
    for (unsigned o = 1; o < per; o <<= 1) {
        run += __shfl_xor_sync(0xffffffffu, run, o);
        total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    const u64 target = mass_target(want.u, total);
    if (part == 0 && kept && run <= target && target < run + kept) out[s.row] = (float)(0xffffffffu - place);
    return true;
}

// The usual case of a row with a cut: it falls among the few largest tokens.
// Those from `bound` on are listed in rank 0, which ranks them, cuts, and
// finds the token.  False where they are too many (`mass` is then 0) or do not
// reach the cut (`mass` is then the row's, for a cut by mass alone).  `mine` is
// the thread's maximum: where more of a CTA's reach the bound of a cut by mass
// than its share of the list, the list would overflow, and it and the weights
// are left to the histogram's pass (512 rows with top-p 0.95 at temperature
// 1.3: 259 us for 277; mixed 113 for 115).
template <bool kStaged>
__device__ __forceinline__ bool sample_near(cg::cluster_group &cluster, Shared &s, const Slice<kStaged> &slice,
                                            const Row &row, const Wanted &want, float bound, float mine, float *out,
                                            u64 &mass) {
    static_assert(kList <= kSampleThreads, "a listed token a thread");
    const int tid = threadIdx.x, lane = tid & 31;
    const unsigned ranks = cluster.num_blocks(), rank = cluster.block_rank();
    Shared *lead = cluster.map_shared_rank(&s, 0);
    auto list = [&](int c, const float4 &v4) {
        const float v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int at = c * kChunk + lane * 4 + j;
            if (v[j] >= bound && at < slice.size) add_to_list(s, lead, v[j], slice.first + at);
        }
    };
    const bool whole = want.by_mass && !want.by_count;
    mass = 0;
    const bool flat = whole && __syncthreads_count(mine >= bound) > (int)(kList / ranks);
    if (flat) {
        if (tid == 0) atomicAdd(&lead->listed, kList + 1u);
    } else if (whole) {
        const u64 unit4 = 4 * (u64)__double_as_longlong(row.unit);
        slice.template each<2>([&](int c, const float4 &v) {
            mass += weight_bits(v.x, row, s) + weight_bits(v.y, row, s) + weight_bits(v.z, row, s) +
                    weight_bits(v.w, row, s) - unit4;
            if (__any_sync(0xffffffffu, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= bound)) list(c, v);
        });
        mass = block_sum(mass, s.part);
        if (tid < ranks) cluster.map_shared_rank(&s, tid)->kept[rank] = mass;
    } else {
        slice.template each<8>([&](int c, const float4 &v) {
            if (fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= bound) list(c, v);
        });
    }
    cluster.sync();
    const unsigned n = lead->listed;
    if (whole) {
        mass = 0;
        if (n > kList) return false;
        for (unsigned q = 0; q < ranks; ++q) mass += s.kept[q];
    }
    // Without a mass of the row to reach, the list's length says whether it
    // settles the row, and the CTAs without it are done (rank 0 stays until they
    // have read it and left).
    bool done = n <= kList && (!want.by_count || n >= want.count);
    if (!whole && (!done || rank != 0)) return done;
    if (rank == 0) {
        if (done && n <= kPairs) {
            done = draw_pairs(s, row, want, n, whole, mass, out);
        } else if (done) {
            const uint32_t key = tid < n ? s.keys[tid] : 0, place = tid < n ? s.places[tid] : 0;
            const float value = key_value(key);
            const u64 weight = tid < n ? weight_of(value, row, s) : 0;
            const unsigned ahead = rank_of(s, s.sort_count[0], n, (u64)key << 32 | place,
                                           sort_bin(row, value, fmaxf(bound, row.floor)));
            bool stay = tid < n && (!want.by_count || ahead < want.count);
            if (want.by_mass) {
                u64 listed_mass;
                const u64 before = ranked_before(s, n, ahead, stay ? weight : 0, listed_mass);
                const u64 limit = mass_limit(want.p, whole ? mass : listed_mass);
                done = listed_mass >= limit;
                stay = stay && before < limit;
            }
            if (done) {
                // In index order: larger places first.
                const u64 w = stay && weight >= want.least ? weight : 0;
                u64 total;
                const u64 run = ranked_before(s, n, rank_of(s, s.sort_count[1], n, place, index_bin(slice, place)), w, total);
                const u64 target = mass_target(want.u, total);
                if (w && run <= target && target < run + w) out[s.row] = (float)(0xffffffffu - place);
            }
        }
        if (whole && tid < ranks) cluster.map_shared_rank(&s, tid)->settled = done;
    }
    cluster.sync();
    return whole ? s.settled : true;
}

// The cut of a row, by count or by mass: the place in the row's order of the
// last token with fewer than `limit` tokens (or less than `limit` mass) before
// it, 0 where every token with weight stays; and the mass of what stays.
// With a limit of 0 it is the share p of the row's mass, which the histogram's
// pass then adds up.
// Returns whether chunk_mass then holds each chunk's mass of what stays (and
// is at least `least`).
template <bool kStaged>
__device__ __forceinline__ bool find_cut(cg::cluster_group &cluster, Shared &s, const Slice<kStaged> &slice,
                                         const Row &row, bool by_mass, u64 limit, float p, u64 least, int shift,
                                         u64 *chunk_mass, u64 &cut, u64 &cut_mass) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned ranks = cluster.num_blocks(), rank = cluster.block_rank();
    Shared *lead = cluster.map_shared_rank(&s, 0);

    // The histogram.  Counts are exact.  Masses are sums of F32 weights' first
    // bits, as many as 32-bit sums hold (one native atomic a token): weights
    // of bin b are at most 2^(shift - log2(e) b / 124), and at least half that.
    // They are off by at most 2^-slack of themselves.
    int bits = 31;
    while (bits > 0 && (u64)(slice.most_chunks * kChunk) >> (31 - bits)) --bits;
    const int slack = min(max(bits - 3, 0), 12);
    const float rate = -2.0f * (float)row.rate;  // of half a gap
    auto coarse = [&](int b) { return max(0, shift - (int)(b * (1.4426950408889634f / kBinScale)) - bits); };
    for (int i = tid; i < kBins; i += kSampleThreads) s.count[i] = 0;
    if (tid < kSortBins) s.sort_count[0][tid] = 0;
    if (tid == 0) s.full = 0, s.cross_first = kBins, s.cross_last = -1;
    __syncthreads();
    if (limit) {
        slice.template each<1>([&](int, const float4 &v4) {
            const float v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int b = bin_of(v[j], row);
                if (b < kBins - 1)
                    atomicAdd(&s.count[b],
                              by_mass ? (unsigned)exp2f(fmaf(half_gap(v[j], row), rate, (float)(shift - coarse(b)))) : 1u);
            }
        });
    } else {
        u64 weight = 0;
        slice.template each<1>([&](int, const float4 &v4) {
            const float v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int b = bin_of(v[j], row);
                if (b == kBins - 1) continue;
                const u64 w = weight_of(v[j], row, s);
                weight += w;
                atomicAdd(&s.count[b], (unsigned)(w >> coarse(b)));
            }
        });
        weight = block_sum(weight, s.part);
        if (tid < ranks) cluster.map_shared_rank(&s, tid)->weight[rank] = weight;
    }
    cluster.sync();
    // Each rank adds up its part of the bins, a few consecutive ones a thread,
    // and finds those that the cut can lie in: the running sum reaches the
    // limit there.
    if (rank == 0 && tid == 0) s.listed = 0, s.last_rank = 0;
    constexpr int kMost = kBins / kSampleThreads;
    const int per = kMost / (int)ranks, bin0 = ((int)rank * kSampleThreads + tid) * per;
    u64 m[kMost], sum = 0;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        m[i] = 0;
        if (i >= per) continue;
        for (unsigned q = 0; q < ranks; ++q) m[i] += cluster.map_shared_rank(&s, q)->count[bin0 + i];
        if (by_mass) m[i] <<= coarse(bin0 + i);
        sum += m[i];
    }
    const u64 upto = warp_upto(sum);
    if (lane == 31) s.part[warp] = upto;
    __syncthreads();
    u64 at = upto - sum, share = 0;
    for (int w = 0; w < kSampleWarps; ++w) {
        if (w < warp) at += s.part[w];
        share += s.part[w];
    }
    if (tid < ranks) cluster.map_shared_rank(&s, tid)->kept[rank] = share;
    cluster.sync();
    for (unsigned q = 0; q < rank; ++q) at += s.kept[q];
    if (!limit) {
        u64 weight = 0;
        for (unsigned q = 0; q < ranks; ++q) weight += s.weight[q];
        limit = mass_limit(p, weight);
    }
    auto off = [&](u64 v) { return by_mass ? v >> slack : 0; };
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        if (m[i] && at - off(at) < limit && at + m[i] + off(at + m[i]) >= limit)
            for (unsigned q = 0; q < ranks; ++q) {
                Shared *o = cluster.map_shared_rank(&s, q);
                atomicMin(&o->cross_first, bin0 + i);
                atomicMax(&o->cross_last, bin0 + i);
                if (!by_mass) o->cross_before = at;
            }
        at += m[i];
    }
    cluster.sync();
    const int first = s.cross_first, last = s.cross_last;
    // Tokens before those bins: their number (a cut by count), their mass.
    u64 before = by_mass ? 0 : s.cross_before, mass_before = 0;
    slice.template each<1>([&](int c, const float4 &v4) {
        const float v[4] = {v4.x, v4.y, v4.z, v4.w};
        u64 sum = 0, kept = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int b = bin_of(v[j], row);
            if (b == kBins - 1 || (b > last && first < kBins)) continue;
            if (b >= first) {
                add_to_list(s, lead, v[j], slice.first + c * kChunk + lane * 4 + j);
                continue;
            }
            const u64 w = weight_of(v[j], row, s);
            sum += w, kept += w >= least ? w : 0;
        }
        mass_before += sum;
        kept = warp_sum48(kept);
        if (lane == 0) chunk_mass[c] = kept;
    });
    mass_before = block_sum(mass_before, s.part);
    if (tid < ranks) cluster.map_shared_rank(&s, tid)->kept[rank] = mass_before;
    cluster.sync();
    mass_before = 0;
    for (unsigned q = 0; q < ranks; ++q) mass_before += s.kept[q];
    if (first == kBins) {  // the limit lies behind the last token
        cut = 0, cut_mass = mass_before;
        cluster.sync();
        return true;
    }
    unsigned listed = lead->listed;
    const bool split = listed > kList;
    u64 prefix = 0;
    int digit = 64;
    // Too many to rank: split the bins by the order's bits, from the top, 8 at
    // a time, into exact counts and masses (equal logits end at their indexes).
    while (listed > kList && digit > 0) {
        digit -= 8;
        for (int i = tid; i < 256; i += kSampleThreads) s.mass[i] = 0, s.count[i] = 0;
        __syncthreads();
        slice.template each<1>([&](int c, const float4 &v4) {
            const float v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int b = bin_of(v[j], row);
                if (b < first || b > last) continue;
                const u64 o = order_of(v[j], slice.first + c * kChunk + lane * 4 + j);
                if (digit < 56 && o >> (digit + 8) != prefix) continue;
                atomicAdd(&s.count[255 - (o >> digit & 255)], 1u);
                atomicAdd(&s.mass[255 - (o >> digit & 255)], weight_of(v[j], row, s));
            }
        });
        cluster.sync();
        // Rank 0 walks the bins; the others take its word.
        if (rank == 0 && warp == 0) {
            u64 at = before, at_mass = mass_before;
            int found = 0;
            unsigned n = 0;
            for (int b0 = 0; b0 < 256 && !n; b0 += 32) {
                u64 m = 0;
                unsigned k = 0;
                for (unsigned q = 0; q < ranks; ++q) {
                    Shared *o = cluster.map_shared_rank(&s, q);
                    m += o->mass[b0 + lane], k += o->count[b0 + lane];
                }
                const u64 um = warp_upto(m), uk = warp_upto(k);
                const unsigned here = __ballot_sync(0xffffffffu, k && (by_mass ? at_mass + um : at + uk) >= limit);
                const int l = here ? __ffs(here) - 1 : 31;
                const u64 em = here ? um - m : um, ek = here ? uk - k : uk;  // ahead of the bin, or of the next 32
                at += __shfl_sync(0xffffffffu, ek, l), at_mass += __shfl_sync(0xffffffffu, em, l);
                if (here) n = __shfl_sync(0xffffffffu, k, l), found = b0 + l;
            }
            if (lane == 0)
                for (unsigned q = 0; q < ranks; ++q) {
                    Shared *o = cluster.map_shared_rank(&s, q);
                    o->cut = prefix << 8 | (255 - found);
                    o->cut_mass = at_mass;
                    o->kept[0] = at;
                    o->listed = n;
                }
        }
        cluster.sync();
        prefix = s.cut, mass_before = s.cut_mass, before = s.kept[0], listed = s.listed;
        cluster.sync();
        if (listed > kList && digit > 0) continue;
        if (rank == 0 && tid == 0) s.listed = 0;
        if (tid == 0) s.full = 0;
        cluster.sync();
        slice.template each<1>([&](int c, const float4 &v4) {
            const float v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int b = bin_of(v[j], row);
                if (b < first || b > last) continue;
                const u64 o = order_of(v[j], slice.first + c * kChunk + lane * 4 + j);
                if (o >> digit != prefix) continue;
                add_to_list(s, lead, v[j], slice.first + c * kChunk + lane * 4 + j);
            }
        });
        cluster.sync();
    }
    if (rank == 0) {
        const unsigned n = min(s.listed, (unsigned)kList);
        const uint32_t key = tid < n ? s.keys[tid] : 0, place = tid < n ? s.places[tid] : 0;
        const float value = key_value(key);
        const u64 weight = tid < n ? weight_of(value, row, s) : 0;
        // Bins of the few histogram bins listed; all in one where those were split.
        const int bin = split ? 0
                              : (int)fminf(fmaxf((half_gap(value, row) * row.inverse * kBinScale - first) *
                                                     ((float)kSortBins / (last + 1 - first)), 0.0f), (float)(kSortBins - 1));
        const unsigned ahead = rank_of(s, s.sort_count[0], n, (u64)key << 32 | place, bin);
        u64 unused;
        const u64 mass = ranked_before(s, n, ahead, weight, unused);
        const bool stay = tid < n && (by_mass ? mass_before + mass : before + ahead) < limit;
        if (stay) atomicMax(&s.last_rank, ahead + 1);
        __syncthreads();
        if (stay && ahead + 1 == s.last_rank)
            for (unsigned q = 0; q < ranks; ++q) {
                Shared *o = cluster.map_shared_rank(&s, q);
                o->cut = (u64)key << 32 | place;
                o->cut_mass = mass_before + mass + weight;
            }
        if (stay && !split && weight >= least) {
            // Into its chunk, wherever that is.
            const uint64_t chunk = (0xffffffffu - place) / kChunk;
            const unsigned owner = (unsigned)(((chunk + 1) * ranks - 1) / slice.row_chunks);
            atomicAdd(cluster.map_shared_rank(chunk_mass, owner) + (chunk - slice.row_chunks * owner / ranks), weight);
        }
    }
    cluster.sync();
    cut = s.cut, cut_mass = s.cut_mass;
    return !split;
}

// The row that a cluster takes.  A cut by mass alone can turn out flat and take
// three times as long as others: begun among the last, it would hold up the
// end.  So of every 32 rows, `step` apart, those come first.  (A lane a row: no
// barrier, one round trip.  512 rows of mixed settings 109 us for 113, 512 of
// one kind up to 3 us more.)
__device__ __forceinline__ unsigned ordered_row(unsigned at, unsigned step, unsigned rows, uint64_t width,
                                                const SampleSettings &set) {
    const unsigned lane = threadIdx.x & 31, i = at % step + step * lane;
    bool slow = false;
    if (i < rows) {
        const int k = set.top_k ? set.top_k[i] : 0;
        slow = set.top_p[i] < 1.0f && (k <= 0 || (uint64_t)k >= width);
    }
    const unsigned first = __ballot_sync(0xffffffffu, slow), before = (1u << lane) - 1;
    const unsigned place = slow ? __popc(first & before) : __popc(first) + __popc(~first & before);
    return at % step + step * (__ffs(__ballot_sync(0xffffffffu, place == at / step)) - 1);
}

template <bool kStaged>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(float *out, const float *logits, uint64_t width,
                                                                   int shift, uint32_t slice_chunks, unsigned step,
                                                                   SampleSettings set) {
    extern __shared__ __align__(16) unsigned char smem[];
    Shared &s = *reinterpret_cast<Shared *>(smem);
    float *staged = reinterpret_cast<float *>(smem + sizeof(Shared));  // 16-byte aligned, as Shared is
    u64 *chunk_mass = reinterpret_cast<u64 *>(staged + (kStaged ? slice_chunks * kChunk : 0));
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned ranks = cluster.num_blocks(), rank = cluster.block_rank();
    auto started = cluster.barrier_arrive();
    pdl_wait();
    pdl_trigger();
    unsigned at = blockIdx.x / ranks;
    if (step) at = ordered_row(at, step, gridDim.x / ranks, width, set);
    if (tid == 0) s.row = at;  // for the id's way out: read from here, it costs no register until then

    Slice<kStaged> slice;
    // Even shares (to a chunk), so that every CTA's maxima speak for its tokens.
    const uint64_t row_chunks = (width + kChunk - 1) / kChunk, chunk0 = row_chunks * rank / ranks;
    slice.first = chunk0 * kChunk;
    slice.chunks = (int)(row_chunks * (rank + 1) / ranks - chunk0);
    slice.most_chunks = (int)slice_chunks;
    slice.row_chunks = row_chunks;
    slice.index_scale = (float)kSortBins / (float)(row_chunks * kChunk);
    slice.size = (int)(min(width, slice.first + (uint64_t)slice.chunks * kChunk) - slice.first);
    const float *x = logits + at * width + slice.first;
    slice.x = kStaged ? staged : x;
    slice.aligned = (reinterpret_cast<uintptr_t>(x) & 15) == 0;

    // Largest logit; NaN and +infinity poison the row.
    float mine = -INFINITY;
    bool bad = false;
    auto look = [&](float v) {
        bad |= !(v < INFINITY);
        mine = fmaxf(mine, v);
    };
    const int whole = slice.aligned ? slice.size / 4 : 0;
    if constexpr (kStaged) {  // the whole slice in flight at once; a thread looks at what it loaded itself
        for (int i = tid; i < whole; i += kSampleThreads)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(sm100::smem_u32(staged + 4 * i)), "l"(x + 4 * i)
                         : "memory");
        for (int i = whole * 4 + tid; i < slice.size; i += kSampleThreads)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(sm100::smem_u32(staged + i)), "l"(x + i) : "memory");
    }
    // (While the loads are under way.)
    for (int i = tid; i < kPowers * kCopies; i += kSampleThreads) s.powers[i] = kPowerTable[i / kCopies];
    if (tid < 256) s.count[tid] = 0;
    if (tid < kSortBins) s.sort_count[0][tid] = s.sort_count[1][tid] = 0;
    if (tid == 0) s.listed = 0, s.full = 0;
    const float u = set.uniform[at], wanted_t = set.temperature[at];
    const float top_p = set.top_p ? set.top_p[at] : 1.0f, min_p = set.min_p ? set.min_p[at] : 0.0f;
    const bool valid = wanted_t >= 0.0f && wanted_t < INFINITY && !isnan(u) && !isnan(top_p) && !isnan(min_p);
    const float temperature = wanted_t == 0.0f ? 1.0f : fmaxf(wanted_t, 1e-38f);
    const int64_t top_k = wanted_t == 0.0f ? 1 : set.top_k ? set.top_k[at] : 0;
    Wanted want;
    want.by_count = top_k > 0 && (uint64_t)top_k < width;
    want.by_mass = top_p < 1.0f;
    want.count = (u64)top_k;
    want.p = fmaxf(top_p, 0.0f), want.u = u;
    Row row;
    row.inverse = 2.0f / temperature;
    row.rate = 1.4426950408889634074 / (double)temperature;
    row.unit = 1.5 * (double)(1ull << (52 - shift));
    want.least = (u64)ceil((double)fminf(fmaxf(min_p, 0.0f), 1.0f) * (double)(1ull << shift));
    if (kStaged) asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 8
    for (int i = tid; i < whole; i += kSampleThreads) {
        const float4 v = kStaged ? reinterpret_cast<const float4 *>(staged)[i] : __ldg(reinterpret_cast<const float4 *>(x) + i);
        look(v.x), look(v.y), look(v.z), look(v.w);
    }
#pragma unroll 8
    for (int i = whole * 4 + tid; i < slice.size; i += kSampleThreads) look(kStaged ? staged[i] : __ldg(x + i));
    if (kStaged)
        for (int i = slice.size + tid; i < slice.chunks * kChunk; i += kSampleThreads) staged[i] = -INFINITY;
    float top = warp_max(mine), low = mine == -INFINITY ? INFINITY : mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    if (lane == 0) s.part_top[warp] = top, s.part_low[warp] = low;
    bad = __syncthreads_or(bad);
    for (int w = 0; w < kSampleWarps; ++w) top = fmaxf(top, s.part_top[w]), low = fminf(low, s.part_low[w]);

    // With top-k: at least ceil(top_k / ranks) tokens of every CTA are at or
    // above its bound, so top_k of the row's are at or above the least bound.
    float bound = -INFINITY;
    if (valid && want.by_count && top_k <= kList)
        bound = top_k == 1 ? top : near_bound(s, mine, top, low, (int)((top_k + ranks - 1) / ranks), temperature);
    cluster.barrier_wait(std::move(started));  // every CTA's shared memory is there
    if (tid < ranks) {
        Shared *o = cluster.map_shared_rank(&s, tid);
        o->top[rank] = top;
        o->near[rank] = bound;
        o->bad[rank] = bad;
    }
    cluster.sync();
    row.top = -INFINITY;
    for (unsigned q = 0; q < ranks; ++q) {
        row.top = fmaxf(row.top, s.top[q]);
        bound = fminf(bound, s.near[q]);
        bad |= s.bad[q] != 0;
    }
    if (bad || row.top == -INFINITY || !valid) {
        if (rank == 0 && tid == 0) out[s.row] = __int_as_float(0x7fc00000);
        return;
    }
    row.half_top = 0.5f * row.top;
    row.floor = fmaxf(row.top - 34.0f * temperature, -FLT_MAX);  // -infinity stays below it

    u64 cut = 0, mass = 0;
    bool summed = false;
    if (want.by_count || want.by_mass || min_p > 0.0f) {
        // min_p alone keeps (max - l) / T <= -log(min_p): with a margin far
        // above F32's rounding, the weights decide.
        if (want.by_count && top_k == 1) bound = row.top;
        else if (want.by_mass && !want.by_count) bound = row.top - kNear * temperature;
        else if (!want.by_count) bound = row.top + fminf(logf(min_p), 0.0f) * 1.001f * temperature - 1e-3f * temperature;
        if (sample_near(cluster, s, slice, row, want, bound, mine, out, mass)) return;
#pragma unroll 1
        for (int by_mass = want.by_count ? 0 : 1; by_mass <= (int)want.by_mass; ++by_mass)
            summed = find_cut(cluster, s, slice, row, by_mass, !by_mass ? want.count : mass ? mass_limit(want.p, mass) : 0,
                              want.p, want.least, shift, chunk_mass, cut, mass);
    }

    // Kept mass of each chunk, of the CTA, of the row.
    const float least_value = cut ? key_value((uint32_t)(cut >> 32)) : -INFINITY;
    auto kept = [&](float v, uint64_t index) -> u64 {
        if (v < least_value || (v == least_value && order_of(v, index) < cut)) return 0;
        const u64 w = weight_of(v, row, s);
        return w >= want.least ? w : 0;
    };
    const bool all = cut == 0 && want.least == 0;
    u64 kept_mass = 0;
    if (summed) {
        for (int c = lane == 0 ? warp : slice.chunks; c < slice.chunks; c += kSampleWarps) kept_mass += chunk_mass[c];
    } else {
        slice.template each<2>([&](int c, const float4 &v) {
            u64 sum = 0;
            if (all) {
                sum = warp_sum48(weight_bits(v.x, row, s) + weight_bits(v.y, row, s) + weight_bits(v.z, row, s) +
                                 weight_bits(v.w, row, s) - 4 * (u64)__double_as_longlong(row.unit));
            } else if (__any_sync(0xffffffffu, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= least_value)) {
                const uint64_t i = slice.first + c * kChunk + lane * 4;
                sum = warp_sum48(kept(v.x, i) + kept(v.y, i + 1) + kept(v.z, i + 2) + kept(v.w, i + 3));
            }
            if (lane == 0) chunk_mass[c] = sum;
            kept_mass += sum;
        });
    }
    __syncthreads();
    if (lane == 0) s.part[warp] = kept_mass;
    __syncthreads();
    if (tid < ranks) {
        u64 sum = 0;
        for (int w = 0; w < kSampleWarps; ++w) sum += s.part[w];
        cluster.map_shared_rank(&s, tid)->kept[rank] = sum;
    }
    cluster.sync();
    u64 total = 0, ahead = 0;
    for (unsigned q = 0; q < ranks; ++q) {
        if (q < rank) ahead += s.kept[q];
        total += s.kept[q];
    }
    u64 target = mass_target(u, total);
    if (target < ahead || target >= ahead + s.kept[rank] || warp != 0) return;

    // The CTA, then the chunk, then the token in which the target falls.
    for (int c0 = 0; c0 < slice.chunks; c0 += 32) {
        const u64 m = c0 + lane < slice.chunks ? chunk_mass[c0 + lane] : 0;
        const u64 upto = warp_upto(m);
        const unsigned past = __ballot_sync(0xffffffffu, ahead + upto > target);
        if (!past) {
            ahead += __shfl_sync(0xffffffffu, upto, 31);
            continue;
        }
        const int l = __ffs(past) - 1, c = c0 + l;
        ahead += __shfl_sync(0xffffffffu, upto - m, l);
        const float4 v = slice.four(c);
        const uint64_t i = slice.first + c * kChunk + lane * 4;
        const u64 w[4] = {kept(v.x, i), kept(v.y, i + 1), kept(v.z, i + 2), kept(v.w, i + 3)};
        const u64 sum = w[0] + w[1] + w[2] + w[3];
        const u64 run = ahead + warp_upto(sum) - sum;
        if (run <= target && target < run + sum) {
            target -= run;
            const int j = target < w[0] ? 0 : target < w[0] + w[1] ? 1 : target < w[0] + w[1] + w[2] ? 2 : 3;
            out[s.row] = (float)(i + j);
        }
        return;
    }
}

template <bool kStaged>
int32_t run(float *out, const float *logits, uint64_t rows, uint64_t width, int shift, unsigned ranks, uint32_t chunks,
            const SampleSettings &set, cudaStream_t stream) {
    // In order of cost only where some clusters wait for others to end.
    const unsigned step = set.top_p && rows * ranks > 2 * (uint64_t)sm_count() ? (unsigned)((rows + 31) / 32) : 0;
    const size_t smem = sizeof(Shared) + chunks * sizeof(u64) + (kStaged ? (size_t)chunks * kChunk * 4 : 0);
    static std::atomic<uint64_t> ready{0};
    if (int32_t st = allow_smem(sample_kernel<kStaged>, kMostSmem, ready)) return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * ranks));
    cfg.blockDim = dim3(kSampleThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return launch_config(cfg, "sample_kernel", sample_kernel<kStaged>, out, logits, width, shift, chunks, step, set);
}

}  // namespace

int32_t sample(float *out, const float *logits, uint64_t rows, uint64_t width, const SampleSettings &set,
               cudaStream_t stream) {
    if (!rows) return MF_OK;
    int bits = 0;
    while ((1ull << bits) < width) ++bits;
    const int shift = std::min(46, 62 - bits);
    // CTAs per row: slices of 16384 tokens or fewer (64 KB of shared memory:
    // two CTAs share an SM, so one's loads meet the other's arithmetic), and
    // more of them while they fit the SMs' two at once and keep 1024 tokens.
    // 65536 tokens: 37 rows 26 us with 8 CTAs, 32 with 4; 64 rows 34 and 35;
    // 512 rows 166 and 113.  8000 tokens, 512 rows: 40 us with 1, 50 with 2.
    unsigned ranks = 1;
    while (ranks < kMaxCluster && (width > 16384ull * ranks || (rows * ranks <= (uint64_t)sm_count() &&
                                                                width >= 2048ull * ranks)))
        ranks *= 2;
    const uint64_t chunks = ((width + kChunk - 1) / kChunk + ranks - 1) / ranks;
    return chunks * kChunk <= kStageFloats
               ? run<true>(out, logits, rows, width, shift, ranks, (uint32_t)chunks, set, stream)
               : run<false>(out, logits, rows, width, shift, ranks, (uint32_t)chunks, set, stream);
}

}  // namespace mf
