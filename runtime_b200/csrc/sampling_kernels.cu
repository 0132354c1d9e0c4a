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
// once, and shares maxima, histograms and masses through distributed shared
// memory.  A cut is found from a histogram of (max - l) / T (1024 bins of
// 1/31 up to the weight that rounds to 0), in which the bin that the cut
// falls in is known at once; that bin's tokens, a few dozen, are gathered in
// one CTA and ranked directly.  A bin with more than kList tokens (equal
// logits) is first split by the bits of (logit, index).
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "mf_common.cuh"
#include "packed_kernels.h"

namespace mf {

namespace {

namespace cg = cooperative_groups;

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kChunk = 128;              // tokens of a warp's step: four a lane
constexpr int kBins = 1024;
constexpr float kBinScale = 31.0f;
constexpr int kList = 512;
constexpr int kMaxCluster = 8;
constexpr uint64_t kStageFloats = 48 * 1024;  // of a CTA at most

using u64 = unsigned long long;

// Logits as unsigned integers of the same order.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v == 0.0f ? 0.0f : v);  // -0 equals +0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// A token's place in a row's order: larger is earlier.
__device__ __forceinline__ u64 order_of(float v, uint64_t index) {
    return (u64)order_key(v) << 32 | (0xffffffffu - (uint32_t)index);
}

struct Row {
    float top;      // largest logit
    float inverse;  // 1 / T in F32, for the bins
    double rate;    // log2(e) / T
    double unit;    // 1.5 * 2^(52 - shift): adding it rounds to steps of 2^-shift
};

struct Listed {
    u64 order, weight;
};

// What the CTAs of a cluster tell one another.
struct alignas(16) Shared {
    double powers[32 * 16];  // 2^(j / 32), 16 copies: a half-warp's reads hit 16 banks
    u64 mass[kBins];
    unsigned count[kBins];
    Listed list[kList];
    unsigned listed;
    float top[kMaxCluster];
    int bad[kMaxCluster];
    u64 kept[kMaxCluster];
    u64 cut, cut_mass;  // the last token that stays and the mass up to it
    // Within the CTA.
    u64 part[kSampleWarps];
    unsigned part_count[kSampleWarps];
    float part_top[kSampleWarps];
    unsigned cross_bin, cross_count;
    u64 cross_before, cross_mass, total_mass;
    unsigned last_rank;
};

// round(exp((v - top) / T) * 2^shift).  2^y for y = n + j / 32 + r, |r| <= 1/64:
// the power of the fraction j from a table, the rest by its Taylor series to
// r^4 (next term 2^-39 of the weight), n into the exponent.
__device__ __forceinline__ u64 weight_of(float v, const Row &r, const Shared &s) {
    if (!((r.top - v) * r.inverse < 34.0f)) return 0;  // below half a step
    constexpr double kMagic = 6755399441055744.0 / 32;  // 1.5 * 2^52 / 32: sums round to 1/32
    const double d = (double)v - (double)r.top;
    const double t = fma(d, r.rate, kMagic);
    const int k = __double2loint(t);
    const double f = fma(d, r.rate, kMagic - t);
    constexpr double kLn2 = 0.69314718055994530942;
    double p = fma(f, kLn2 * kLn2 * kLn2 * kLn2 / 24, kLn2 * kLn2 * kLn2 / 6);
    p = fma(f, p, kLn2 * kLn2 / 2);
    p = fma(f, p, kLn2);
    p = fma(f, p, 1.0);
    p *= s.powers[(k & 31) * 16 + (threadIdx.x & 15)];
    p = __hiloint2double(__double2hiint(p) + (k >> 5) * (1 << 20), __double2loint(p));
    return (u64)(__double_as_longlong(p + r.unit) - __double_as_longlong(r.unit));
}

__device__ __forceinline__ int bin_of(float v, const Row &r) {
    return (int)fminf((r.top - v) * r.inverse * kBinScale, (float)(kBins - 1));
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

// A CTA's share of a row: `size` tokens from index `first`, in shared memory
// or (rows too wide for a cluster) in global memory.
template <bool kStaged>
struct Slice {
    const float *x;
    uint64_t first;
    int size, chunks;

    // Tokens 4 lane .. 4 lane + 3 of a chunk; -infinity past the end.
    __device__ __forceinline__ float4 four(int chunk) const {
        const int at = chunk * kChunk + (threadIdx.x & 31) * 4;
        if constexpr (kStaged) return *reinterpret_cast<const float4 *>(x + at);
        float4 v;
        v.x = at + 0 < size ? x[at + 0] : -INFINITY;
        v.y = at + 1 < size ? x[at + 1] : -INFINITY;
        v.z = at + 2 < size ? x[at + 2] : -INFINITY;
        v.w = at + 3 < size ? x[at + 3] : -INFINITY;
        return v;
    }
};

// The place of the cut in a row's order: the last token with fewer than
// `limit` tokens (or less than `limit` mass) before it, 0 where every token
// with weight stays; and the mass of what stays.  With share >= 0 the limit is
// that share of the row's mass.  `ready`: s.mass and s.count still hold the
// first histogram; returns whether they do afterwards.
template <bool kStaged>
__device__ bool find_cut(cg::cluster_group &cluster, Shared &s, const Slice<kStaged> &slice, const Row &row, bool by_mass,
                         double share, u64 limit, bool ready, u64 &cut, u64 &cut_mass) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned ranks = cluster.num_blocks(), rank = cluster.block_rank();
    u64 before = 0, mass_before = 0;  // tokens and mass ahead of the bin
    unsigned bin0 = 0;
    u64 prefix = 0;
    for (int round = 0;; ++round) {
        const int digit = 64 - 8 * round;  // rounds after the first: 8 bits of the order, from the top
        const int bins = round ? 256 : kBins;
        if (round || !ready) {
            for (int i = tid; i < bins; i += kSampleThreads) s.mass[i] = 0, s.count[i] = 0;
            __syncthreads();
            for (int c = warp; c < slice.chunks; c += kSampleWarps) {
                const float4 v4 = slice.four(c);
                const float v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    unsigned b = bin_of(v[j], row);
                    if (round) {
                        if (b != bin0) continue;
                        const u64 o = order_of(v[j], slice.first + c * kChunk + lane * 4 + j);
                        if (round > 1 && o >> (digit + 8) != prefix) continue;
                        b = 255 - (unsigned)(o >> digit & 255);
                    }
                    const u64 w = weight_of(v[j], row, s);
                    if (!w) continue;
                    atomicAdd(&s.count[b], 1u);
                    atomicAdd(&s.mass[b], w);
                }
            }
            cluster.sync();
            // Each rank adds up its part of the bins and hands the sums to all.
            if (ranks > 1) {
                const int share_bins = bins / (int)ranks;
                for (int i = tid; i < share_bins; i += kSampleThreads) {
                    const int b = rank * share_bins + i;
                    u64 m = 0;
                    unsigned n = 0;
                    for (unsigned q = 0; q < ranks; ++q) {
                        Shared *o = cluster.map_shared_rank(&s, q);
                        m += o->mass[b];
                        n += o->count[b];
                    }
                    for (unsigned q = 0; q < ranks; ++q) {
                        Shared *o = cluster.map_shared_rank(&s, q);
                        o->mass[b] = m;
                        o->count[b] = n;
                    }
                }
                cluster.sync();
            }
        }
        // Running sums over the bins, two a thread.
        const int b0 = tid * 2;
        u64 m0 = 0, m1 = 0;
        unsigned n0 = 0, n1 = 0;
        if (b0 < bins) m0 = s.mass[b0], m1 = s.mass[b0 + 1], n0 = s.count[b0], n1 = s.count[b0 + 1];
        const u64 mu = warp_upto(m0 + m1);
        const unsigned nu = (unsigned)warp_upto(n0 + n1);
        if (lane == 31) s.part[warp] = mu, s.part_count[warp] = nu;
        if (tid == 0) s.cross_count = 0;
        __syncthreads();
        u64 mb = mass_before + mu - m0 - m1, nb = before + nu - n0 - n1, all = mass_before;
        for (int w = 0; w < kSampleWarps; ++w) {
            if (w < warp) mb += s.part[w], nb += s.part_count[w];
            all += s.part[w];
        }
        if (by_mass && share >= 0.0) {  // the first round of a cut by mass of the whole row
            limit = max((u64)ceil(share * (double)all), 1ull);
            share = -1.0;
        }
        // The last bin with tokens and fewer than the limit before it.
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const unsigned n = i ? n1 : n0;
            const u64 m = i ? m1 : m0, ahead = by_mass ? mb : nb;
            if (n && ahead < limit && ahead + (by_mass ? m : n) >= limit)
                s.cross_bin = b0 + i, s.cross_count = n, s.cross_before = nb, s.cross_mass = mb;
            mb += m, nb += n;
        }
        __syncthreads();
        const unsigned count = s.cross_count, bin = s.cross_bin;
        if (count == 0) {  // the limit lies behind the last token
            cut = 0, cut_mass = all;
            __syncthreads();
            return true;
        }
        before = s.cross_before, mass_before = s.cross_mass;
        if (round == 0) bin0 = bin;
        else prefix = prefix << 8 | (255 - bin);
        if (count <= kList || round == 8) {
            // The bin's tokens, gathered in rank 0.
            Shared *lead = cluster.map_shared_rank(&s, 0);
            if (rank == 0 && tid == 0) s.listed = 0, s.last_rank = 0;
            cluster.sync();
            for (int c = warp; c < slice.chunks; c += kSampleWarps) {
                const float4 v4 = slice.four(c);
                const float v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (bin_of(v[j], row) != (int)bin0) continue;
                    const u64 o = order_of(v[j], slice.first + c * kChunk + lane * 4 + j);
                    if (round && o >> digit != prefix) continue;
                    const u64 w = weight_of(v[j], row, s);
                    if (!w) continue;
                    const unsigned at = atomicAdd(&lead->listed, 1u);
                    if (at < kList) lead->list[at] = {o, w};
                }
            }
            cluster.sync();
            if (rank == 0) {
                const unsigned n = min(s.listed, (unsigned)kList);
                u64 mine = 0, mine_mass = 0;
                unsigned ahead = 0;
                if (tid < n) {
                    const Listed e = s.list[tid];
                    u64 mass = 0;
                    for (unsigned i = 0; i < n; ++i) {
                        const Listed q = s.list[i];
                        if (q.order > e.order) ++ahead, mass += q.weight;
                    }
                    if ((by_mass ? mass_before + mass : before + ahead) < limit)
                        mine = e.order, mine_mass = mass_before + mass + e.weight;
                }
                if (mine) atomicMax(&s.last_rank, ahead + 1);
                __syncthreads();
                if (mine && ahead + 1 == s.last_rank)
                    for (unsigned q = 0; q < ranks; ++q) {
                        Shared *o = cluster.map_shared_rank(&s, q);
                        o->cut = mine;
                        o->cut_mass = mine_mass;
                    }
            }
            cluster.sync();
            cut = s.cut, cut_mass = s.cut_mass;
            __syncthreads();
            return round == 0;
        }
    }
}

template <bool kStaged>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(float *out, const float *logits, uint64_t width,
                                                                int shift, uint32_t slice_chunks, SampleSettings set) {
    extern __shared__ __align__(16) unsigned char smem[];
    Shared &s = *reinterpret_cast<Shared *>(smem);
    float *staged = reinterpret_cast<float *>(smem + sizeof(Shared));  // 16-byte aligned, as Shared is
    u64 *chunk_mass = reinterpret_cast<u64 *>(staged + (kStaged ? slice_chunks * kChunk : 0));
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned ranks = cluster.num_blocks(), rank = cluster.block_rank();
    const uint64_t at = blockIdx.x / ranks;
    auto started = cluster.barrier_arrive();
    // The table: 32 powers by the library's exponential, 16 copies.
    s.powers[tid] = exp2((double)(tid / 16) / 32);
    pdl_wait();
    pdl_trigger();

    Slice<kStaged> slice;
    slice.first = min(width, (uint64_t)rank * slice_chunks * kChunk);
    slice.size = (int)min(width - slice.first, (uint64_t)slice_chunks * kChunk);
    slice.chunks = (slice.size + kChunk - 1) / kChunk;
    const float *x = logits + at * width + slice.first;
    slice.x = kStaged ? staged : x;

    // Largest logit; NaN and +infinity poison the row.
    float top = -INFINITY;
    bool bad = false;
    auto look = [&](float v) {
        bad |= !(v < INFINITY);
        top = fmaxf(top, v);
    };
    if (kStaged) {
        const int whole = (reinterpret_cast<uintptr_t>(x) & 15) ? 0 : slice.size / 4;
#pragma unroll 8
        for (int i = tid; i < whole; i += kSampleThreads) {
            const float4 v = __ldcs(reinterpret_cast<const float4 *>(x) + i);
            reinterpret_cast<float4 *>(staged)[i] = v;
            look(v.x), look(v.y), look(v.z), look(v.w);
        }
#pragma unroll 8
        for (int i = whole * 4 + tid; i < slice.size; i += kSampleThreads) {
            const float v = __ldcs(x + i);
            staged[i] = v;
            look(v);
        }
        for (int i = slice.size + tid; i < slice.chunks * kChunk; i += kSampleThreads) staged[i] = -INFINITY;
    } else {
#pragma unroll 4
        for (int i = tid; i < slice.size; i += kSampleThreads) look(x[i]);
    }
    top = warp_max(top);
    if (lane == 0) s.part_top[warp] = top;
    bad = __syncthreads_or(bad);
    cluster.barrier_wait(std::move(started));  // every CTA's shared memory is there
    if (tid < ranks) {
        for (int w = 0; w < kSampleWarps; ++w) top = fmaxf(top, s.part_top[w]);
        Shared *o = cluster.map_shared_rank(&s, tid);
        o->top[rank] = top;
        o->bad[rank] = bad;
    }
    cluster.sync();
    Row row;
    row.top = -INFINITY;
    for (unsigned q = 0; q < ranks; ++q) row.top = fmaxf(row.top, s.top[q]), bad |= s.bad[q] != 0;

    const float temperature = set.temperature[at], u = set.uniform[at];
    const float top_p = set.top_p ? set.top_p[at] : 1.0f, min_p = set.min_p ? set.min_p[at] : 0.0f;
    int64_t top_k = set.top_k ? set.top_k[at] : 0;
    if (bad || row.top == -INFINITY || !(temperature >= 0.0f && temperature < INFINITY) || isnan(u) || isnan(top_p) ||
        isnan(min_p)) {
        if (rank == 0 && tid == 0) out[at] = __int_as_float(0x7fc00000);
        return;
    }
    if (temperature == 0.0f) top_k = 1;
    const double inverse = temperature == 0.0f ? 1.0 : fmin(1.0 / (double)temperature, 1e38);
    row.inverse = (float)inverse;
    row.rate = inverse * 1.4426950408889634074;
    row.unit = 1.5 * (double)(1ull << (52 - shift));

    u64 cut = 0, mass = 0;
    const bool by_count = top_k > 0 && (uint64_t)top_k < width;
    bool ready = false;
    if (by_count) ready = find_cut(cluster, s, slice, row, false, -1.0, (u64)top_k, false, cut, mass);
    if (top_p < 1.0f) {
        const float p = fmaxf(top_p, 0.0f);
        u64 unused;
        find_cut(cluster, s, slice, row, true, by_count ? -1.0 : (double)p,
                 by_count ? max((u64)ceil((double)p * (double)mass), 1ull) : 0, ready, cut, unused);
    }
    const u64 least = (u64)ceil((double)fminf(fmaxf(min_p, 0.0f), 1.0f) * (double)(1ull << shift));

    // Kept mass of each chunk, of the CTA, of the row.
    auto kept = [&](float v, uint64_t index) -> u64 {
        if (cut && order_of(v, index) < cut) return 0;
        const u64 w = weight_of(v, row, s);
        return w >= least ? w : 0;
    };
    u64 mine = 0;
#pragma unroll 2
    for (int c = warp; c < slice.chunks; c += kSampleWarps) {
        const float4 v = slice.four(c);
        const uint64_t i = slice.first + c * kChunk + lane * 4;
        const u64 sum = warp_sum48(kept(v.x, i) + kept(v.y, i + 1) + kept(v.z, i + 2) + kept(v.w, i + 3));
        if (lane == 0) chunk_mass[c] = sum;
        mine += sum;
    }
    if (lane == 0) s.part[warp] = mine;
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
    u64 target = u > 0.0f ? (u64)floor((double)fminf(u, 1.0f) * (double)total) : 0;
    if (target >= total) target = total - 1;
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
            out[at] = (float)(i + j);
        }
        return;
    }
}

template <bool kStaged>
int32_t run(float *out, const float *logits, uint64_t rows, uint64_t width, int shift, unsigned ranks, uint32_t chunks,
            const SampleSettings &set, cudaStream_t stream) {
    const size_t smem = sizeof(Shared) + chunks * sizeof(u64) + (kStaged ? (size_t)chunks * kChunk * 4 : 0);
    MF_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<kStaged>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
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
    return launch_config(cfg, "sample_kernel", sample_kernel<kStaged>, out, logits, width, shift, chunks, set);
}

}  // namespace

int32_t sample(float *out, const float *logits, uint64_t rows, uint64_t width, const SampleSettings &set,
               cudaStream_t stream) {
    if (!rows) return MF_OK;
    int bits = 0;
    while ((1ull << bits) < width) ++bits;
    const int shift = std::min(46, 62 - bits);
    // CTAs per row: slices of 16384 tokens or fewer (64 KB: three CTAs share
    // an SM, so one loads while another computes); more of them, down to 2048
    // tokens, while rows leave SMs idle.
    unsigned ranks = 1;
    while (ranks < kMaxCluster && (width > 16384ull * ranks || (rows * ranks * 2 <= (uint64_t)sm_count() && width >= 4096ull * ranks)))
        ranks *= 2;
    const uint64_t chunks = ((width + kChunk - 1) / kChunk + ranks - 1) / ranks;
    return chunks * kChunk <= kStageFloats ? run<true>(out, logits, rows, width, shift, ranks, (uint32_t)chunks, set, stream)
                                           : run<false>(out, logits, rows, width, shift, ranks, (uint32_t)chunks, set, stream);
}

}  // namespace mf
