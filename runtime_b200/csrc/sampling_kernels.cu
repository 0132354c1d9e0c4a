// Sampling a token id per row of logits.
//
// With w_i = exp((l_i - max) / T) and the order "larger logit first, equal
// logits by index", a row keeps the first top_k tokens (their mass M), of
// those each whose mass before it is below top_p * M, of those each with
// w_i >= min_p; the id is the first kept token, in index order, whose running
// kept mass exceeds u times the kept mass.  Every kept set is a prefix of the
// same order, so a row is described by one threshold logit, the number of
// tokens equal to it that stay (the lowest indexes), and the min_p bound.
//
// Weights are integers, round(w * 2^shift) with 2^shift * width < 2^62: sums
// are exact in any order, so a result does not depend on how the row was
// split, and a running mass near its border is not moved by rounding (32-bit
// sums over 65536 tokens would move borders by 1e-3 of a token's weight).
#include <cuda_runtime.h>

#include "mf_common.cuh"
#include "packed_kernels.h"

namespace mf {

namespace {

constexpr int kSampleThreads = 1024;
constexpr int kSampleWarps = kSampleThreads / 32;

// Logits as unsigned integers of the same order.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v == 0.0f ? 0.0f : v);  // -0 equals +0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct SampleRow {
    float top;       // largest logit
    double inverse;  // 1 / temperature
    double unit;     // 2^shift
};

__device__ __forceinline__ unsigned long long sample_weight(float v, const SampleRow &r) {
    return (unsigned long long)__double2ll_rn(exp(((double)v - (double)r.top) * r.inverse) * r.unit);
}

__device__ __forceinline__ unsigned long long block_sum(unsigned long long v, unsigned long long *part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < kSampleWarps; ++w) v += part[w];
    return v;
}

// Sum of the values of the threads before this one.
__device__ __forceinline__ unsigned long long block_before(unsigned long long v, unsigned long long *part) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long sum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long t = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += t;
    }
    __syncthreads();
    if (lane == 31) part[warp] = sum;
    __syncthreads();
    unsigned long long before = sum - v;
    for (int w = 0; w < warp; ++w) before += part[w];
    return before;
}

// One CTA per row; every pass reads the row again.
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(float *out, const float *logits, uint64_t width,
                                                                int shift, SampleSettings set) {
    __shared__ unsigned long long s_part[kSampleWarps], s_mass[256];
    __shared__ unsigned s_count[256];
    __shared__ float s_top[kSampleWarps];
    __shared__ uint32_t s_prefix;
    __shared__ unsigned long long s_above;
    __shared__ unsigned s_id;
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint64_t row = blockIdx.x;
    const float *x = logits + row * width;
    const float nan = __int_as_float(0x7fc00000);

    // Largest logit; NaN and +infinity poison the row.
    float top = -INFINITY;
    bool bad = false;
    for (uint64_t i = tid; i < width; i += kSampleThreads) {
        const float v = x[i];
        bad |= !(v < INFINITY);
        top = fmaxf(top, v);
    }
    top = warp_max(top);
    if (lane == 0) s_top[warp] = top;
    bad = __syncthreads_or(bad);
    for (int w = 0; w < kSampleWarps; ++w) top = fmaxf(top, s_top[w]);
    const float temperature = set.temperature[row], u = set.uniform[row];
    const float top_p = set.top_p ? set.top_p[row] : 1.0f, min_p = set.min_p ? set.min_p[row] : 0.0f;
    int64_t top_k = set.top_k ? set.top_k[row] : 0;
    if (bad || top == -INFINITY || !(temperature >= 0.0f && temperature < INFINITY) || isnan(u) || isnan(top_p) ||
        isnan(min_p)) {
        if (tid == 0) out[row] = nan;
        return;
    }
    if (temperature == 0.0f) top_k = 1;
    SampleRow r;
    r.top = top;
    r.inverse = temperature == 0.0f ? 1.0 : 1.0 / (double)temperature;
    r.unit = (double)(1ull << shift);

    // The threshold: tokens above `key` stay, and `ties` of those equal to it.
    uint32_t key = 0;
    unsigned long long ties = ~0ull;
    for (int filter = 0; filter < 2; ++filter) {
        const bool by_mass = filter == 1;
        if (by_mass ? !(top_p < 1.0f) : !(top_k > 0 && (uint64_t)top_k < width)) continue;
        unsigned long long limit;
        if (by_mass) {
            unsigned long long sum = 0, equal = 0, one = 0;
            for (uint64_t i = tid; i < width; i += kSampleThreads) {
                const uint32_t o = order_key(x[i]);
                if (o > key) sum += sample_weight(x[i], r);
                if (o == key) one = sample_weight(x[i], r), ++equal;
            }
            const unsigned long long n = block_sum(equal, s_part);
            const unsigned long long stay = min(n, ties);
            // `one` is the same for every token of the key.
            unsigned long long most = one;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
            __syncthreads();
            if (lane == 0) s_part[warp] = most;
            __syncthreads();
            for (int w = 0; w < kSampleWarps; ++w) most = max(most, s_part[w]);
            __syncthreads();
            const unsigned long long mass = block_sum(sum, s_part) + stay * most;
            limit = (unsigned long long)ceil((double)fmaxf(top_p, 0.0f) * (double)mass);
            if (limit == 0) limit = 1;  // the first token always stays
        } else {
            limit = (unsigned long long)top_k;
        }
        // Digit by digit from the top: the bin in which the running count or
        // mass reaches the limit.
        uint32_t prefix = 0, mask = 0;
        unsigned long long above = 0;
        for (int d = 24; d >= 0; d -= 8) {
            for (int i = tid; i < 256; i += kSampleThreads) s_mass[i] = 0, s_count[i] = 0;
            __syncthreads();
            for (uint64_t i = tid; i < width; i += kSampleThreads) {
                const uint32_t o = order_key(x[i]);
                if ((o & mask) != prefix) continue;
                if (by_mass) atomicAdd(&s_mass[o >> d & 255], sample_weight(x[i], r));
                atomicAdd(&s_count[o >> d & 255], 1u);
            }
            __syncthreads();
            if (tid == 0) {
                int b = 255, found = -1;
                unsigned long long run = above, at = above;
                for (; b >= 0; --b) {
                    if (!s_count[b]) continue;
                    if (run >= limit) break;
                    found = b, at = run;
                    run += by_mass ? s_mass[b] : s_count[b];
                }
                s_prefix = prefix | (uint32_t)found << d;
                s_above = at;
            }
            __syncthreads();
            prefix = s_prefix;
            above = s_above;
            mask |= 255u << d;
        }
        // Tokens of this key that stay: those with fewer than `limit` before.
        unsigned long long stay;
        if (by_mass) {
            const uint32_t b = prefix & 0x80000000u ? prefix & 0x7fffffffu : ~prefix;
            const unsigned long long w = sample_weight(__uint_as_float(b), r);
            stay = w ? (limit - above + w - 1) / w : ~0ull;
        } else {
            stay = limit - above;
        }
        if (prefix > key || filter == 0) {
            key = prefix;
            ties = stay;
        } else if (prefix == key) {
            ties = min(ties, stay);
        }
        __syncthreads();
    }

    // Each thread a run of consecutive tokens: kept mass before it, then the
    // token in which the target falls.
    const uint64_t span = (width + kSampleThreads - 1) / kSampleThreads;
    const uint64_t begin = min(width, tid * span), end = min(width, begin + span);
    unsigned long long equal = 0;
    for (uint64_t i = begin; i < end; ++i) equal += order_key(x[i]) == key;
    const unsigned long long rank = block_before(equal, s_part);
    const double floor_p = fminf(fmaxf(min_p, 0.0f), 1.0f) * r.unit;
    auto kept = [&](uint64_t i, unsigned long long &at) -> unsigned long long {
        const uint32_t o = order_key(x[i]);
        if (o < key || (o == key && at++ >= ties)) return 0;
        const unsigned long long w = sample_weight(x[i], r);
        return (double)w >= floor_p ? w : 0;
    };
    unsigned long long mine = 0, at = rank;
    for (uint64_t i = begin; i < end; ++i) mine += kept(i, at);
    __syncthreads();
    const unsigned long long mass = block_sum(mine, s_part);
    unsigned long long run = block_before(mine, s_part);
    unsigned long long target = u > 0.0f ? (unsigned long long)floor((double)fminf(u, 1.0f) * (double)mass) : 0;
    if (target >= mass) target = mass - 1;
    if (tid == 0) s_id = 0;
    __syncthreads();
    if (mine && run <= target && target < run + mine) {
        at = rank;
        for (uint64_t i = begin; i < end; ++i) {
            const unsigned long long w = kept(i, at);
            if (w && target < run + w) {
                s_id = (unsigned)i;
                break;
            }
            run += w;
        }
    }
    __syncthreads();
    if (tid == 0) out[row] = (float)s_id;
}

}  // namespace

int32_t sample(float *out, const float *logits, uint64_t rows, uint64_t width, const SampleSettings &set,
               cudaStream_t stream) {
    if (!rows) return MF_OK;
    int bits = 0;
    while ((1ull << bits) < width) ++bits;
    return launch(sample_kernel, dim3((unsigned)rows), dim3(kSampleThreads), 0, stream, "sample_kernel", out, logits,
                  width, 62 - bits, set);
}

}  // namespace mf
