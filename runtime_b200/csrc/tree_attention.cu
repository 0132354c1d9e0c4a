// Attention of several rows per sequence over a paged cache: drafted trees,
// and prompts that go on in chunks (layout: paged_kernels.cu; trees:
// tree_kernels.cu).
//
// Row r of a sequence's n rows is its token L - n + r.  It sees the tokens
// before the rows, its ancestors and itself:
// out = sum_j p_j v_j / sum_j p_j, p_j = exp(q . k_j / sqrt(D) - m), one pass
// over the tokens with the running maximum m and sum (held in F32).
//
// Tiles.  Rows and the query heads of a KV head, 128 of them at most, are the
// rows of tcgen05 products: S = Q K^T and O = P V over tiles of 64 tokens, Q
// and the tiles of K and V in shared memory, S, P and O in tensor memory.  V
// lies there as in its page, [token][dimension], and is read transposed.  A
// softmax thread owns a row, so maxima and sums need no exchange.  With 64 or
// 32 rows (or fewer) there are two or four copies of them, each of which takes
// its share of a tile's tokens (its P is zero for the others'), so that the
// softmax takes a half or a quarter of the time; copies are joined at the end.
//
// Roles.  Four softmax warps for each of two tiles in turn (one where D is 128:
// its 128 sums fill the registers), each with sums of its own, joined at the
// end; two warps that load tiles; one that issues the products.
//
// F32 accuracy.  Q and P are held in parts of the pages' type whose products
// the tensor core sums in F32, low parts first: three of BF16 (8 bits each:
// all 24), two of F16 (22 bits; q scaled to [2^14, 2^15) by a power of two per
// row and p by 2^14, so that low parts stay above F16's smallest step).  F32
// pages are split into three BF16 parts too, and the six products of order up
// to 2 are summed.  Every tile's O starts from zero and is added by FMA, since
// the tensor core cuts its sums where an FMA rounds.
//
// Split.  The work is a list of tiles, item by item (a block of rows, a KV
// head), built on the device; CTAs take equal runs of it.  A run that ends
// inside an item leaves its maxima, sums and weighted values in the workspace;
// the last CTA to arrive joins them in one order.  Tiles are taken from the
// last to the first: a row's ancestors are met on the way up the tree.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "mf_common.cuh"
#include "packed_kernels.h"
#include "paged_common.cuh"
#include "tc_sm100.cuh"

namespace mf {

// Set (bit 0) by a tree attention whose pipeline wait timed out.
__device__ unsigned int g_tree_fault = 0;

namespace {

using namespace sm100;

constexpr int kTgRows = 128;   // rows of a block: the products' M
constexpr int kTgLoaders = 2;  // warps (11 and 7 in all leave 168 and 255 registers to a thread)

struct TreeGqaArgs {
    float *out;
    const float *q;
    const void *keys, *values;
    PagedTable pt;
    uint64_t tokens;
    const int32_t *lengths, *offsets, *parents;
    uint32_t q_heads, kv_heads, head_dim;
    uint32_t head_blocks, block_heads, block_nodes;  // of a KV head's query heads; heads and rows of a block at most
    uint32_t page_magic, page_shift;                 // as in paged_attention.cu
    uint32_t aligned;                                // pages of 16 tokens or a multiple, rows without padding
    unsigned *arrived;                               // [CTAs], zero between calls
    float *partial;                                  // [2 * CTAs][kPart]
};

template <typename T, int D>
struct TreeShape {
    static constexpr bool kF32 = sizeof(T) == 4;
    static constexpr bool kHalf = std::is_same<T, __half>::value;
    static constexpr int kQParts = kHalf ? 2 : 3;  // of Q and P
    static constexpr int kKvParts = kF32 ? 3 : 1;
    static constexpr int kPairs = kF32 ? 6 : kQParts;
    static constexpr int kTile = kF32 && D == 128 ? 32 : 64;  // (F32's parts of 64 tokens of 128 do not fit)
    static constexpr int kGroups = D == 64 ? 2 : 1;           // groups of softmax warps
    static constexpr int kSoftmax = 4 * kGroups;              // warps
    static constexpr int kThreads = 32 * (kSoftmax + kTgLoaders + 1);
    static constexpr int kCopies = kTile / 16;  // of the rows at most
    static constexpr uint32_t kQPart = kTgRows * D * 2, kKvPart = kTile * D * 2;
    static constexpr int kPitch = D + 4;  // floats of a row in the joins: float4 accesses without conflicts
    static constexpr uint32_t kQBytes = std::max(kQParts * kQPart, (uint32_t)(kTgRows * kPitch * 4 + 1023) / 1024 * 1024);
    static constexpr uint32_t kStage = 2 * kKvParts * kKvPart;  // K parts, then V parts
    static constexpr int kStages = kF32 ? 2 : D == 64 ? 8 : 4;
    static constexpr int kRaw = !kF32 ? 0 : D == 64 ? 4 : 2;  // slots of raw F32 rows (K or V of a tile: 16 KB)
    static constexpr uint32_t kRawSlot = kTile * D * 4;
    static constexpr size_t kSmem = kQBytes + kStages * kStage + kRaw * kRawSlot + 1024 + 512;
    static constexpr int kPart = kTgRows * (D + 2);  // a run's partial: values [128][D], maxima, sums
    // Tensor memory: columns of S (two), P (two), O.
    static constexpr uint32_t kPBuf = kQParts * kTile / 2, kPCol = 2 * kTile, kOCol = kPCol + 2 * kPBuf;
    static_assert(kOCol + kGroups * D <= 512, "tensor memory");
    static_assert(kSmem + 512 <= 227 * 1024, "shared memory");
    static constexpr float kShift = kHalf ? 14.0f : 0.0f;  // exponent added to every weight
};

// The products of parts, small ones first: part of Q or P, part of K or V.
template <typename T, int D>
__host__ __device__ constexpr int pair_q(int i) {
    if (!TreeShape<T, D>::kF32) return TreeShape<T, D>::kQParts - 1 - i;
    return i == 0 ? 2 : i == 1 ? 1 : i == 2 ? 0 : i == 3 ? 1 : 0;
}
template <typename T, int D>
__host__ __device__ constexpr int pair_kv(int i) {
    if (!TreeShape<T, D>::kF32) return 0;
    return i == 0 ? 0 : i == 1 ? 1 : i == 2 ? 2 : i == 3 ? 0 : i == 4 ? 1 : 0;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// 2^x, 0 for -infinity (the hardware's exponential, 2 units in the last place).
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two F32 values in a register pair: Blackwell adds and multiplies both at once.
__device__ __forceinline__ uint64_t pack2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}

// The parts of a pair, packed (x in the low half).  BF16: each part cuts the
// next 8 bits off, and three hold the value exactly.
__device__ __forceinline__ void split_parts(float x, float y, uint32_t (&part)[3]) {
    const uint64_t minus = pack2(-1.0f, -1.0f);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
        part[i] = __byte_perm(a, b, 0x7632);
        if (i < 2)
            unpack2(fma2(pack2(__uint_as_float(a & 0xffff0000u), __uint_as_float(b & 0xffff0000u)), minus, pack2(x, y)), x, y);
    }
}
__device__ __forceinline__ void split_parts(float x, float y, uint32_t (&part)[2]) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    part[0] = *reinterpret_cast<const uint32_t *>(&h);
    part[1] = *reinterpret_cast<const uint32_t *>(&l);
}

// 32 TMEM lanes x N consecutive columns (no wait).
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Instruction descriptor of kind::f16 (F16 or BF16 operands, F32 sums); the B
// operand's rows are K's (`transposed`: B lies [K][N]).
template <bool kHalf>
__host__ __device__ constexpr uint32_t idesc(int m, int n, bool transposed) {
    return (1u << 4) | (kHalf ? 0u : (1u << 7) | (1u << 10)) | (transposed ? 1u << 16 : 0u) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
// Descriptor of an operand [K][N] in the 128-byte swizzle: rows of 64 values of
// N, 8 rows of K to an atom of 1024 bytes; blocks of 64 of N `block` bytes apart.
__device__ __forceinline__ uint64_t sw128_mnmajor_desc(uint32_t saddr, uint32_t block) {
    return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(block >> 4) << 16) |
           (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// A place in the list of tiles.  Each item has a place more than tiles, its
// first, in which nothing is done (as in paged_attention.cu).
template <int kTile>
struct TreeCursor {
    uint32_t seq, block, inner;  // inner: KV head * head blocks + head block
    int unit, units;
    long long at;  // places from the run's first
    // Of the sequence: rows, where they begin, rows of a block, blocks; the
    // token that row 0 is, the tokens that the table reaches.
    int rows, block_rows, blocks;
    int64_t first;
    long long start, reach;

    __device__ __forceinline__ void open(const TreeGqaArgs &a, uint32_t s) {
        seq = s;
        if (a.offsets) {
            const int32_t o0 = a.offsets[s], o1 = a.offsets[s + 1];
            first = o0;
            rows = o0 < 0 || (uint64_t)o0 >= a.tokens ? 0 : (int)(max((long long)o0, min((long long)o1, (long long)a.tokens)) - o0);
        } else {
            first = s;
            rows = s < a.tokens;
        }
        const int64_t slot = a.pt.slot_ids ? a.pt.slot_ids[s] : (int64_t)s;
        const long long length = a.lengths[s];
        reach = slot < 0 || slot >= (int64_t)a.pt.slots ? 0 : max(0ll, min(length, (long long)a.pt.max_pages * a.pt.page_tokens));
        start = length - rows;
        blocks = (rows + (int)a.block_nodes - 1) / (int)a.block_nodes;
        block_rows = blocks ? (rows + blocks - 1) / blocks : 1;
    }
    // The tokens that block b sees, and its tiles.
    __device__ __forceinline__ long long tokens_of(const TreeGqaArgs &a, uint32_t b) const {
        if (a.parents) return reach;
        return min(reach, start + min((long long)rows, (long long)(b + 1) * block_rows));
    }
    __device__ __forceinline__ int units_of(const TreeGqaArgs &a, uint32_t b) const {
        return (int)((max(0ll, tokens_of(a, b)) + kTile - 1) / kTile);
    }
    // The places of all items of the sequence.
    __device__ __forceinline__ long long places(const TreeGqaArgs &a, uint32_t inners) const {
        long long n = 0;
        if (a.parents) {
            const int u = units_of(a, 0);
            return u ? (long long)blocks * (u + 1) * inners : 0;
        }
        for (int b = 0; b < blocks; ++b) {
            const int u = units_of(a, b);
            n += u ? u + 1 : 0;
        }
        return n * inners;
    }
    __device__ __forceinline__ void next(const TreeGqaArgs &a, uint32_t inners) {
        ++at;
        if (++unit < units) return;
        ++at;
        unit = 0;
        if (++inner < inners) return;
        inner = 0;
        do {
            if (++block >= (uint32_t)blocks) {
                block = 0;
                do {
                    if (seq + 1 >= a.pt.sequences) {
                        units = 0;
                        return;
                    }
                    open(a, seq + 1);
                } while (!blocks);
            }
            units = units_of(a, block);
        } while (!units);
    }
};

// Rows of blocks that see no token: zeros.
template <int kTile, int kThreads>
__device__ __forceinline__ void zero_rows(const TreeGqaArgs &a, int thread) {
    for (uint32_t s = blockIdx.x; s < a.pt.sequences; s += gridDim.x) {
        TreeCursor<kTile> c;
        c.open(a, s);
        long long none = c.reach == 0 ? c.rows : 0;
        if (!a.parents && c.reach > 0)  // whole blocks at places below 0
            none = min((long long)c.rows, max(0ll, -c.start) / c.block_rows * c.block_rows);
        const uint64_t width = (uint64_t)a.q_heads * a.head_dim;
        for (uint64_t e = thread; e < none * width; e += kThreads) a.out[c.first * width + e] = 0.0f;
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(TreeShape<T, D>::kThreads, 1) tree_gqa_kernel(const TreeGqaArgs a) {
    using S = TreeShape<T, D>;
    using Cursor = TreeCursor<S::kTile>;
    constexpr int kTile = S::kTile, kWarps = S::kThreads / 32, kMmaWarp = S::kSoftmax + kTgLoaders;
    extern __shared__ uint8_t smem_raw[];
    __shared__ long long s_scan[kWarps];
    __shared__ Cursor s_start;
    __shared__ uint8_t s_seen[S::kStages][kTile / 8];  // a bit for each token of a tile that exists
    __shared__ volatile int s_fail;
    __shared__ unsigned s_last;
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t *gbase = smem_raw + (base - raw);
    const uint32_t stages0 = base + S::kQBytes, raw0 = stages0 + S::kStages * S::kStage, bars = raw0 + S::kRaw * S::kRawSlot;
    auto q_full = [&]() { return bars; };
    auto s_full = [&](int b) { return bars + 8u * (1 + b); };
    auto p_full = [&](int b) { return bars + 8u * (3 + b); };
    auto o_full = [&](int b) { return bars + 8u * (5 + b); };
    auto kv_full = [&](int s) { return bars + 8u * (8 + s); };
    auto kv_empty = [&](int s) { return bars + 8u * (8 + S::kStages + s); };
    const uint32_t end_bar = bars + 8u * 7, tmem_slot = bars + 8u * (8 + 2 * S::kStages);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        mbar_init(q_full(), S::kSoftmax);
        for (int b = 0; b < 2; ++b) {
            mbar_init(s_full(b), 1);
            mbar_init(p_full(b), 4);
            mbar_init(o_full(b), 1);
        }
        mbar_init(end_bar, 1);
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(kv_full(s), kTgLoaders);
            mbar_init(kv_empty(s), 1);
        }
        mbar_init_fence();
        s_fail = 0;
    }
    if (warp == kMmaWarp) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    pdl_wait();
    pdl_trigger();

    // The list: places before each thread's sequences, and their total.
    const uint32_t inners = a.kv_heads * a.head_blocks, sequences = a.pt.sequences;
    const uint32_t per = (sequences + S::kThreads - 1) / S::kThreads;
    const uint32_t seq0 = min(sequences, tid * per), seq1 = min(sequences, seq0 + per);
    long long mine = 0;
    for (uint32_t s = seq0; s < seq1; ++s) {
        Cursor c;
        c.open(a, s);
        mine += c.places(a, inners);
    }
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) s_scan[warp] = upto;
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(gbase + (tmem_slot - base));
    long long before = upto - mine, total = 0;
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += s_scan[w];
        total += s_scan[w];
    }
    const long long ctas = min((long long)gridDim.x, total);
    const bool idle = (long long)blockIdx.x >= ctas;
    const long long first = idle ? 0 : total * blockIdx.x / ctas, end = idle ? 0 : total * (blockIdx.x + 1) / ctas;
    if (!idle && first >= before && first < before + mine) {
        long long left = first - before;
        Cursor c;
        c.unit = c.units = 0, c.block = c.inner = 0, c.at = 0;
        for (uint32_t s = seq0;; ++s) {  // (bounded whatever another stream does to the lengths)
            c.open(a, s);
            const long long n = c.places(a, inners);
            if (left < n || s + 1 >= seq1) break;
            left -= n;
        }
        for (;; ++c.block) {
            c.units = c.blocks ? c.units_of(a, c.block) : 0;
            const long long n = c.units ? (long long)(c.units + 1) * inners : 0;
            if (left < n || c.block + 1 >= (uint32_t)c.blocks) break;
            left -= n;
        }
        c.inner = (uint32_t)min(left / (c.units + 1), (long long)inners - 1);
        const long long place = left - (long long)c.inner * (c.units + 1);
        c.unit = (int)max(place - 1, 0ll), c.at = place == 0;
        s_start = c;
    }
    __syncthreads();
    const long long count = end - first;  // places
    // A wait that gives up once any has: every thread still reaches every barrier.
    auto wait = [&](uint32_t bar, uint32_t parity) {
        if (!s_fail && !mbar_wait(bar, parity)) s_fail = 1;
    };
    const uint32_t group = a.q_heads / a.kv_heads;

    if (warp >= S::kSoftmax && warp < kMmaWarp) {
        // ---------------------------------------------------------- loaders
        constexpr int kLt = 32 * kTgLoaders;
        constexpr int kChunks = D / 8, kStepRows = 32 / kChunks, kWarpRows = kTile / kTgLoaders, kSteps = kWarpRows / kStepRows;
        constexpr int kLook = 4;  // tiles whose rows are looked up ahead
        constexpr uint32_t kNone = 0xffffffffu;
        const int lw = warp - S::kSoftmax, lt = tid - 32 * S::kSoftmax, chunk = lane % kChunks, sub = lane / kChunks;
        const uint32_t row_bytes = a.head_dim * (uint32_t)sizeof(T);
        const bool in_row = (uint32_t)chunk * 8 < a.head_dim;
        const unsigned char *keys = static_cast<const unsigned char *>(a.keys) + chunk * 8 * sizeof(T);
        const unsigned char *values = static_cast<const unsigned char *>(a.values) + chunk * 8 * sizeof(T);
        Cursor look;
        look.at = 0, look.unit = 0;
        if (!idle) look = s_start;
        // Lane r finds token r of the warp's part of the tile at the cursor (its row
        // among all rows of the pages) and moves on; queries of a new item are
        // fetched to L2.
        auto find = [&]() -> uint32_t {
            if (look.at >= count) return kNone;
            const long long pos = (long long)(look.units - 1 - look.unit) * kTile + lw * kWarpRows + lane % kWarpRows;
            uint32_t row = kNone;
            if (pos < look.tokens_of(a, look.block)) {
                const uint32_t slot = a.pt.slot_ids ? (uint32_t)a.pt.slot_ids[look.seq] : look.seq;
                const uint32_t p = a.page_magic ? __umulhi((uint32_t)pos, a.page_magic) >> a.page_shift : (uint32_t)pos;
                const int page = a.pt.table[(uint64_t)slot * a.pt.max_pages + p];
                if (page >= 0 && (uint64_t)page < a.pt.pages)
                    row = ((uint32_t)page * a.kv_heads + look.inner / a.head_blocks) * a.pt.page_tokens +
                          ((uint32_t)pos - p * a.pt.page_tokens);
            }
            look.next(a, inners);
            if (look.unit == 0 && look.at < count) {
                const uint32_t head = look.inner % a.head_blocks * a.block_heads, heads = min(a.block_heads, group - head);
                const uint32_t to = min((uint32_t)look.rows, (look.block + 1) * look.block_rows);
                for (uint32_t r = lt; r < kTgRows; r += kLt) {
                    const uint32_t node = look.block * look.block_rows + r / heads;
                    if (node >= to) break;
                    const float *q = a.q + ((uint64_t)(look.first + node) * a.q_heads + look.inner / a.head_blocks * group + head + r % heads) * a.head_dim;
                    for (uint32_t d = 0; d < a.head_dim; d += 32) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + d));
                }
            }
            return row;
        };
        // The tiles of this run.
        uint32_t ahead[kLook];
        long long tiles = 0, found = 0;
        auto shift = [&]() {
#pragma unroll
            for (int i = 0; i + 1 < kLook; ++i) ahead[i] = ahead[i + 1];
            const bool more = look.at < count;
            ahead[kLook - 1] = find();
            found += more;
        };
        for (int i = 0; i < kLook; ++i) shift();
        auto offset = [&](int i) {  // of this lane's chunk of step i in a part's tile
            const int row = lw * kWarpRows + i * kStepRows + sub, c = chunk % 8;
            return (uint32_t)(chunk / 8 * kTile * 128 + row * 128 + ((c ^ (row & 7)) << 4));
        };
        auto mark = [&](int stage, uint32_t row_at) {  // which of the warp's tokens exist
            const unsigned seen = __ballot_sync(0xffffffffu, row_at != kNone);
            if (lane < kWarpRows / 8) s_seen[stage][lw * (kWarpRows / 8) + lane] = (uint8_t)(seen >> (8 * lane));
        };
        if constexpr (!S::kF32) {
            // Tiles between a load and its arrival.  (O of a tile is issued after S of the
            // next, so a stage is only free when the tile after its own has arrived.)
            constexpr int kLag = S::kStages - 2;
            for (; tiles < found || tiles < kLag; ++tiles) {  // (at least kLag groups, so that the waits below count right)
                if (tiles < found) {
                    const int stage = (int)(tiles % S::kStages);
                    if (tiles >= S::kStages) wait(kv_empty(stage), (uint32_t)(tiles / S::kStages - 1) & 1);
                    __syncwarp();
                    const uint32_t row_at = ahead[0], to = stages0 + stage * S::kStage;
                    mark(stage, row_at);
                    if (a.aligned && __all_sync(0xffffffffu, row_at != kNone)) {
                        // Whole rows, and 16 tokens to a page at least: one address for each 16.
                        constexpr int kRun = 16 / kStepRows;
#pragma unroll
                        for (int u = 0; u < kSteps / kRun; ++u) {
                            const uint64_t from = (uint64_t)(__shfl_sync(0xffffffffu, row_at, u * 16) + sub) * (D * 2);
#pragma unroll
                            for (int i = 0; i < kRun; ++i) {
                                cp_async16(to + offset(u * kRun + i), keys + from + i * kStepRows * D * 2, 16);
                                cp_async16(to + S::kKvPart + offset(u * kRun + i), values + from + i * kStepRows * D * 2, 16);
                            }
                        }
                    } else {
#pragma unroll 2
                        for (int i = 0; i < kSteps; ++i) {
                            const uint32_t row = __shfl_sync(0xffffffffu, row_at, i * kStepRows + sub);
                            const bool there = row != kNone && in_row;
                            const uint64_t from = (uint64_t)(there ? row : 0) * row_bytes;
                            cp_async16(to + offset(i), keys + (there ? from : 0) - (there ? 0 : chunk * 8 * sizeof(T)), there ? 16 : 0);
                            cp_async16(to + S::kKvPart + offset(i), values + (there ? from : 0) - (there ? 0 : chunk * 8 * sizeof(T)), there ? 16 : 0);
                        }
                    }
                    shift();
                }
                cp_async_commit();
                if (tiles >= kLag) {
                    cp_async_wait<kLag>();
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(kv_full((int)((tiles - kLag) % S::kStages)));
                }
            }
            cp_async_wait<0>();
            fence_async_smem();
            __syncwarp();
            if (lane == 0)
                for (long long t = max(tiles - kLag, 0ll); t < found; ++t) mbar_arrive(kv_full((int)(t % S::kStages)));
        } else {
            // Raw rows arrive in slots that only this thread reads, K and V of a tile
            // one after the other; the parts go to the tile's stage.
            uint32_t rows[S::kRaw / 2];  // of the tiles under way
            auto fetch = [&](long long unit, uint32_t row_at) {  // unit: tile * 2, + 1 for V
                const uint32_t to = raw0 + (uint32_t)(unit % S::kRaw) * S::kRawSlot + lt * 16;
                const unsigned char *src = unit & 1 ? values : keys;
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    const uint32_t row = __shfl_sync(0xffffffffu, row_at, i * kStepRows + sub);
                    const bool there = row != kNone && in_row;
                    const unsigned char *from = there ? src + (uint64_t)row * row_bytes : src - chunk * 8 * sizeof(T);
                    cp_async16(to + 2 * i * kLt * 16, from, there ? 16 : 0);
                    cp_async16(to + (2 * i + 1) * kLt * 16, from + (there ? 16 : 0), there ? 16 : 0);
                }
            };
#pragma unroll
            for (int i = 0; i < S::kRaw / 2; ++i) {
                rows[i] = ahead[0];
                const bool any = i < found;
                shift();
                if (any) fetch(2 * i, rows[i]);
                cp_async_commit();
                if (any) fetch(2 * i + 1, rows[i]);
                cp_async_commit();
            }
            for (; tiles < found; ++tiles) {
                const int stage = (int)(tiles % S::kStages);
                if (tiles >= S::kStages) wait(kv_empty(stage), (uint32_t)(tiles / S::kStages - 1) & 1);
                __syncwarp();
                const uint32_t row_at = rows[0];
                mark(stage, row_at);
#pragma unroll
                for (int i = 0; i + 1 < S::kRaw / 2; ++i) rows[i] = rows[i + 1];
                const bool more = tiles + S::kRaw / 2 < found;
                rows[S::kRaw / 2 - 1] = ahead[0];
                if (more) shift();
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    cp_async_wait<S::kRaw - 1>();
                    const long long unit = 2 * tiles + v;
                    const uint8_t *from = gbase + (raw0 - base) + (unit % S::kRaw) * S::kRawSlot + lt * 16;
                    uint8_t *to = gbase + (stages0 - base) + stage * S::kStage + v * 3 * S::kKvPart;
#pragma unroll
                    for (int i = 0; i < kSteps; ++i) {
                        const float4 x = *reinterpret_cast<const float4 *>(from + 2 * i * kLt * 16);
                        const float4 y = *reinterpret_cast<const float4 *>(from + (2 * i + 1) * kLt * 16);
                        uint32_t w0[3], w1[3], w2[3], w3[3];
                        split_parts(x.x, x.y, w0), split_parts(x.z, x.w, w1);
                        split_parts(y.x, y.y, w2), split_parts(y.z, y.w, w3);
#pragma unroll
                        for (int p = 0; p < 3; ++p)
                            *reinterpret_cast<uint4 *>(to + p * S::kKvPart + offset(i)) = make_uint4(w0[p], w1[p], w2[p], w3[p]);
                    }
                    if (more) fetch(unit + S::kRaw, rows[S::kRaw / 2 - 1]);
                    cp_async_commit();
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(kv_full(stage));
            }
            cp_async_wait<0>();
        }
        zero_rows<kTile, kLt>(a, lt);
    } else if (!idle && warp < S::kSoftmax) {
        // ---------------------------------------------------------- softmax
        const int wg = warp / 4, row = 32 * (warp & 3) + lane;  // row: TMEM lane
        const uint32_t quarter = (uint32_t)(32 * (warp & 3)) << 16;
        // log2(e) / sqrt(D), and 1.2e-7 of it: the tensor core cuts a score's sums, which
        // measured 0.7e-7 to 2e-7 less than they should be.
        const float to_base2 = 1.4426950408889634f * (1.0f + 1.2e-7f) / sqrtf((float)a.head_dim);
        Cursor use = s_start;
        long long tile = 0;  // of the run
        int copies_before = 1;
        uint32_t item = 0;
        float *join = reinterpret_cast<float *>(gbase);  // [128][kPitch]: values, maximum, sum (over Q, once its products are done)
        while (use.at < count) {
            // The item: its rows, copies of them, this thread's row.
            const uint32_t kvh = use.inner / a.head_blocks, head = use.inner % a.head_blocks * a.block_heads;
            const uint32_t heads = min(a.block_heads, group - head), node0 = use.block * use.block_rows;
            const int rows = (int)((min((uint32_t)use.rows, node0 + use.block_rows) - node0) * heads);
            const int copies = rows <= 32 && S::kCopies >= 4 ? 4 : rows <= 64 ? 2 : 1, span = kTgRows / copies;
            const int mine_row = row % span, copy = row / span;
            const bool active = mine_row < rows, warp_active = __any_sync(0xffffffffu, active);
            const int node = (int)node0 + mine_row / (int)heads;
            const uint64_t q_row = (uint64_t)(use.first + (active ? node : 0)) * a.q_heads + kvh * group + head + mine_row % heads;
            float unit_scale = 1.0f;
            if (active) {
                const float *q = a.q + q_row * a.head_dim;
                float up = to_base2;
                if constexpr (S::kHalf) {
                    float most = 0.0f;
                    for (uint32_t d = 0; d < a.head_dim; d += 4) {
                        const float4 v = *reinterpret_cast<const float4 *>(q + d);
                        most = fmaxf(fmaxf(fmaxf(most, fabsf(v.x)), fmaxf(fabsf(v.y), fabsf(v.z))), fabsf(v.w));
                    }
                    most *= to_base2;
                    if (most > 0.0f && most < INFINITY) {
                        const int e = min(max(14 - ilogbf(most), -100), 100);
                        up = ldexpf(to_base2, e), unit_scale = ldexpf(1.0f, -e);
                    }
                }
#pragma unroll 4
                for (int c = wg; c < D / 8; c += S::kGroups) {
                    float4 x = make_float4(0, 0, 0, 0), y = x;
                    if ((uint32_t)c * 8 < a.head_dim) {
                        x = *reinterpret_cast<const float4 *>(q + c * 8);
                        y = *reinterpret_cast<const float4 *>(q + c * 8 + 4);
                    }
                    uint32_t w0[S::kQParts], w1[S::kQParts], w2[S::kQParts], w3[S::kQParts];
                    split_parts(x.x * up, x.y * up, w0), split_parts(x.z * up, x.w * up, w1);
                    split_parts(y.x * up, y.y * up, w2), split_parts(y.z * up, y.w * up, w3);
                    uint8_t *to = gbase + c / 8 * (kTgRows * 128) + row * 128 + ((c % 8 ^ (row & 7)) << 4);
#pragma unroll
                    for (int p = 0; p < S::kQParts; ++p)
                        *reinterpret_cast<uint4 *>(to + p * S::kQPart) = make_uint4(w0[p], w1[p], w2[p], w3[p]);
                }
            }
            fence_async_smem();
            // A copy's weights are zero for the other copies' tokens, from here on.
            if (copies != copies_before && copies > 1) {
                const uint32_t zeros[8] = {};
                for (uint32_t c = 0; c < 2 * S::kPBuf; c += 8) tmem_st8(tmem + quarter + S::kPCol + c, zeros);
                tmem_wait_st();
                tc_fence_before_sync();
            }
            copies_before = copies;
            if constexpr (S::kGroups == 2) named_barrier(1, 256);  // (both groups write zeros over both buffers)
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full());

            float m = -INFINITY, l = 0.0f, o[D], keep_last = 0.0f;
#pragma unroll
            for (int i = 0; i < D; ++i) o[i] = 0.0f;
            long long last = -1;  // the tile whose O has not been added
            auto add = [&]() {
                const int b = (int)(last & 1);
                wait(o_full(b), (uint32_t)(last >> 1) & 1);
                __syncwarp();
                tc_fence_after_sync();
                const uint64_t keep2 = pack2(keep_last, keep_last);
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    uint32_t x[2][16];
                    tmem_ld(tmem + quarter + S::kOCol + (S::kGroups == 2 ? b * D : 0) + c, x[0]);
                    tmem_ld(tmem + quarter + S::kOCol + (S::kGroups == 2 ? b * D : 0) + c + 16, x[1]);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i += 2)
                        unpack2(fma2(pack2(o[c + i], o[c + i + 1]), keep2, pack2(__uint_as_float(x[i / 16][i % 16]), __uint_as_float(x[i / 16][i % 16 + 1]))),
                                o[c + i], o[c + i + 1]);
                }
                tc_fence_before_sync();
            };
            int ancestor = active ? node : -1;  // the next to be met
            const long long begun = use.at;
            const int unit0 = use.unit;
            // One tile: this thread's tokens are columns [c0, c0 + 16 * chunks).
            const int chunks = kTile / 16 / copies;
            auto softmax = [&]() {
                const int b = (int)(tile & 1), c0 = copy * 16 * chunks, stage = (int)(tile % S::kStages);
                wait(kv_full(stage), (uint32_t)(tile / S::kStages) & 1);  // (for s_seen)
                wait(s_full(b), (uint32_t)(tile >> 1) & 1);
                __syncwarp();
                tc_fence_after_sync();
                if (!warp_active) {  // (keeps step: its arrivals count)
                    if (lane == 0) mbar_arrive(p_full(b));
                    return;
                }
                // Which of the tokens this row sees.
                uint64_t seen = kTile == 64 ? *reinterpret_cast<const volatile uint64_t *>(s_seen[stage])
                                            : (uint64_t)*reinterpret_cast<const volatile uint32_t *>(s_seen[stage]);
                const long long t0 = (long long)(use.units - 1 - use.unit) * kTile;
                if (t0 + kTile > use.start) {
                    const long long low = t0 - use.start;  // the row that the tile's first token is
                    uint64_t drafted = low < 0 ? ~0ull >> (64 + low) : 0;
                    if (!a.parents) {
                        const long long own = node - low;  // (at least: rows before it are seen)
                        drafted = own < 0 ? 0 : own >= 63 ? ~0ull : ~0ull >> (63 - own);
                    } else {
                        while (ancestor >= 0 && ancestor >= low) {
                            if (ancestor - low < kTile) drafted |= 1ull << (ancestor - low);
                            const int up = a.parents[use.first + ancestor];
                            ancestor = up < ancestor ? max(up, -1) : -1;
                        }
                    }
                    seen &= drafted;
                }
                if (copies > 1) seen >>= c0;
                const uint64_t every = copies == 1 && kTile == 64 ? ~0ull : (1ull << (kTile / copies)) - 1;
                const bool all = __all_sync(0xffffffffu, !active || (seen & every) == every);
                const uint32_t from = tmem + quarter + b * kTile + c0;
                // What the row does not see has a score of -infinity.
                auto hide = [&](uint32_t (&x)[16], int c) {
                    const uint32_t bits = active ? (uint32_t)(seen >> (16 * c)) : 0xffffu;  // (nobody reads the others' rows)
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] = bits >> i & 1 ? x[i] : 0xff800000u;
                };
                float most = -INFINITY;
#pragma unroll 1
                for (int c = 0; c < chunks; ++c) {
                    uint32_t x[16];
                    tmem_ld(from + 16 * c, x);
                    tmem_wait_ld();
                    if (!all) hide(x, c);
#pragma unroll
                    for (int i = 0; i < 16; i += 2)
                        most = fmaxf(most, fmaxf(__uint_as_float(x[i]), __uint_as_float(x[i + 1])));
                }
                if constexpr (S::kHalf) most *= unit_scale;
                const float now = fmaxf(m, most), reference = now == -INFINITY ? 0.0f : now;
                const float keep = exp2_fast(m - reference);
                m = now;
                if (S::kGroups == 2 && last >= 0) add();  // (its P buffer is free then)
                uint64_t sum = 0;  // two sums
                const uint64_t scale2 = pack2(unit_scale, unit_scale), shift2 = pack2(S::kShift - reference, S::kShift - reference);
                const uint32_t to = tmem + quarter + S::kPCol + b * S::kPBuf + c0 / 2;
#pragma unroll 1
                for (int c = 0; c < chunks; ++c) {
                    uint32_t x[16];
                    tmem_ld(from + 16 * c, x);
                    tmem_wait_ld();
                    if (!all) hide(x, c);
                    uint32_t part[S::kQParts][8];
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const uint64_t s = pack2(__uint_as_float(x[i]), __uint_as_float(x[i + 1]));
                        float p0, p1;
                        unpack2(S::kHalf ? fma2(s, scale2, shift2) : add2(s, shift2), p0, p1);
                        p0 = exp2_fast(p0), p1 = exp2_fast(p1);
                        sum = add2(sum, pack2(p0, p1));
                        uint32_t w[S::kQParts];
                        split_parts(p0, p1, w);
#pragma unroll
                        for (int k = 0; k < S::kQParts; ++k) part[k][i / 2] = w[k];
                    }
#pragma unroll
                    for (int k = 0; k < S::kQParts; ++k) tmem_st8(to + k * (kTile / 2) + 8 * c, part[k]);
                }
                tmem_wait_st();
                if (S::kGroups == 1 && last >= 0) add();  // (O has one buffer)
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(b));
                float sum0, sum1;
                unpack2(sum, sum0, sum1);
                l = fmaf(l, keep, sum0 + sum1);
                keep_last = keep;
                last = tile;
            };
            bool whole = false;  // the item's last tile is this run's
            for (bool more = true; more;) {
                if (S::kGroups == 1 || (tile & 1) == wg) softmax();
                ++tile;
                if (use.unit + 1 == use.units || use.at + 1 >= count) {
                    whole = use.unit + 1 == use.units;
                    more = false;
                } else {
                    use.next(a, inners);
                }
            }
            if (last >= 0) add();

            // Join: the other group, then the other copies.
            auto put = [&]() {
                float *to = join + row * S::kPitch;
#pragma unroll
                for (int i = 0; i < D; i += 4) *reinterpret_cast<float4 *>(to + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                *reinterpret_cast<float2 *>(to + D) = make_float2(m, l);
            };
            auto take = [&](int other) {
                const float *from = join + other * S::kPitch;
                const float2 ml = *reinterpret_cast<const float2 *>(from + D);
                const float now = fmaxf(m, ml.x), reference = now == -INFINITY ? 0.0f : now;
                const float f = exp2_fast(m - reference), g = exp2_fast(ml.x - reference);
                m = now, l = fmaf(ml.y, g, l * f);
#pragma unroll
                for (int i = 0; i < D; i += 4) {
                    const float4 v = *reinterpret_cast<const float4 *>(from + i);
                    o[i] = fmaf(v.x, g, o[i] * f), o[i + 1] = fmaf(v.y, g, o[i + 1] * f);
                    o[i + 2] = fmaf(v.z, g, o[i + 2] * f), o[i + 3] = fmaf(v.w, g, o[i + 3] * f);
                }
            };
            if constexpr (S::kGroups == 2) {
                named_barrier(1, 256);  // (all products of Q are done)
                if (wg == 1) put();
                named_barrier(1, 256);
                if (wg == 0) take(row);
            } else {
                named_barrier(2, 128);
            }
            if (copies > 1 && wg == 0) {
                if (S::kGroups == 2) named_barrier(2, 128);
                if (copy) put();
                named_barrier(2, 128);
                if (!copy)
                    for (int c = 1; c < copies; ++c) take(c * span + mine_row);
            }
            const bool starts = unit0 == 0;
            const bool writer = wg == 0 && copy == 0 && active;
            if (starts && whole) {
                if (writer) {
                    float *to = a.out + q_row * a.head_dim;
                    const float inverse = s_fail ? NAN : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
                    for (int i = 0; i < D; i += 4)
                        if ((uint32_t)i < a.head_dim)
                            *reinterpret_cast<float4 *>(to + i) = make_float4(o[i] * inverse, o[i + 1] * inverse, o[i + 2] * inverse, o[i + 3] * inverse);
                }
            } else {
                // A run that starts the item writes slot 1 of its CTA, one that goes on with it slot 0.
                if (writer) {
                    float *part = a.partial + (uint64_t)(2 * blockIdx.x + starts) * S::kPart;
#pragma unroll
                    for (int i = 0; i < D; i += 4)
                        *reinterpret_cast<float4 *>(part + mine_row * D + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    part[kTgRows * D + mine_row] = m, part[kTgRows * (D + 1) + mine_row] = s_fail ? NAN : l;
                }
                // The places [u0, u1) of the item's tiles and the CTAs that own its ends.
                const long long u0 = first + begun - unit0, u1 = u0 + use.units;
                const int cta0 = (int)(((u0 + 1) * ctas - 1) / total), runs = (int)((u1 * ctas - 1) / total) - cta0 + 1;
                if constexpr (S::kGroups == 2) named_barrier(1, 256); else named_barrier(2, 128);
                if (tid == 0) {
                    __threadfence();  // the block's partial, then its arrival
                    s_last = atomicAdd(&a.arrived[cta0], 1u) + 1 == (unsigned)runs;
                    if (s_last) a.arrived[cta0] = 0;
                    __threadfence();  // and the others' before what the block reads next
                }
                if constexpr (S::kGroups == 2) named_barrier(1, 256); else named_barrier(2, 128);
                if (s_last) {
                    const float *partial = a.partial + (uint64_t)2 * cta0 * S::kPart;
                    auto slot = [&](int k) { return partial + (uint64_t)(k ? 2 * k : 1) * S::kPart; };
                    for (int e = tid; e < rows * (D / 4); e += S::kSoftmax * 32) {
                        const int r = e / (D / 4), d = e % (D / 4) * 4;
                        float most = -INFINITY, sum = 0.0f;
#pragma unroll 8
                        for (int k = 0; k < runs; ++k) most = fmaxf(most, __ldcg(slot(k) + kTgRows * D + r));
                        const float reference = most == -INFINITY ? 0.0f : most;
                        float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll 4
                        for (int k = 0; k < runs; ++k) {
                            const float *from = slot(k);
                            const float f = exp2_fast(__ldcg(from + kTgRows * D + r) - reference);
                            sum = fmaf(__ldcg(from + kTgRows * (D + 1) + r), f, sum);
                            const float4 v = __ldcg(reinterpret_cast<const float4 *>(from + r * D + d));
                            acc.x = fmaf(v.x, f, acc.x), acc.y = fmaf(v.y, f, acc.y);
                            acc.z = fmaf(v.z, f, acc.z), acc.w = fmaf(v.w, f, acc.w);
                        }
                        if ((uint32_t)d < a.head_dim) {
                            const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
                            float *to = a.out + ((uint64_t)(use.first + node0 + r / heads) * a.q_heads + kvh * group + head + r % heads) * a.head_dim;
                            *reinterpret_cast<float4 *>(to + d) = make_float4(acc.x * inverse, acc.y * inverse, acc.z * inverse, acc.w * inverse);
                        }
                    }
                }
            }
            if constexpr (S::kGroups == 2) named_barrier(1, 256); else named_barrier(2, 128);  // (the join has been read)
            use.next(a, inners);
            ++item;
        }
    } else if (!idle && warp == kMmaWarp) {
        // ---------------------------------------------------------- products
        if (lane == 0) {
            constexpr uint32_t kIdescS = idesc<S::kHalf>(kTgRows, kTile, false), kIdescO = idesc<S::kHalf>(kTgRows, D, true);
            Cursor use = s_start;
            long long tile = 0;
            uint32_t item = 0;
            auto scores = [&](long long t) {
                const int stage = (int)(t % S::kStages), b = (int)(t & 1);
                wait(kv_full(stage), (uint32_t)(t / S::kStages) & 1);
                if (s_fail) return;
                tc_fence_after_sync();
                // (Descriptors hold addresses in units of 16 bytes in their low bits.)
                const uint64_t q = sw128_kmajor_desc(base), k = sw128_kmajor_desc(stages0 + stage * S::kStage);
                const uint32_t to = tmem + b * kTile;
#pragma unroll
                for (int i = 0; i < S::kPairs; ++i)
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
                        mma_bf16_ss(to, q + (pair_q<T, D>(i) * S::kQPart + kk / 4 * (kTgRows * 128) + kk % 4 * 32) / 16,
                                    k + (pair_kv<T, D>(i) * S::kKvPart + kk / 4 * (kTile * 128) + kk % 4 * 32) / 16, kIdescS,
                                    (i | kk) != 0);
                mma_commit(s_full(b));
            };
            while (use.at < count) {
                // Tiles of the item in this run.
                const long long n = min((long long)(use.units - use.unit), count - use.at);
                wait(q_full(), item & 1);
                tc_fence_after_sync();
                scores(tile);
                for (long long t = tile; t < tile + n; ++t) {
                    if (t + 1 < tile + n) scores(t + 1);
                    const int stage = (int)(t % S::kStages), b = (int)(t & 1);
                    wait(p_full(b), (uint32_t)(t >> 1) & 1);
                    if (s_fail) continue;
                    tc_fence_after_sync();
                    const uint64_t v = sw128_mnmajor_desc(stages0 + stage * S::kStage + S::kKvParts * S::kKvPart, kTile * 128);
                    const uint32_t p = tmem + S::kPCol + b * S::kPBuf, to = tmem + S::kOCol + (S::kGroups == 2 ? b * D : 0);
#pragma unroll
                    for (int i = 0; i < S::kPairs; ++i)
#pragma unroll
                        for (int kk = 0; kk < kTile / 16; ++kk)
                            mma_bf16_ts(to, p + pair_q<T, D>(i) * (kTile / 2) + kk * 8,
                                        v + (pair_kv<T, D>(i) * S::kKvPart + kk * 2048) / 16, kIdescO, (i | kk) != 0);
                    mma_commit(o_full(b));
                    mma_commit(kv_empty(stage));
                }
                tile += n;
                for (long long i = 0; i < n; ++i) use.next(a, inners);
                ++item;
            }
            // Nothing is under way when the tensor memory goes back.
            mma_commit(end_bar);
            mbar_wait(end_bar, 0);
        }
        __syncwarp();
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
    if (tid == 0 && s_fail) atomicOr(&g_tree_fault, 1u);
}

template <typename T, int D>
int32_t tree_gqa_run(const TreeGqaArgs &a0, void *workspace, cudaStream_t stream) {
    using S = TreeShape<T, D>;
    TreeGqaArgs a = a0;
    a.aligned = a.pt.page_tokens % 16 == 0 && a.head_dim == D;
    a.arrived = static_cast<unsigned *>(workspace);
    a.partial = reinterpret_cast<float *>(static_cast<char *>(workspace) + 16384);
    // As many CTAs as the workspace has slots for, whatever the device.
    const int64_t slots = (MF_PAGED_TREE_WORKSPACE_BYTES - 16384) / (sizeof(float) * 2 * S::kPart);
    const int64_t grid = std::min({(int64_t)sm_count(), slots, (int64_t)4096});
    static std::atomic<uint64_t> ready{0};
    if (int32_t st = allow_smem(tree_gqa_kernel<T, D>, S::kSmem, ready)) return st;
    return launch(tree_gqa_kernel<T, D>, dim3((unsigned)grid), dim3(S::kThreads), S::kSmem, stream, "tree_gqa_kernel", a);
}

}  // namespace

int32_t paged_tree_gqa(float *out, const float *q, const void *key_pages, const void *value_pages, int32_t dtype,
                       const PagedTable &pt, uint64_t tokens, const int32_t *lengths, const int32_t *offsets,
                       const int32_t *parents, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, void *workspace,
                       cudaStream_t stream) {
    if (!pt.sequences || !tokens) return MF_OK;
    TreeGqaArgs a;
    a.out = out, a.q = q, a.keys = key_pages, a.values = value_pages, a.pt = pt, a.tokens = tokens;
    a.lengths = lengths, a.offsets = offsets, a.parents = parents;
    a.q_heads = q_heads, a.kv_heads = kv_heads, a.head_dim = head_dim;
    const uint32_t group = q_heads / kv_heads;
    a.head_blocks = (group + kTgRows - 1) / kTgRows;
    a.block_heads = (group + a.head_blocks - 1) / a.head_blocks;
    a.block_nodes = kTgRows / a.block_heads;
    a.page_shift = 0;
    while ((2u << a.page_shift) < pt.page_tokens) ++a.page_shift;
    a.page_magic = pt.page_tokens == 1 ? 0 : (uint32_t)(((1ull << (32 + a.page_shift)) + pt.page_tokens - 1) / pt.page_tokens);
    if (head_dim <= 64)
        return dtype == MF_PAGE_F32   ? tree_gqa_run<float, 64>(a, workspace, stream)
               : dtype == MF_PAGE_F16 ? tree_gqa_run<__half, 64>(a, workspace, stream)
                                      : tree_gqa_run<__nv_bfloat16, 64>(a, workspace, stream);
    return dtype == MF_PAGE_F32   ? tree_gqa_run<float, 128>(a, workspace, stream)
           : dtype == MF_PAGE_F16 ? tree_gqa_run<__half, 128>(a, workspace, stream)
                                  : tree_gqa_run<__nv_bfloat16, 128>(a, workspace, stream);
}

int32_t tree_attention_faults(uint32_t *flags) {
    unsigned v = 0;
    MF_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_tree_fault, sizeof(v)));
    const unsigned zero = 0;
    MF_CUDA_TRY(cudaMemcpyToSymbol(g_tree_fault, &zero, sizeof(zero)));
    *flags = v;
    return MF_OK;
}

}  // namespace mf
