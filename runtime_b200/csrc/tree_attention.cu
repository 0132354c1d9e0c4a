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
// lies there as in its page, [token][dimension], and is read transposed.  Two
// softmax threads own a row: each takes half of a tile's tokens and, later, half
// of the dimensions of its O; they exchange their maxima.  (One thread a row
// needs twice the registers, which leaves two warps to a scheduler, too few to
// hide one another's latencies: 64 large trees 313 us.)  Of 64 rows
// or fewer there are two copies, each of which takes half of the tokens (its P
// is zero for the others'); copies are joined at the end.
//
// Roles.  Eight softmax warps for each of two tiles in turn (for one where D is
// 128: its sums fill the registers), each with sums of its own, joined at the
// end; warps that issue the loads (runs of a page's rows by TMA, gathers of four
// where some do not exist, which are filled with zeros; some 100 cycles each, so
// K and V have a warp each: with one, 64 large trees take 240 us); several that
// split the tiles of F32 pages (whose softmax then has one group: with two
// splitting warps 32 ragged sequences took 158 us for 105 with eight, and with
// two groups, which leaves those eight 40 registers a thread, 118); one that issues the products
// S and one for O (a single one spent as long on its waits as the products take).
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
//
// Measured.  64 trees of 24-32 rows over 1000-4000 tokens, 32/8 heads of 64, BF16
// pages (364 MB; 112 GFLOP, parts counted): 211 us, 1.7 TB/s and 0.53 PFLOP/s.
// The bound is the softmax and what every tile and item costs beside its arithmetic:
// in builds that leave parts out (of then 222 us) the softmax alone, without loads and
// products, takes 191 us, the rest without it 147, and with softmax, products, loads
// and the queries' split all left out 86 of then 208 remain: waits, exchanges,
// arrivals, joins.  Its warps issue in 62% of cycles, four to a scheduler, all
// that the registers allow; what keeps the rest are TMEM reads, exchanges and
// dependent chains: a tenth fewer instructions (pairs of values in one) took the
// same time.  Not kept, each for the registers it spills: the scores of both
// halves of a chunk in one read (234 us), scores kept from maximum to weights
// (262), weights against the last tile's maximum, without an exchange (233).
// One tree of 8 rows over 257 tokens: 16 us, half of it the chain lengths - table -
// rows - parts - S - softmax - O, a fifth the join of five CTAs.
// Spilled (bytes stored): F32 pages 8 with heads of 64, 204 with 128 (128 registers a
// thread, sums of 64 dimensions); F16 and BF16 16 and 20 with 128, none with 64.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>

#include "mf_common.cuh"
#include "packed_kernels.h"
#include "paged_common.cuh"
#include "tc_sm100.cuh"

namespace mf {

// Set (bit 0) by a tree attention whose pipeline wait timed out.
__device__ unsigned int g_tree_fault = 0;

static std::atomic<uint32_t> g_tree_tries{kTreeMostTries};
void set_tree_tries(uint32_t tries) { g_tree_tries.store(tries, std::memory_order_relaxed); }

namespace {

using namespace sm100;

constexpr int kTgRows = 128;   // rows of a block: the products' M

struct TreeGqaArgs {
    float *out;
    const float *q;
    const void *keys, *values;
    PagedTable pt;
    uint64_t tokens;
    const int32_t *lengths, *offsets, *parents;
    uint32_t q_heads, kv_heads, head_dim;
    float scale, scale_low;                          // log2(e) / sqrt(head_dim) and what the scores lose, in two parts
    uint32_t head_blocks, block_heads, block_nodes;  // of a KV head's query heads; heads and rows of a block at most
    uint32_t page_magic, page_shift;                 // as in paged_attention.cu
    uint32_t tries;                                  // of a wait; 0: the call gives up at once
    uint32_t run;                                    // rows of a page that a load takes at once; below 4: gathers only
    unsigned *arrived;                               // [CTAs], zero between calls
    float *partial;                                  // [2 * CTAs][kPart]
};

// The rows of K and V pages (kind 0 and 1), to be loaded in runs and one by one.
struct TreeMaps {
    CUtensorMap runs[2], rows[2];
};

template <typename T, int D>
struct TreeShape {
    static constexpr bool kF32 = sizeof(T) == 4;
    static constexpr bool kHalf = std::is_same<T, __half>::value;
    static constexpr int kQParts = kHalf ? 2 : 3;  // of Q and P
    static constexpr int kKvParts = kF32 ? 3 : 1;
    static constexpr int kPairs = kF32 ? 6 : kQParts;
    static constexpr int kTile = kF32 && D == 128 ? 32 : 64;  // (F32's parts of 64 tokens of 128 do not fit)
    static constexpr int kGroups = D == 64 && !kF32 ? 2 : 1;  // groups of softmax warps
    static constexpr int kSoftmax = 8 * kGroups;              // warps
    static constexpr int kLoads = kF32 ? 1 : 2, kHelpers = !kF32 ? 0 : D == 64 ? 8 : 4;  // warps
    static constexpr int kLoadWarp = kSoftmax, kHelperWarp = kLoadWarp + kLoads, kMmaWarp = kHelperWarp + kHelpers;
    static constexpr int kThreads = 32 * (kMmaWarp + 2);
    // Registers a thread where all warps but the softmax's are one warpgroup, which
    // needs fewer: what it gives up keeps sums from being spilled (64 large trees
    // 222 -> 215 us).
    static constexpr bool kMoreRegs = kGroups == 2 && kMmaWarp + 2 - kSoftmax == 4;
    static constexpr int kSoftmaxRegs = 104, kOtherRegs = 64, kAllRegs = 32 * kSoftmax * kSoftmaxRegs + 128 * kOtherRegs;
    static constexpr uint32_t kQPart = kTgRows * D * 2, kKvPart = kTile * D * 2;
    static constexpr uint32_t kQBytes = kQParts * kQPart;
    // Joins go through shared memory kCols dimensions at a time, rows kPitch
    // floats apart (16-byte accesses without conflicts).
    static constexpr int kCols = 8, kPitch = 12;
    static constexpr uint32_t kJoinBytes = 2 * kGroups * kTgRows * kPitch * 4;
    static constexpr int kMostCopies = kTile / 32;  // of the rows
    static constexpr uint32_t kStage = 2 * kKvParts * kKvPart;  // K parts, then V parts
    static constexpr int kStages = kF32 ? 2 : D == 64 ? 9 : 3;
    static constexpr int kRaw = !kF32 ? 0 : D == 64 ? 4 : 2;  // slots of raw F32 rows (K or V of a tile: 16 KB)
    static constexpr uint32_t kRawSlot = kTile * D * 4;
    static constexpr uint32_t kStageAt = kQBytes, kRawAt = kStageAt + kStages * kStage,
                              kJoinAt = kRawAt + kRaw * kRawSlot, kBarAt = kJoinAt + (kGroups == 2 || kMostCopies == 2 ? kJoinBytes : 0);
    static constexpr size_t kSmem = kBarAt + 1008 + (kF32 ? 256 : 512);  // (from a 16-byte boundary on to one of 1024)
    static constexpr int kPart = kTgRows * (D + 2);  // a run's partial: values [128][D], maxima, sums
    // Tensor memory: columns of S (one more than groups, so that a group finds its
    // next scores there: 64 large trees 206 us for 224 without, prompt chunks 94 for
    // 124), P (two), O.
    static constexpr int kSBufs = kGroups + 1;
    static constexpr uint32_t kPBuf = kQParts * kTile / 2, kPCol = kSBufs * kTile, kOCol = kPCol + 2 * kPBuf;
    static_assert(kOCol + kGroups * D <= 512, "tensor memory");
    static_assert(23 + 4 * kStages < (kF32 ? 32 : 64) && kRaw <= 4, "barriers");
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

// Four rows of a tensor [rows][columns] (from column x on, as many as its box
// has) to `dst`; rows past the last are zeros.
__device__ __forceinline__ void gather4(uint32_t dst, const CUtensorMap *map, int32_t x, const uint32_t (&row)[4], uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, "
        "%6}], [%7];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(row[0]), "r"(row[1]), "r"(row[2]), "r"(row[3]), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tile_load(uint32_t dst, const CUtensorMap *map, int32_t x, uint32_t row, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(row), "r"(bar)
        : "memory");
}
// Whether the phase with `parity` is complete.  (A try_wait takes 200 cycles even
// then, and three of them were a third of the time between two products.)
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// The same; the thread sleeps for up to a microsecond until it is.
__device__ __forceinline__ bool mbar_doze(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(1000u)
        : "memory");
    return ok != 0;
}
// A place in a ring of buffers and the parity of its present round.
template <int kBuffers>
struct Ring {
    int at = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next() {
        if (++at == kBuffers) at = 0, parity ^= 1;
    }
};
// One lane of the warp, where all are together.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

// 2^x, 0 for -infinity (the hardware's exponential, 2 units in the last place).
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The parts of a pair, packed (x in the low half).  BF16: each part cuts the
// next 8 bits off, and three hold the value exactly.
__device__ __forceinline__ void split_parts(float x, float y, uint32_t (&part)[3]) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
        part[i] = __byte_perm(a, b, 0x7632);
        x -= __uint_as_float(a & 0xffff0000u);
        y -= __uint_as_float(b & 0xffff0000u);
    }
}
__device__ __forceinline__ void split_parts(float x, float y, uint32_t (&part)[2]) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    part[0] = *reinterpret_cast<const uint32_t *>(&h);
    part[1] = *reinterpret_cast<const uint32_t *>(&l);
}

// Adds one; releases what the block wrote before (behind a barrier), acquires
// what others released here.
__device__ __forceinline__ unsigned arrive_gpu(unsigned *count) {
    unsigned before;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(count) : "memory");
    return before;
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
// Waits for loads; what they loaded counts as written here, so that nothing
// uses it before.
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint32_t (&r)[4]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3])
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

// a / b for a >= 0, b > 0: mostly of small numbers, where 32 bits do.
__device__ __forceinline__ long long divide(long long a, long long b) {
    return a <= 0xffffffffll ? (long long)((uint32_t)a / (uint32_t)min(b, 0xffffffffll)) : a / b;
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
    int rows, block_rows, blocks, reach;
    uint32_t first;
    long long start;

    __device__ __forceinline__ void open(const TreeGqaArgs &a, uint32_t s) {
        seq = s;
        // (All loads before the first use of one.)
        const long long length = a.lengths[s];
        const int64_t slot = a.pt.slot_ids ? a.pt.slot_ids[s] : (int64_t)s;
        int32_t o0 = 0, o1 = 0;
        if (a.offsets) o0 = a.offsets[s], o1 = a.offsets[s + 1];
        if (a.offsets) {
            const SequenceRows own = rows_between(o0, o1, a.tokens);
            first = (uint32_t)own.first, rows = (int)own.n;
        } else {
            first = s;
            rows = s < a.tokens;
        }
        reach = slot < 0 || slot >= (int64_t)a.pt.slots ? 0 : (int)max(0ll, min(length, (long long)a.pt.max_pages * a.pt.page_tokens));
        start = length - rows;
        blocks = (rows + (int)a.block_nodes - 1) / (int)a.block_nodes;
        block_rows = blocks ? (rows + blocks - 1) / blocks : 1;
    }
    // The tokens that block b sees, and its tiles.
    __device__ __forceinline__ long long tokens_of(const TreeGqaArgs &a, uint32_t b) const {
        if (a.parents) return reach;
        return min((long long)reach, start + min((long long)rows, (long long)(b + 1) * block_rows));
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
        for (uint64_t e = thread; e < none * width; e += kThreads) a.out[(uint64_t)c.first * width + e] = 0.0f;
    }
}

// The rows of an item: nodes (rows of the sequence) times query heads.
struct Block {
    uint32_t head, heads, node0, kvh;  // head: the first, of the KV head's
    int rows, copies, span;            // span: rows from one copy to the next
    // The row of q and out (of head_dim values) of row r.
    template <typename C>
    __device__ __forceinline__ uint64_t query(const TreeGqaArgs &a, const C &c, int r) const {
        return (uint64_t)(c.first + node0 + r / heads) * a.q_heads + kvh * (a.q_heads / a.kv_heads) + head + r % heads;
    }
};
template <int kTile>
__device__ __forceinline__ Block block_of(const TreeGqaArgs &a, const TreeCursor<kTile> &c) {
    Block b;
    b.kvh = c.inner / a.head_blocks, b.head = c.inner % a.head_blocks * a.block_heads;
    b.heads = min(a.block_heads, a.q_heads / a.kv_heads - b.head), b.node0 = c.block * c.block_rows;
    b.rows = (int)((min((uint32_t)c.rows, b.node0 + c.block_rows) - b.node0) * b.heads);
    b.copies = b.rows <= 64 && kTile == 64 ? 2 : 1;
    b.span = kTgRows / b.copies;
    return b;
}

// What the tensor core cuts off a score, relative to it.  Each of its steps (16
// dimensions) cuts the sum so far: half a last place is 0.43e-7 of it on the average
// (over mantissas), and a score that matters, a sum of mostly one sign, grows evenly
// over its n steps: 0.43e-7 (n + 1) / 2.  Measured (scores of 4 to 40, 4,096 each): F32
// and F16 pages 1.0e-7 to 1.2e-7 with heads of 64, 1.7e-7 to 1.9e-7 with 128; BF16
// pages, whose products have 16 bits, two thirds.  The scale holds as much more; in
// two parts, since F32's own step is 0.6e-7 to 1.2e-7 of it.  (A score of a single
// product is not cut, and comes out up to 1.9e-7 too large.)
inline double score_cut(uint32_t head_dim, bool bf16) {
    return 0.43e-7 * ((head_dim + 15) / 16 + 1) / 2 * (bf16 ? 2.0 / 3.0 : 1.0);
}

template <typename T, int D>
__global__ void __launch_bounds__(TreeShape<T, D>::kThreads, 1) tree_gqa_kernel(
    const __grid_constant__ TreeMaps maps, const TreeGqaArgs a) {
    using S = TreeShape<T, D>;
    using Cursor = TreeCursor<S::kTile>;
    constexpr int kTile = S::kTile, kWarps = S::kThreads / 32, kMmaWarp = S::kMmaWarp;
    extern __shared__ uint8_t smem_raw[];
    // A cursor for each softmax group and other warp, and the loads' second; the
    // first is where the run begins.  (In shared memory: registers are for the sums.)
    __shared__ Cursor s_use[S::kGroups + kWarps - S::kSoftmax + S::kLoads];
    __shared__ long long s_run[3];                 // the run's first place and length; all places
    __shared__ uint64_t s_seen[16];                       // a bit for each token of a tile that exists (no load is 16 tiles ahead)
    __shared__ float s_scale[kTgRows];                    // what a row's scores are multiplied by (F16)
    constexpr int kTurns = S::kF32 && D == 128 ? 1 : 2;   // (no room for two)
    __shared__ __align__(16) float s_half[kTurns][S::kGroups][2][kTgRows];  // a thread's maximum of a tile, or sum, for the row's other thread
    __shared__ volatile int s_fail;
    __shared__ unsigned s_last;
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t *gbase = smem_raw + (base - raw);
    const uint32_t stages0 = base + S::kStageAt, raw0 = base + S::kRawAt, bars = base + S::kBarAt;
    auto s_full = [&](int b) { return bars + 8u * b; };
    auto p_full = [&](int b) { return bars + 8u * (3 + b); };
    auto o_full = [&](int b) { return bars + 8u * (5 + b); };
    auto raw_full = [&](int s) { return bars + 8u * (12 + s); };
    auto raw_empty = [&](int s) { return bars + 8u * (16 + s); };
    auto s_free = [&](int b) { return bars + 8u * (20 + b); };
    // Of K and V (v: 0, 1) of a stage: K is free when its scores are, V later.
    auto kv_full = [&](int v, int s) { return bars + 8u * (23 + v * S::kStages + s); };
    auto kv_empty = [&](int v, int s) { return bars + 8u * (23 + (2 + v) * S::kStages + s); };
    const uint32_t q_full = bars + 8u * 7, end_bar = bars + 8u * 11, tmem_slot = bars + 8u * (23 + 4 * S::kStages);

    long long *s_scan = reinterpret_cast<long long *>(s_half);  // [kWarps], for the list alone
    Cursor &s_start = s_use[0];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int b = 0; b < 2; ++b) {
            mbar_init(p_full(b), 8);
            mbar_init(o_full(b), 1);
        }
        for (int b = 0; b < S::kSBufs; ++b) {
            mbar_init(s_full(b), 1);
            mbar_init(s_free(b), 8);
        }
        mbar_init(end_bar, 2);
        mbar_init(q_full, S::kSoftmax);
        for (int s = 0; s < S::kRaw; ++s) {
            mbar_init(raw_full(s), 1);
            mbar_init(raw_empty(s), S::kHelpers);
        }
        for (int v = 0; v < 2; ++v)
            for (int s = 0; s < S::kStages; ++s) {
                mbar_init(kv_full(v, s), S::kF32 ? S::kHelpers : 1);  // (the splitting warps or the loading one)
                mbar_init(kv_empty(v, s), 1);
            }
        mbar_init_fence();
        s_fail = a.tries == 0;  // (as if a wait had run out already)
    }
    if (warp == kMmaWarp) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    if (tid == 32 * S::kLoadWarp) {
        for (int i = 0; i < 2; ++i) tma_prefetch_map(&maps.runs[i]), tma_prefetch_map(&maps.rows[i]);
    }
    pdl_wait();
    pdl_trigger();

    // The list: places before each thread's sequences, and their total.
    const uint32_t inners = a.kv_heads * a.head_blocks, sequences = a.pt.sequences;
    const uint32_t per = (sequences + S::kThreads - 1) / S::kThreads;
    const uint32_t seq0 = min(sequences, tid * per), seq1 = min(sequences, seq0 + per);
    long long mine = 0;
    Cursor c;
    for (uint32_t s = seq0; s < seq1; ++s) {
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
    const int listing = per > 1 ? kWarps : (int)(sequences + 31) / 32;  // warps that have sequences
    for (int w = 0; w < listing; ++w) {
        if (w < warp) before += s_scan[w];
        total += s_scan[w];
    }
    const long long ctas = min((long long)gridDim.x, total);
    const bool idle = (long long)blockIdx.x >= ctas;
    long long first = 0, end = 0;
    if (!idle && total * (blockIdx.x + 1) <= 0xffffffffll)
        first = (uint32_t)total * blockIdx.x / (uint32_t)ctas, end = (uint32_t)total * (blockIdx.x + 1) / (uint32_t)ctas;
    else if (!idle)
        first = total * blockIdx.x / ctas, end = total * (blockIdx.x + 1) / ctas;
    if (!idle && first >= before && first < before + mine) {
        long long left = first - before;
        c.unit = c.units = 0, c.block = c.inner = 0, c.at = 0;
        for (uint32_t s = seq0;; ++s) {  // (bounded whatever another stream does to the lengths)
            if (per > 1) c.open(a, s);
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
        c.inner = (uint32_t)min(divide(left, c.units + 1), (long long)inners - 1);
        const long long place = left - (long long)c.inner * (c.units + 1);
        c.unit = (int)max(place - 1, 0ll), c.at = place == 0;
        s_start = c;
    }
    if (tid == 0) s_run[0] = first, s_run[1] = end - first, s_run[2] = total;
    __syncthreads();
    const long long &count = s_run[1];  // places
    Cursor &use = s_use[warp < S::kSoftmax ? warp / 8 : S::kGroups + warp - S::kSoftmax];
    if (!idle && lane == 0 && (warp >= S::kSoftmax || warp % 8 == 0) && &use != &s_start) use = s_start;
    if (!idle && lane == 0 && warp >= S::kLoadWarp && warp < S::kHelperWarp)
        s_use[S::kGroups + kWarps - S::kLoadWarp + warp - S::kLoadWarp] = s_start;
    __syncthreads();
    // To the item after the next `tiles` tiles, or as many tiles on in this one.
    auto skip = [&](Cursor &c, int tiles) {
        __syncwarp();
        if (lane == 0) {
            c.unit += tiles - 1, c.at += tiles - 1;
            c.next(a, inners);
        }
        __syncwarp();
    };
    // Tiles of the item at the cursor that are left in this run.
    auto left = [&](const Cursor &c) { return (int)min((long long)(c.units - c.unit), count - c.at); };
    // A wait gives up after a.tries tries and one (2^22 take 0.1 to 4 seconds; a tile
    // takes microseconds), or when another has; false then.  Loads and products end at once,
    // so that none is begun over another; the other warps go through their items all
    // the same (every thread reaches every barrier, every run arrives at its joins),
    // and what is written from then on is NaN.
    auto wait = [&](uint32_t bar, uint32_t parity) {
        if (mbar_test(bar, parity)) return true;
        for (uint32_t i = 0; !mbar_doze(bar, parity); ++i)
            if (s_fail || i >= a.tries) {
                s_fail = 1;
                return false;
            }
        return true;
    };
    // The wait for what this block has under way, before it ends.
    auto drain = [&](uint32_t bar, uint32_t parity) {
        const bool done = mbar_wait(bar, parity);
        if (!done) s_fail = 1;
        return done;
    };

    // Splits an item's queries into the parts of Q, each softmax thread 8 values of a
    // row at a time, copies and all.
    auto split_queries = [&](const Block &blk) {
        constexpr int kChunks = D / 8, kRowsAtOnce = 32 * S::kSoftmax / kChunks, kBatch = S::kF32 && D == 64 ? 4 : 2;
        const int chunk = tid % kChunks, sub = tid / kChunks;
        const float *q0 = a.q + blk.query(a, use, 0) * a.head_dim + chunk * 8;
        const uint64_t node_pitch = (uint64_t)a.q_heads * a.head_dim;
        uint32_t node = sub / blk.heads, head = sub % blk.heads;  // of the row, from the block's first
#pragma unroll 1
        for (int r0 = 0; r0 < kTgRows; r0 += kBatch * kRowsAtOnce) {
            float4 x[kBatch], y[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int own = (r0 + k * kRowsAtOnce + sub) & (blk.span - 1);
                if (own == sub) node = sub / blk.heads, head = sub % blk.heads;  // (the next copy)
                x[k] = y[k] = make_float4(0, 0, 0, 0);
                if (own < blk.rows && (uint32_t)chunk * 8 < a.head_dim) {
                    const float *q = q0 + node * node_pitch + (uint64_t)head * a.head_dim;
                    x[k] = *reinterpret_cast<const float4 *>(q), y[k] = *reinterpret_cast<const float4 *>(q + 4);
                }
                for (head += kRowsAtOnce; head >= blk.heads; head -= blk.heads) ++node;
            }
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int row = r0 + k * kRowsAtOnce + sub;
                float up = a.scale, up_low = a.scale_low;
                if constexpr (S::kHalf) {
                    float most = fmaxf(fmaxf(fmaxf(fabsf(x[k].x), fabsf(x[k].y)), fmaxf(fabsf(x[k].z), fabsf(x[k].w))),
                                       fmaxf(fmaxf(fabsf(y[k].x), fabsf(y[k].y)), fmaxf(fabsf(y[k].z), fabsf(y[k].w))));
#pragma unroll
                    for (int o = 1; o < kChunks; o *= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                    most *= a.scale;
                    float down = 1.0f;
                    if (most > 0.0f && most < INFINITY) {
                        const int e = min(max(14 - ilogbf(most), -100), 100);
                        up = ldexpf(a.scale, e), up_low = ldexpf(a.scale_low, e), down = ldexpf(1.0f, -e);
                    }
                    if (chunk == 0) s_scale[row] = down;
                }
                uint32_t w0[S::kQParts], w1[S::kQParts], w2[S::kQParts], w3[S::kQParts];
                auto scaled = [&](float v) { return fmaf(v, up, v * up_low); };
                split_parts(scaled(x[k].x), scaled(x[k].y), w0), split_parts(scaled(x[k].z), scaled(x[k].w), w1);
                split_parts(scaled(y[k].x), scaled(y[k].y), w2), split_parts(scaled(y[k].z), scaled(y[k].w), w3);
                uint8_t *to = gbase + chunk / 8 * (kTgRows * 128) + row * 128 + ((chunk % 8 ^ (row & 7)) << 4);
#pragma unroll
                for (int p = 0; p < S::kQParts; ++p)
                    *reinterpret_cast<uint4 *>(to + p * S::kQPart) = make_uint4(w0[p], w1[p], w2[p], w3[p]);
            }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
    };

    if (warp >= S::kSoftmax) {
        if constexpr (S::kMoreRegs) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kOtherRegs));
        if (warp >= S::kLoadWarp && warp < S::kHelperWarp) {
            // ---------------------------------------------------------- loads
            if (!idle) {
                // A tile's tokens lie in runs of a.run rows of a page.  The lanes look up the
                // runs of several tiles at once (`batch` of them), a batch ahead; a tile whose
                // tokens all exist is loaded run by run, any other in gathers of four rows,
                // where a token that does not exist has the row past the last: zeros.
                const uint32_t none = (uint32_t)a.pt.pages * a.kv_heads * a.pt.page_tokens;
                const int runs = a.run >= 4 ? kTile / (int)a.run : 32, batch = a.run >= 4 ? 32 / runs : 1;
                auto row_of = [&](const Cursor &c, long long pos) -> uint32_t {
                    const uint32_t slot = a.pt.slot_ids ? (uint32_t)a.pt.slot_ids[c.seq] : c.seq;
                    const uint32_t p = a.page_magic ? __umulhi((uint32_t)pos, a.page_magic) >> a.page_shift : (uint32_t)pos;
                    const int page = a.pt.table[(uint64_t)slot * a.pt.max_pages + p];
                    if (page < 0 || (uint64_t)page >= a.pt.pages) return none;
                    return ((uint32_t)page * a.kv_heads + c.inner / a.head_blocks) * a.pt.page_tokens + ((uint32_t)pos - p * a.pt.page_tokens);
                };
                // This lane's run of the batch at the cursor (tile: lane / runs).
                auto find = [&](const Cursor &c) -> uint32_t {
                    if (a.run < 4 || c.at >= count || lane / runs >= left(c)) return none;
                    const long long pos = (long long)(c.units - 1 - c.unit - lane / runs) * kTile + lane % runs * a.run;
                    return pos + a.run <= c.tokens_of(a, c.block) ? row_of(c, pos) : none;
                };
                const int kind = warp - S::kLoadWarp;  // K or V, where each has a warp
                Cursor &look = s_use[S::kGroups + kWarps - S::kSoftmax + kind];
                uint32_t ahead = find(look);
                Ring<S::kStages> ring;
                Ring<S::kRaw ? S::kRaw : 1> raw_ring;
                uint32_t rounds = 0, raw_rounds = 0, tile = 0;  // (rounds: loads so far, up to the ring's size)
                bool failed = false;  // (a wait was: nothing more is loaded)
                while (use.at < count && !failed) {
                    const int n = min(batch, left(use));
                    const uint32_t now = ahead;
                    const long long to = use.tokens_of(a, use.block);
                    for (int i = 0; i < n; ++i) {
                        const uint32_t here = __ballot_sync(0xffffffffu, now != none) >> (i * runs % 32);
                        const uint32_t want = runs == 32 ? 0xffffffffu : (1u << runs) - 1;
                        const bool whole = a.run >= 4 && (here & want) == want;
                        // (Otherwise: the rows of tokens `lane` and, of 64, lane + 32.)
                        uint32_t row[2] = {none, none};
                        uint64_t seen = kTile == 64 ? ~0ull : 0xffffffffull;
                        if (!whole) {
                            seen = 0;
#pragma unroll
                            for (int k = 0; k < kTile / 32; ++k) {
                                const long long pos = (long long)(use.units - 1 - use.unit - i) * kTile + 32 * k + lane;
                                if (pos < to) row[k] = row_of(use, pos);
                                seen |= (uint64_t)__ballot_sync(0xffffffffu, row[k] != none) << (32 * k);
                            }
                        }
                        const int stage = ring.at;
                        constexpr uint32_t kRowBytes = S::kF32 ? D * 4 : 128, kBytes = S::kF32 ? S::kRawSlot : S::kKvPart;
#pragma unroll
                        for (int w = 0; w < 2 / S::kLoads; ++w) {
                            const int v = S::kLoads == 2 ? kind : w;
                            uint32_t dst = stages0 + stage * S::kStage + v * S::kKvPart, bar = kv_full(v, stage);
                            if constexpr (S::kF32) {
                                dst = raw0 + raw_ring.at * S::kRawSlot, bar = raw_full(raw_ring.at);
                                if (raw_rounds >= S::kRaw) wait(raw_empty(raw_ring.at), raw_ring.parity ^ 1);
                            } else if (rounds >= S::kStages) {
                                wait(kv_empty(v, stage), ring.parity ^ 1);
                            }
                            failed = __any_sync(0xffffffffu, s_fail);
                            if (failed) break;
                            if constexpr (S::kF32) {
                                raw_rounds = min(raw_rounds + 1, (uint32_t)S::kRaw);
                                raw_ring.next();
                            }
                            // (No load is 16 tiles ahead of the softmax: V waits for its stage, or raw rows
                            // for theirs.)
                            if (lane == 0) {
                                if (v == 1 || S::kF32) s_seen[tile & 15] = seen;
                                mbar_arrive_expect_tx(bar, kBytes);
                            }
                            __syncwarp();
                            if (whole) {
                                for (int r0 = 0; r0 < runs; r0 += 4) {
                                    uint32_t from[4];
#pragma unroll
                                    for (int k = 0; k < 4; ++k) from[k] = __shfl_sync(0xffffffffu, now, (i * runs + r0 + k) % 32);
                                    if (elect_one()) {
#pragma unroll
                                        for (int k = 0; k < 4; ++k)
                                            if (r0 + k < runs)
#pragma unroll
                                                for (int x = 0; x < (S::kF32 ? 1 : D / 64); ++x)
                                                    tile_load(dst + x * kTile * 128 + (r0 + k) * a.run * kRowBytes, &maps.runs[v], x * 64, from[k], bar);
                                    }
                                    __syncwarp();
                                }
                            } else {
                                const int quad = lane % (kTile / 4);
                                uint32_t from[4];
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    const uint32_t low = __shfl_sync(0xffffffffu, row[0], (4 * quad + k) % 32);
                                    const uint32_t high = __shfl_sync(0xffffffffu, row[1], (4 * quad + k) % 32);
                                    from[k] = quad < 8 ? low : high;
                                }
#pragma unroll
                                for (int x = 0; x < (S::kF32 ? 1 : D / 64); ++x)
                                    if (lane < kTile / 4) gather4(dst + x * kTile * 128 + quad * 4 * kRowBytes, &maps.rows[v], x * 64, from, bar);
                            }
                        }
                        if (failed) break;
                        rounds = min(rounds + 1, (uint32_t)S::kStages);
                        ring.next();
                        ++tile;
                        if (i == 0) {
                            skip(look, n);
                            ahead = find(look);
                        }
                    }
                    skip(use, n);
                }
                // Every load has arrived when the block ends, or a wait of 2 s has been for nothing.
                bool arrived = true;
                if constexpr (!S::kF32) {
                    for (uint32_t i = 0; i < S::kStages && arrived; ++i, ring.next())
                        if (i + rounds >= S::kStages) arrived = drain(kv_full(kind, ring.at), ring.parity ^ 1);
                } else {
                    for (uint32_t i = 0; i < S::kRaw && arrived; ++i, raw_ring.next())
                        if (i + raw_rounds >= S::kRaw) arrived = drain(raw_full(raw_ring.at), raw_ring.parity ^ 1);
                }
                __syncwarp();
            }
            zero_rows<kTile, 32 * S::kLoads>(a, tid - 32 * S::kLoadWarp);
        } else if (!idle && warp >= S::kHelperWarp && warp < kMmaWarp) {
            // ---------------------------------------------------------- parts
            if constexpr (S::kF32) {
                constexpr int kLt = 32 * S::kHelpers, kChunks = D / 8, kRowsAtOnce = kLt / kChunks;
                const int lt = tid - 32 * S::kHelperWarp, chunk = lt % kChunks, sub = lt / kChunks;
                Ring<S::kStages> ring;
                Ring<S::kRaw> raw_ring;
                uint32_t rounds = 0;
                while (use.at < count) {
                    const int n = left(use);
                    for (int t = 0; t < n; ++t, ring.next()) {
                        const int stage = ring.at;
                        const bool again = rounds >= S::kStages;
                        if (!again) ++rounds;
#pragma unroll 1
                        for (int v = 0; v < 2; ++v, raw_ring.next()) {
                            const int slot = raw_ring.at;
                            if (again) wait(kv_empty(v, stage), ring.parity ^ 1);
                            wait(raw_full(slot), raw_ring.parity);
                            __syncwarp();
                            const uint8_t *from = gbase + S::kRawAt + slot * S::kRawSlot + chunk * 32;
                            uint8_t *to = gbase + S::kStageAt + stage * S::kStage + v * 3 * S::kKvPart + chunk / 8 * (kTile * 128);
#pragma unroll 4
                            for (int r0 = 0; r0 < kTile; r0 += kRowsAtOnce) {
                                const int row = r0 + sub;
                                const float4 x = *reinterpret_cast<const float4 *>(from + row * D * 4);
                                const float4 y = *reinterpret_cast<const float4 *>(from + row * D * 4 + 16);
                                uint32_t w0[3], w1[3], w2[3], w3[3];
                                split_parts(x.x, x.y, w0), split_parts(x.z, x.w, w1);
                                split_parts(y.x, y.y, w2), split_parts(y.z, y.w, w3);
#pragma unroll
                                for (int p = 0; p < 3; ++p)
                                    *reinterpret_cast<uint4 *>(to + p * S::kKvPart + row * 128 + ((chunk % 8 ^ (row & 7)) << 4)) =
                                        make_uint4(w0[p], w1[p], w2[p], w3[p]);
                            }
                            fence_async_smem();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(raw_empty(slot)), mbar_arrive(kv_full(v, stage));
                        }
                    }
                    skip(use, n);
                }
            }
        } else if (!idle && warp == kMmaWarp) {
            // ---------------------------------------------------------- scores
            // The whole warp goes through it, so that addresses stay in uniform
            // registers; one lane issues.
            constexpr uint32_t kIdesc = idesc<S::kHalf>(kTgRows, kTile, false);
            Ring<S::kStages> ring;
            Ring<S::kSBufs> s_ring;
            Ring<1> q_ring;
            int rounds = 0;
            bool ok = true;
            for (; ok && use.at < count; q_ring.next()) {
                const int n = left(use);
                // (Descriptors hold addresses in units of 16 bytes in their low bits.)
                const uint64_t q = sw128_kmajor_desc(base);
                ok = wait(q_full, q_ring.parity);
                for (int t = 0; t < n; ++t, ring.next(), s_ring.next()) {
                    if (rounds >= S::kSBufs) ok = wait(s_free(s_ring.at), s_ring.parity ^ 1) && ok;
                    else ++rounds;
                    ok = wait(kv_full(0, ring.at), ring.parity) && ok;
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after_sync();
                    const uint64_t k = sw128_kmajor_desc(stages0 + ring.at * S::kStage);
                    const uint32_t to = tmem + s_ring.at * kTile;
                    if (elect_one()) {
#pragma unroll
                        for (int i = 0; i < S::kPairs; ++i)
#pragma unroll
                            for (int kk = 0; kk < D / 16; ++kk)
                                mma_bf16_ss(to, q + (pair_q<T, D>(i) * S::kQPart + kk / 4 * (kTgRows * 128) + kk % 4 * 32) / 16,
                                            k + (pair_kv<T, D>(i) * S::kKvPart + kk / 4 * (kTile * 128) + kk % 4 * 32) / 16, kIdesc,
                                            (i | kk) != 0);
                        mma_commit(s_full(s_ring.at));
                        mma_commit(kv_empty(0, ring.at));
                    }
                    __syncwarp();
                }
                skip(use, n);
            }
            // Nothing is under way when the tensor memory goes back (or a wait of 2 s has been
            // for nothing).  The lane that issued the products commits them.
            if (elect_one()) mma_commit(end_bar);
            drain(end_bar, 0);
            __syncwarp();
        } else if (!idle && warp == kMmaWarp + 1) {
            // ---------------------------------------------------------- weighted values
            constexpr uint32_t kIdesc = idesc<S::kHalf>(kTgRows, D, true);
            Ring<S::kStages> ring;
            uint32_t p_round = 0, tile = 0;
            bool ok = true;
            while (ok && use.at < count) {
                const int n = left(use);
                for (int t = 0; t < n; ++t, ++tile, ring.next()) {
                    const int b = tile & 1;
                    ok = wait(kv_full(1, ring.at), ring.parity) && wait(p_full(b), p_round >> b & 1);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    p_round ^= 1u << b;
                    tc_fence_after_sync();
                    const uint64_t v = sw128_mnmajor_desc(stages0 + ring.at * S::kStage + S::kKvParts * S::kKvPart, kTile * 128);
                    const uint32_t p = tmem + S::kPCol + b * S::kPBuf, to = tmem + S::kOCol + (S::kGroups == 2 ? b * D : 0);
                    if (elect_one()) {
#pragma unroll
                        for (int i = 0; i < S::kPairs; ++i)
#pragma unroll
                            for (int kk = 0; kk < kTile / 16; ++kk)
                                mma_bf16_ts(to, p + pair_q<T, D>(i) * (kTile / 2) + kk * 8,
                                            v + (pair_kv<T, D>(i) * S::kKvPart + kk * 2048) / 16, kIdesc, (i | kk) != 0);
                        mma_commit(o_full(b));
                        mma_commit(kv_empty(1, ring.at));
                    }
                    __syncwarp();
                }
                skip(use, n);
            }
            if (elect_one()) mma_commit(end_bar);
            drain(end_bar, 0);
            __syncwarp();
        }
    } else if (!idle) {
        // ---------------------------------------------------------- softmax
        if constexpr (S::kMoreRegs) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kSoftmaxRegs));
        // (group, half, row): the group's tiles, this thread's half of tokens and
        // dimensions, its TMEM lane.
        constexpr int kOwn = D / 2, kMost = kTile / 32;  // dimensions; chunks of 16 tokens at most
        const int wg = warp / 8, half = warp >> 2 & 1, row = 32 * (warp & 3) + lane;
        const uint32_t quarter = (uint32_t)(32 * (warp & 3)) << 16, pair = 4 + wg * 4 + (warp & 3);
        uint32_t tile = 0;  // of the run: its parity is the buffer of P and O
        Ring<S::kSBufs> s_ring;
        Ring<S::kStages> ring;
        Ring<1> q_ring;
        uint32_t o_round = 0;  // a bit for each buffer: the parity of its next round
        int copies_before = 1;
        float *join = reinterpret_cast<float *>(gbase + S::kJoinAt);
        // The other thread's value for `mine`.
        int turn = 0;
        auto exchange = [&](float mine) {
            // (The other thread may still read what it got last.)
            if (kTurns == 1) named_barrier(pair, 64);
            else turn ^= 1;
            s_half[turn][wg][half][row] = mine;
            named_barrier(pair, 64);
            return s_half[turn][wg][half ^ 1][row];
        };
        for (; use.at < count; q_ring.next()) {
            // The item: its rows, copies of them, this thread's row.
            int copies, copy, node;
            bool active;
            {
                const Block blk = block_of(a, use);
                const int mine_row = row % blk.span;
                copies = blk.copies, copy = row / blk.span, active = mine_row < blk.rows;
                node = (int)blk.node0 + mine_row / (int)blk.heads;
            }
            const bool warp_active = __any_sync(0xffffffffu, active);
            named_barrier(1, 32 * S::kSoftmax);  // (all products of the Q before are done)
            split_queries(block_of(a, use));
            // A copy's weights are zero for the other copy's tokens, from here on.
            if (copies != copies_before && copies > 1) {
                const uint32_t zeros[8] = {};
                for (uint32_t c = 8 * half; c < S::kPBuf; c += 16)
#pragma unroll
                    for (int b = 0; b < 2; ++b)
                        if (S::kGroups == 1 || b == wg) tmem_st8(tmem + quarter + S::kPCol + b * S::kPBuf + c, zeros);
                tmem_wait_st();
                named_barrier(pair, 64);  // (both halves' zeros are there before either's weights)
            }
            copies_before = copies;
            float unit_scale = 1.0f;
            if constexpr (S::kHalf) {
                wait(q_full, q_ring.parity);
                __syncwarp();
                unit_scale = s_scale[row];
            }
            float m = -INFINITY, l = 0.0f, o[kOwn], keep_last = 0.0f;
#pragma unroll
            for (int i = 0; i < kOwn; ++i) o[i] = 0.0f;
            int last = -1;  // the buffer of O that has not been added
            auto add = [&]() {
                const int b = last;
                wait(o_full(b), o_round >> b & 1);
                o_round ^= 1u << b;
                __syncwarp();
                tc_fence_after_sync();
                const uint32_t from = tmem + quarter + S::kOCol + (S::kGroups == 2 ? b * D : 0) + half * kOwn;
#pragma unroll
                for (int c = 0; c < kOwn; c += 32) {
                    uint32_t x[2][16];
                    tmem_ld(from + c, x[0]);
                    tmem_ld(from + c + 16, x[1]);
                    tmem_wait_ld(x[0]);
                    tmem_wait_ld(x[1]);
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[c + i] = fmaf(o[c + i], keep_last, __uint_as_float(x[i / 16][i % 16]));
                }
            };
            int ancestor = active ? node : -1;  // the next to be met
            const int n = left(use);
            const int chunks = kMost / copies, c0 = (copy * 2 + half) * 16 * chunks;  // this thread's columns
            long long low = (long long)(use.units - 1 - use.unit) * kTile - use.start;  // the row that the tile's first token is
            for (int i = 0; i < n; ++i, ++tile, ring.next(), s_ring.next(), low -= kTile) {
                const int b = tile & 1;
                if (S::kGroups == 2 && b != wg) continue;  // (the other group's)
                wait(s_full(s_ring.at), s_ring.parity);
                wait(kv_full(1, ring.at), ring.parity);  // (for s_seen)
                __syncwarp();
                tc_fence_after_sync();
                if (!warp_active) {
                    // (Keeps step: its arrival counts, and must not come before the others' for
                    // the tile before.)
                    if (last >= 0) wait(o_full(last), o_round >> last & 1), o_round ^= 1u << last;
                    last = b;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s_free(s_ring.at)), mbar_arrive(p_full(b));
                    continue;
                }
                const uint32_t from = tmem + quarter + s_ring.at * kTile + c0;
                // Which of the tokens this row sees.
                uint64_t seen = *const_cast<const volatile uint64_t *>(&s_seen[tile & 15]);
                if (low > -kTile) {
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
                const uint32_t every = 0xffffffffu >> (32 - 16 * chunks);
                const uint32_t bits = active ? (uint32_t)(seen >> c0) & every : every;  // (nobody reads the others' rows)
                const bool all = __all_sync(0xffffffffu, bits == every);
                // What the row does not see has a score of -infinity.
                auto hide = [&](uint32_t (&x)[16], int c) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[j] = bits >> (16 * c + j) & 1 ? x[j] : 0xff800000u;
                };
                // (The scores are read twice: to keep them would cost the registers of the
                // sums, which then spill.)
                float most = -INFINITY;
#pragma unroll
                for (int c = 0; c < kMost; ++c)
                    if (c < chunks) {
                        uint32_t x[16];
                        tmem_ld(from + 16 * c, x);
                        tmem_wait_ld(x);
                        if (!all) hide(x, c);
#pragma unroll
                        for (int j = 0; j < 16; j += 2)
                            most = fmaxf(most, fmaxf(__uint_as_float(x[j]), __uint_as_float(x[j + 1])));
                    }
                most = fmaxf(most, exchange(most));
                if (S::kGroups == 2 && last >= 0) add();  // (its P buffer is free then)
                if constexpr (S::kHalf) most *= unit_scale;
                const float now = fmaxf(m, most), reference = now == -INFINITY ? 0.0f : now;
                const float keep = exp2_fast(m - reference), shift = S::kShift - reference;
                m = now;
                float sum[2] = {0.0f, 0.0f};
                const uint32_t to = tmem + quarter + S::kPCol + b * S::kPBuf + c0 / 2;
#pragma unroll
                for (int c = 0; c < kMost; ++c)
                    if (c < chunks) {
                        uint32_t x[16];
                        tmem_ld(from + 16 * c, x);
                        tmem_wait_ld(x);
                        if (!all) hide(x, c);
#pragma unroll
                        for (int j0 = 0; j0 < 16; j0 += 8) {
                            uint32_t part[S::kQParts][4];
#pragma unroll
                            for (int j = j0; j < j0 + 8; j += 2) {
                                const float s0 = __uint_as_float(x[j]), s1 = __uint_as_float(x[j + 1]);
                                const float p0 = exp2_fast(S::kHalf ? fmaf(s0, unit_scale, shift) : s0 + shift);
                                const float p1 = exp2_fast(S::kHalf ? fmaf(s1, unit_scale, shift) : s1 + shift);
                                sum[0] += p0, sum[1] += p1;
                                uint32_t w[S::kQParts];
                                split_parts(p0, p1, w);
#pragma unroll
                                for (int k = 0; k < S::kQParts; ++k) part[k][j / 2 % 4] = w[k];
                            }
#pragma unroll
                            for (int k = 0; k < S::kQParts; ++k) tmem_st4(to + k * (kTile / 2) + 8 * c + j0 / 2, part[k]);
                        }
                    }
                tmem_wait_st();
                if (S::kGroups == 1 && last >= 0) add();  // (O has one buffer)
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_free(s_ring.at)), mbar_arrive(p_full(b));
                l = fmaf(l, keep, sum[0] + sum[1]);
                keep_last = keep;
                last = b;
            }
            if (last >= 0) add();
            if (warp_active) l += exchange(l);

            const Block blk = block_of(a, use);
            const int unit0 = use.unit, mine_row = row % blk.span;
            const bool whole = unit0 + n == use.units;  // the item's last tile is this run's
            // Join: the other group, then the other copy.  Of two groups each ends
            // with half of this thread's dimensions, as of two copies.
            auto finish = [&](auto first_c) {
                constexpr int kFirst = decltype(first_c)::value, kKept = kOwn / S::kGroups;  // dimensions kept, of o
                auto meet = [&](bool both) {
                    if (S::kGroups == 2 && both) named_barrier(1, 512);
                    else named_barrier(2 + wg, 256);
                };
                float *own = join + ((wg * 2 + half) * kTgRows + row) * S::kPitch;
                auto put = [&](int d0) {
#pragma unroll
                    for (int i = 0; i < S::kCols; i += 4)
                        *reinterpret_cast<float4 *>(own + i) = make_float4(o[d0 + i], o[d0 + i + 1], o[d0 + i + 2], o[d0 + i + 3]);
                    *reinterpret_cast<float2 *>(own + S::kCols) = make_float2(m, l);
                };
                float now = m, f = 1.0f, g = 0.0f, sum = l;
                auto take = [&](const float *other, int d0, bool factors) {
                    if (factors) {
                        const float2 ml = *reinterpret_cast<const float2 *>(other + S::kCols);
                        now = fmaxf(m, ml.x);
                        const float reference = now == -INFINITY ? 0.0f : now;
                        f = exp2_fast(m - reference), g = exp2_fast(ml.x - reference), sum = fmaf(ml.y, g, l * f);
                    }
#pragma unroll
                    for (int i = 0; i < S::kCols; i += 4) {
                        const float4 v = *reinterpret_cast<const float4 *>(other + i);
                        o[d0 + i] = fmaf(v.x, g, o[d0 + i] * f), o[d0 + i + 1] = fmaf(v.y, g, o[d0 + i + 1] * f);
                        o[d0 + i + 2] = fmaf(v.z, g, o[d0 + i + 2] * f), o[d0 + i + 3] = fmaf(v.w, g, o[d0 + i + 3] * f);
                    }
                };
                if constexpr (S::kGroups == 2) {
#pragma unroll
                    for (int c = 0; c < kKept; c += S::kCols) {
                        meet(true);  // (what lay there has been read)
                        put(kKept - kFirst + c);
                        meet(true);
                        take(join + (((wg ^ 1) * 2 + half) * kTgRows + row) * S::kPitch, kFirst + c, c == 0);
                    }
                    m = now, l = sum;
                }
                if (S::kMostCopies > 1 && copies > 1) {
#pragma unroll
                    for (int c = 0; c < kKept; c += S::kCols) {
                        meet(c == 0);
                        if (copy) put(kFirst + c);
                        meet(false);
                        if (!copy) take(own + blk.span * S::kPitch, kFirst + c, c == 0);
                    }
                    m = now, l = sum;
                }
                const bool starts = unit0 == 0, writer = copy == 0 && active;
                const int d0 = half * kOwn + kFirst;
                if (!writer) return;
                if (starts && whole) {
                    float *to = a.out + blk.query(a, use, mine_row) * a.head_dim + d0;
                    const float inverse = s_fail ? NAN : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
                    for (int i = 0; i < kKept; i += 4)
                        if ((uint32_t)(d0 + i) < a.head_dim)
                            *reinterpret_cast<float4 *>(to + i) = make_float4(o[kFirst + i] * inverse, o[kFirst + i + 1] * inverse,
                                                                              o[kFirst + i + 2] * inverse, o[kFirst + i + 3] * inverse);
                    return;
                }
                // A run that starts the item writes slot 1 of its CTA, one that goes on with it slot 0.
                float *part = a.partial + (uint64_t)(2 * blockIdx.x + starts) * S::kPart;
#pragma unroll
                for (int i = 0; i < kKept; i += 4)
                    *reinterpret_cast<float4 *>(part + mine_row * D + d0 + i) =
                        make_float4(o[kFirst + i], o[kFirst + i + 1], o[kFirst + i + 2], o[kFirst + i + 3]);
                if (d0 == 0) part[kTgRows * D + mine_row] = m, part[kTgRows * (D + 1) + mine_row] = s_fail ? NAN : l;
            };
            if (S::kGroups == 2 && wg == 1) finish(std::integral_constant<int, S::kGroups == 2 ? kOwn / 2 : 0>{});
            else finish(std::integral_constant<int, 0>{});
            if (!(unit0 == 0 && whole)) {
                // The places [u0, u1) of the item's tiles and the CTAs that own its ends.
                const long long total = s_run[2], ctas = min((long long)gridDim.x, total);
                const long long u0 = s_run[0] + use.at - unit0, u1 = u0 + use.units;
                const int cta0 = (int)divide((u0 + 1) * ctas - 1, total), runs = (int)divide(u1 * ctas - 1, total) - cta0 + 1;
                named_barrier(1, 32 * S::kSoftmax);
                if (tid == 0) {
                    // The block's partial before its arrival, and the others' before what the
                    // block reads next.
                    s_last = arrive_gpu(&a.arrived[cta0]) + 1 == (unsigned)runs;
                    if (s_last) a.arrived[cta0] = 0;
                }
                named_barrier(1, 32 * S::kSoftmax);
                if (s_last) {
                    const float *partial = a.partial + (uint64_t)2 * cta0 * S::kPart;
                    auto slot = [&](int k) { return partial + (uint64_t)(k ? 2 * k : 1) * S::kPart; };
                    // Each row's maximum and sum over the runs, then what every run counts
                    // (kRuns of them at a time), then the values: two loads under way, eight
                    // where the loop over tiles has registers to spare (prompt chunks with
                    // heads of 128 98 -> 96 us; elsewhere its sums would be spilled).
                    constexpr bool kRoom = S::kGroups == 2 || S::kMostCopies == 2;  // for the weights, in the joins' memory
                    constexpr int kRuns = kRoom ? (int)S::kJoinBytes / (4 * kTgRows) : 2, kBatch = 2, kAtOnce = D == 128 && !S::kF32 ? 4 : 1;
                    float *weight = kRoom ? join : s_half[0][0][0];  // [kRuns][rows]; the runs' maxima first
                    float most = -INFINITY, sum = 0.0f;
                    if (tid < blk.rows) {
#pragma unroll 1
                        for (int k0 = 0; k0 < runs; k0 += 8) {
                            float2 ml[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                const float *from = slot(k0 + k) + kTgRows * D + tid;
                                ml[k] = k0 + k < runs ? make_float2(__ldcg(from), __ldcg(from + kTgRows)) : make_float2(-INFINITY, 0.0f);
                            }
                            float now = most;
#pragma unroll
                            for (int k = 0; k < 8; ++k) now = fmaxf(now, ml[k].x);
                            const float reference = now == -INFINITY ? 0.0f : now;
                            sum *= exp2_fast(most - reference);
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                sum = fmaf(ml[k].y, exp2_fast(ml[k].x - reference), sum);
                                if (k0 + k < min(runs, kRuns)) weight[(k0 + k) * kTgRows + tid] = ml[k].x;
                            }
                            most = now;
                        }
                        if (most == -INFINITY) most = 0.0f;
                        sum = sum == 0.0f ? 0.0f : 1.0f / sum;
                    }
                    for (int k0 = 0; k0 < runs; k0 += kRuns) {
                        const int some = min(runs - k0, kRuns);
                        if (k0) named_barrier(1, 32 * S::kSoftmax);
                        if (tid < blk.rows)
                            for (int k = 0; k < some; ++k) {
                                float *w = weight + k * kTgRows + tid;
                                *w = exp2_fast((k0 ? __ldcg(slot(k0 + k) + kTgRows * D + tid) : *w) - most) * sum;
                            }
                        named_barrier(1, 32 * S::kSoftmax);
#pragma unroll 1
                        for (int e0 = tid; e0 < blk.rows * (D / 4); e0 += kAtOnce * S::kSoftmax * 32) {
                            float4 acc[kAtOnce];
                            float4 *to[kAtOnce];
                            bool in[kAtOnce];
#pragma unroll
                            for (int u = 0; u < kAtOnce; ++u) {
                                const int e = e0 + u * S::kSoftmax * 32, r = e / (D / 4), d = e % (D / 4) * 4;
                                in[u] = r < blk.rows && (uint32_t)d < a.head_dim;
                                to[u] = reinterpret_cast<float4 *>(a.out + blk.query(a, use, r) * a.head_dim + d);
                                acc[u] = in[u] && k0 ? *to[u] : make_float4(0, 0, 0, 0);
                            }
#pragma unroll 1
                            for (int k1 = 0; k1 < some; k1 += kBatch) {
                                float4 v[kAtOnce][kBatch];
#pragma unroll
                                for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
                                    for (int k = 0; k < kBatch; ++k)
                                        if (in[u] && k1 + k < some)
                                            v[u][k] = __ldcg(reinterpret_cast<const float4 *>(slot(k0 + k1 + k) + (e0 + u * S::kSoftmax * 32) * 4));
#pragma unroll
                                for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
                                    for (int k = 0; k < kBatch; ++k)
                                        if (in[u] && k1 + k < some) {
                                            const float f = weight[(k1 + k) * kTgRows + (e0 + u * S::kSoftmax * 32) / (D / 4)];
                                            acc[u].x = fmaf(v[u][k].x, f, acc[u].x), acc[u].y = fmaf(v[u][k].y, f, acc[u].y);
                                            acc[u].z = fmaf(v[u][k].z, f, acc[u].z), acc[u].w = fmaf(v[u][k].w, f, acc[u].w);
                                        }
                            }
#pragma unroll
                            for (int u = 0; u < kAtOnce; ++u)
                                if (in[u]) *to[u] = acc[u];
                        }
                    }
                }
            }
            named_barrier(2 + wg, 256);
            if (warp % 8 == 0) skip(use, n);
            named_barrier(2 + wg, 256);
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
    if (tid == 0 && s_fail) atomicOr(&g_tree_fault, 1u);
}

// All rows of the pages, [rows][head_dim], to be loaded `box_rows` at a time:
// 16-bit rows in blocks of 64 values in the 128-byte swizzle, F32 rows whole.
// (No rows: one that is never read, since a map needs an address.)
template <typename T, int D>
int32_t rows_map(CUtensorMap *map, const void *pages, const TreeGqaArgs &a, uint32_t box_rows) {
    using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                  const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static EncodeFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *ptr = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeFn>(ptr);
    });
    if (!fn) return fail(MF_UNSUPPORTED, "driver entry point cuTensorMapEncodeTiled unavailable");
    constexpr bool kF32 = TreeShape<T, D>::kF32;
    const uint64_t rows = a.pt.max_pages ? a.pt.pages * a.kv_heads * a.pt.page_tokens : 0;
    const cuuint64_t dims[2] = {a.head_dim, std::max<uint64_t>(rows, 1)}, strides[1] = {a.head_dim * sizeof(T)};
    const cuuint32_t box[2] = {kF32 ? (cuuint32_t)D : 64u, box_rows}, step[2] = {1, 1};
    const CUresult r = fn(map,
                          kF32                          ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                          : TreeShape<T, D>::kHalf ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                        : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                          2, const_cast<void *>(rows ? pages : a.q), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          kF32 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(MF_BACKEND_FAILURE, "cuTensorMapEncodeTiled rejected the pages");
    return MF_OK;
}

template <typename T, int D>
int32_t tree_gqa_run(const TreeGqaArgs &a0, void *workspace, cudaStream_t stream) {
    using S = TreeShape<T, D>;
    TreeGqaArgs a = a0;
    a.arrived = static_cast<unsigned *>(workspace);
    a.partial = reinterpret_cast<float *>(static_cast<char *>(workspace) + 16384);
    // As many CTAs as the workspace has slots for, whatever the device.
    const int64_t slots = (MF_PAGED_TREE_WORKSPACE_BYTES - 16384) / (sizeof(float) * 2 * S::kPart);
    const int64_t grid = std::min({(int64_t)sm_count(), slots, (int64_t)4096});
    static std::atomic<uint64_t> ready{0};
    if (S::kMoreRegs && !ready.load(std::memory_order_relaxed)) {
        // (Warps that ask for more than the block was launched with would wait for good.)
        cudaFuncAttributes attr;
        MF_CUDA_TRY(cudaFuncGetAttributes(&attr, tree_gqa_kernel<T, D>));
        if (attr.numRegs * S::kThreads < S::kAllRegs) return fail(MF_UNSUPPORTED, "tree attention was built with too few registers");
    }
    if (int32_t st = allow_smem(tree_gqa_kernel<T, D>, S::kSmem, ready)) return st;
    const double scale = 1.4426950408889634 / std::sqrt((double)a.head_dim) * (1.0 + score_cut(a.head_dim, !S::kF32 && !S::kHalf));
    a.scale = (float)scale, a.scale_low = (float)(scale - a.scale);
    // The longest runs that no page cuts.
    a.run = S::kTile;
    while (a.pt.page_tokens % a.run) a.run /= 2;
    TreeMaps maps;
    for (int v = 0; v < 2; ++v) {
        if (int32_t st = rows_map<T, D>(&maps.runs[v], v ? a.values : a.keys, a, a.run)) return st;
        if (int32_t st = rows_map<T, D>(&maps.rows[v], v ? a.values : a.keys, a, 1)) return st;
    }
    return launch(tree_gqa_kernel<T, D>, dim3((unsigned)grid), dim3(S::kThreads), S::kSmem, stream, "tree_gqa_kernel", maps, a);
}

}  // namespace

int32_t paged_tree_gqa(float *out, const float *q, const void *key_pages, const void *value_pages, int32_t dtype,
                       const PagedTable &pt, uint64_t tokens, const int32_t *lengths, const int32_t *offsets,
                       const int32_t *parents, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, void *workspace,
                       cudaStream_t stream) {
    if (!pt.sequences || !tokens) return MF_OK;
    if (pt.pages * pt.page_tokens * kv_heads >= INT32_MAX)
        return fail(MF_OVERFLOW, "tree attention takes pools of less than 2^31 - 1 rows");
    TreeGqaArgs a;
    a.out = out, a.q = q, a.keys = key_pages, a.values = value_pages, a.pt = pt, a.tokens = tokens;
    a.lengths = lengths, a.offsets = offsets, a.parents = parents;
    a.tries = g_tree_tries.load(std::memory_order_relaxed);
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
