// A paged key/value cache of the handle tier: the pages' bookkeeping on the
// host, beside the pages, table and pass arrays on the device.
//
// A pass names sequences and how many tokens each appends.  mf_paged_begin
// reserves their pages (lowest free page first), copies the last page of a
// sequence that shares it, and sends the table's changes and the pass's arrays;
// each layer then writes its K and V rows and attends.  Everything is enqueued
// on the backend's stream in order, and every check runs before anything
// changes.
#include <cuda_runtime.h>
#include <string.h>

#include <algorithm>
#include <functional>
#include <new>
#include <queue>
#include <vector>

#include "backend_internal.h"
#include "mf_common.cuh"
#include "packed_kernels.h"

using namespace mf;

struct mf_paged_cache {
    mf_backend *b = nullptr;
    mf_paged_config cfg{};
    uint64_t page_bytes = 0;
    mf_buffer *pool = nullptr;    // [layers][K, V][pages] of page_bytes
    mf_buffer *arrays = nullptr;  // table [sequences][max_pages], then the pass's arrays
    mf_buffer *workspace = nullptr;
    std::vector<void *> pools;  // of each layer: K, V
    // Bookkeeping.
    std::vector<int32_t> table;
    std::vector<uint64_t> length;
    std::vector<uint32_t> refs;  // of each page
    std::priority_queue<uint32_t, std::vector<uint32_t>, std::greater<uint32_t>> free;
    // The pass.
    std::vector<int32_t> pass;  // slot ids [n], starts [n], lengths [n], row offsets [n + 1]
    uint64_t pass_n = 0, pass_rows = 0;
    bool in_pass = false;

    int32_t *device_table() const { return static_cast<int32_t *>(arrays->ptr); }
    int32_t *device_pass() const { return device_table() + table.size(); }
    uint64_t pages_of(uint64_t tokens) const { return (tokens + cfg.page_tokens - 1) / cfg.page_tokens; }
    int32_t &page(uint64_t seq, uint64_t nth) { return table[seq * cfg.max_pages + nth]; }
    PagedTable view() const {
        PagedTable pt;
        pt.table = device_table(), pt.slot_ids = device_pass(), pt.pages = cfg.pages;
        pt.slots = cfg.sequences, pt.max_pages = cfg.max_pages, pt.page_tokens = cfg.page_tokens;
        pt.sequences = (uint32_t)pass_n;
        return pt;
    }
    uint32_t take() {
        const uint32_t p = free.top();
        free.pop();
        refs[p] = 1;
        return p;
    }
    void drop(uint32_t p) {
        if (--refs[p] == 0) free.push(p);
    }
};

namespace {

int32_t check_cache(const mf_paged_cache *c) {
    if (!c) return fail(MF_INVALID_ARGUMENT, "null paged cache");
    return check_buffer(c->b, c->pool);
}

int32_t check_rows(const mf_paged_cache *c, const mf_buffer *buf, uint64_t rows, uint64_t width) {
    int32_t st = check_buffer(c->b, buf);
    if (st) return st;
    if (buf->dtype != MF_DTYPE_F32) return fail(MF_INVALID_DTYPE, "expected an f32 operand");
    if (buf->rank != 2 || buf->shape[0] != rows || buf->shape[1] != width)
        return fail(MF_INVALID_SHAPE, "paged operand differs from the pass's rows");
    return MF_OK;
}

// Sends the table's rows [first, last].
int32_t send_rows(mf_paged_cache *c, uint64_t first, uint64_t last) {
    const size_t row = c->cfg.max_pages;
    MF_CUDA_TRY(cudaMemcpyAsync(c->device_table() + first * row, c->table.data() + first * row,
                                (last - first + 1) * row * sizeof(int32_t), cudaMemcpyHostToDevice, c->b->stream));
    c->b->counts.copies++;
    return MF_OK;
}

int32_t copy_all(mf_paged_cache *c, const std::vector<uint32_t> &from, const std::vector<uint32_t> &to) {
    if (from.empty()) return MF_OK;
    return copy_pages(c->pools.data(), (uint32_t)c->pools.size(), c->page_bytes, from.data(), to.data(), from.size(),
                      c->b->stream);
}

}  // namespace

extern "C" {

int32_t mf_paged_create(mf_backend *b, const mf_paged_config *config, mf_paged_cache **out) {
    if (!b || !config || !out) return fail(MF_INVALID_ARGUMENT, "null argument");
    const mf_paged_config &f = *config;
    if (f.page_dtype < MF_PAGE_F32 || f.page_dtype > MF_PAGE_BF16) return fail(MF_INVALID_DTYPE, "unknown page dtype");
    if (!f.layers || !f.kv_heads || !f.head_dim || !f.page_tokens || !f.sequences || !f.max_pages || !f.pages)
        return fail(MF_INVALID_SHAPE, "paged cache sizes must be nonzero");
    if (f.head_dim % 8 || f.head_dim > 128)
        return fail(MF_UNSUPPORTED, "paged attention takes head dimensions of 8 to 128 in steps of 8");
    if (f.layers > 65536 || f.kv_heads > 65536 || f.page_tokens > (1u << 20) || f.sequences > (1u << 20) ||
        (uint64_t)f.max_pages * f.page_tokens > INT32_MAX || f.pages > INT32_MAX ||
        f.pages * f.page_tokens > (UINT32_MAX - 1) / f.kv_heads)
        return fail(MF_OVERFLOW, "paged cache geometry exceeds its limits");
    const uint64_t page_bytes =
        (uint64_t)f.kv_heads * f.page_tokens * f.head_dim * (f.page_dtype == MF_PAGE_F32 ? 4 : 2);
    const uint64_t words = (uint64_t)f.sequences * (f.max_pages + 4ull) + 1;
    if (words > INT32_MAX) return fail(MF_OVERFLOW, "paged cache geometry exceeds its limits");
    mf_paged_cache *c = new (std::nothrow) mf_paged_cache();
    if (!c) return fail(MF_RESOURCE_LIMIT, "host allocation failed");
    c->b = b, c->cfg = f, c->page_bytes = page_bytes;
    int32_t st = MF_OK;
    try {
        c->table.assign((size_t)f.sequences * f.max_pages, -1);
        c->length.assign(f.sequences, 0);
        c->refs.assign(f.pages, 0);
        std::vector<uint32_t> ids(f.pages);
        for (uint64_t p = 0; p < f.pages; ++p) ids[p] = (uint32_t)p;
        c->free = decltype(c->free)(std::greater<uint32_t>(), std::move(ids));
        c->pools.resize(2 * (size_t)f.layers);
        c->pass.reserve(4 * (size_t)f.sequences + 1);
    } catch (const std::bad_alloc &) {
        st = fail(MF_RESOURCE_LIMIT, "host allocation failed");
    }
    const uint64_t pool_shape[2] = {2ull * f.layers, f.pages * page_bytes}, array_shape[1] = {words * 4},
                   work_shape[1] = {MF_PAGED_WORKSPACE_BYTES};
    if (!st) st = backend_alloc_buffer(b, MF_DTYPE_U8, pool_shape, 2, MF_CLASS_CACHE, &c->pool);
    if (!st) st = backend_alloc_buffer(b, MF_DTYPE_U8, array_shape, 1, MF_CLASS_CACHE, &c->arrays);
    if (!st) st = backend_alloc_buffer(b, MF_DTYPE_U8, work_shape, 1, MF_CLASS_SCRATCH, &c->workspace);
    if (!st) {
        for (size_t i = 0; i < c->pools.size(); ++i)
            c->pools[i] = static_cast<char *>(c->pool->ptr) + i * f.pages * page_bytes;
        if (cudaError_t err = cudaMemsetAsync(c->arrays->ptr, 0xff, c->table.size() * sizeof(int32_t), b->stream))
            st = cuda_fail(err, "cudaMemsetAsync");
        if (cudaError_t err = st ? cudaSuccess : cudaMemsetAsync(c->workspace->ptr, 0, MF_PAGED_WORKSPACE_BYTES, b->stream))
            st = cuda_fail(err, "cudaMemsetAsync");
    }
    if (st) {
        mf_paged_destroy(c);
        return st;
    }
    *out = c;
    return MF_OK;
}

int32_t mf_paged_destroy(mf_paged_cache *c) {
    if (!c) return MF_OK;
    for (mf_buffer *buf : {c->pool, c->arrays, c->workspace})
        if (buf) mf_buffer_release(c->b, buf);
    delete c;
    return MF_OK;
}

int32_t mf_paged_begin(mf_paged_cache *c, const uint32_t *sequences, const uint64_t *tokens, uint64_t n) {
    int32_t st = check_cache(c);
    if (st) return st;
    if (n && (!sequences || !tokens)) return fail(MF_INVALID_ARGUMENT, "null argument");
    if (n > c->cfg.sequences) return fail(MF_INVALID_ARGUMENT, "a pass names a sequence twice");
    const uint64_t pt = c->cfg.page_tokens, most = (uint64_t)c->cfg.max_pages * pt;
    try {
        // Checks, and the pages that the pass takes.
        std::vector<uint8_t> named(c->cfg.sequences, 0);
        std::vector<std::pair<uint32_t, uint32_t>> shared;  // (last page, sequence) of those that append into a shared one
        uint64_t need = 0, rows = 0;
        for (uint64_t i = 0; i < n; ++i) {
            const uint32_t s = sequences[i];
            if (s >= c->cfg.sequences) return fail(MF_OUT_OF_BOUNDS, "sequence exceeds the paged cache's sequences");
            if (named[s]) return fail(MF_INVALID_ARGUMENT, "a pass names a sequence twice");
            named[s] = 1;
            if (tokens[i] > most - c->length[s]) return fail(MF_OUT_OF_BOUNDS, "pass exceeds the sequence's pages");
            need += c->pages_of(c->length[s] + tokens[i]) - c->pages_of(c->length[s]);
            rows += tokens[i];
            if (tokens[i] && c->length[s] % pt) {
                const uint32_t last = (uint32_t)c->page(s, c->length[s] / pt);
                if (c->refs[last] > 1) shared.push_back({last, s});
            }
        }
        if (rows > INT32_MAX) return fail(MF_OVERFLOW, "token rows exceed the 32-bit row offsets");
        // Of the sequences that share a page, the last owner keeps it.
        std::sort(shared.begin(), shared.end());
        std::vector<uint32_t> from, to, copier;
        for (size_t i = 0, j; i < shared.size(); i = j) {
            for (j = i; j < shared.size() && shared[j].first == shared[i].first; ++j) {
            }
            const size_t copies = std::min<size_t>(j - i, c->refs[shared[i].first] - 1);
            for (size_t k = 0; k < copies; ++k) from.push_back(shared[i].first), copier.push_back(shared[i + k].second);
        }
        need += from.size();
        if (need > c->free.size()) return fail(MF_RESOURCE_LIMIT, "paged cache has too few free pages");
        to.reserve(from.size());
        std::vector<uint32_t> entries, ids;  // of the table that change (a page taken is an entry), and to what
        entries.reserve(need), ids.reserve(need);
        c->pass.resize(4 * n + 1);  // within its reservation
        // Nothing below fails but the device.
        uint64_t first = c->cfg.sequences, last = 0;
        auto set = [&](uint64_t s, uint64_t nth, uint32_t p) {
            c->page(s, nth) = (int32_t)p;
            entries.push_back((uint32_t)(s * c->cfg.max_pages + nth)), ids.push_back(p);
            first = std::min(first, s), last = std::max(last, s);
        };
        for (size_t k = 0; k < from.size(); ++k) {
            const uint32_t s = copier[k], p = c->take();
            to.push_back(p);
            c->refs[from[k]]--;
            set(s, c->length[s] / pt, p);
        }
        int32_t row = 0;
        for (uint64_t i = 0; i < n; ++i) {
            const uint32_t s = sequences[i];
            const uint64_t before = c->length[s], after = before + tokens[i];
            for (uint64_t p = c->pages_of(before); p < c->pages_of(after); ++p) set(s, p, c->take());
            c->length[s] = after;
            c->pass[i] = (int32_t)s, c->pass[n + i] = (int32_t)before, c->pass[2 * n + i] = (int32_t)after;
            c->pass[3 * n + i] = row;
            row += (int32_t)tokens[i];
        }
        c->pass[4 * n] = row;
        c->pass_n = n, c->pass_rows = rows, c->in_pass = false;
        if ((st = copy_all(c, from, to))) return st;
        // The rows, or the changed entries where those are fewer bytes.  (A
        // decode step of 512 sequences changes some 32 entries all over the
        // table; rows of 256 entries were a copy of 512 KB that the host waited
        // for, with all work before it: 850 us a call in a loop, now 24.)
        if (need && 2 * need >= (last - first + 1) * c->cfg.max_pages) st = send_rows(c, first, last);
        else if (need) st = paged_set_table(c->device_table(), entries.data(), ids.data(), need, c->b->stream);
        if (st) return st;
        MF_CUDA_TRY(cudaMemcpyAsync(c->device_pass(), c->pass.data(), c->pass.size() * sizeof(int32_t),
                                    cudaMemcpyHostToDevice, c->b->stream));
        c->b->counts.copies++;
        c->in_pass = true;
    } catch (const std::bad_alloc &) {
        return fail(MF_RESOURCE_LIMIT, "host allocation failed");
    }
    return MF_OK;
}

int32_t mf_paged_write(mf_paged_cache *c, uint32_t layer, const mf_buffer *key, const mf_buffer *value) {
    int32_t st = check_cache(c);
    if (st) return st;
    if (!c->in_pass) return fail(MF_INVALID_ARGUMENT, "paged cache is not in a pass");
    if (layer >= c->cfg.layers) return fail(MF_OUT_OF_BOUNDS, "layer exceeds the paged cache's layers");
    const uint64_t kvw = (uint64_t)c->cfg.kv_heads * c->cfg.head_dim;
    st = check_rows(c, key, c->pass_rows, kvw);
    if (!st) st = check_rows(c, value, c->pass_rows, kvw);
    if (st) return st;
    const int32_t *pass = c->device_pass();
    const uint64_t n = c->pass_n;
    return paged_append(c->pools[2 * layer], c->pools[2 * layer + 1], c->cfg.page_dtype, c->view(),
                        static_cast<const float *>(key->ptr), static_cast<const float *>(value->ptr), c->pass_rows,
                        pass + n, pass + 3 * n, c->cfg.kv_heads, c->cfg.head_dim, c->b->stream);
}

int32_t mf_paged_gqa(mf_paged_cache *c, uint32_t layer, mf_buffer *output, const mf_buffer *query, uint32_t query_heads) {
    int32_t st = check_cache(c);
    if (st) return st;
    if (!c->in_pass) return fail(MF_INVALID_ARGUMENT, "paged cache is not in a pass");
    if (layer >= c->cfg.layers) return fail(MF_OUT_OF_BOUNDS, "layer exceeds the paged cache's layers");
    if (query_heads == 0 || query_heads % c->cfg.kv_heads)
        return fail(MF_INVALID_SHAPE, "query heads must be a nonzero multiple of key/value heads");
    if (c->pass_n * query_heads > INT32_MAX / 128) return fail(MF_OVERFLOW, "query rows exceed the 32-bit work list");
    const uint64_t width = (uint64_t)query_heads * c->cfg.head_dim;
    st = check_rows(c, query, c->pass_n, width);
    if (!st) st = check_rows(c, output, c->pass_n, width);
    if (st) return st;
    if (output == query) return fail(MF_INVALID_ARGUMENT, "paged attention output must not be its query");
    return paged_gqa(static_cast<float *>(output->ptr), static_cast<const float *>(query->ptr), c->pools[2 * layer],
                     c->pools[2 * layer + 1], c->cfg.page_dtype, c->view(), c->device_pass() + 2 * c->pass_n, query_heads,
                     c->cfg.kv_heads, c->cfg.head_dim, c->workspace->ptr, c->b->stream);
}

int32_t mf_paged_fork(mf_paged_cache *c, uint32_t source, uint32_t destination) {
    int32_t st = check_cache(c);
    if (st) return st;
    if (source >= c->cfg.sequences || destination >= c->cfg.sequences)
        return fail(MF_OUT_OF_BOUNDS, "sequence exceeds the paged cache's sequences");
    if (source == destination || c->length[destination])
        return fail(MF_INVALID_ARGUMENT, "a fork's destination must be another, empty sequence");
    c->in_pass = false;
    c->length[destination] = c->length[source];
    const uint64_t pages = c->pages_of(c->length[source]);
    for (uint64_t p = 0; p < pages; ++p) {
        c->page(destination, p) = c->page(source, p);
        c->refs[c->page(source, p)]++;
    }
    return pages ? send_rows(c, destination, destination) : MF_OK;
}

int32_t mf_paged_truncate(mf_paged_cache *c, uint32_t sequence, uint64_t length) {
    int32_t st = check_cache(c);
    if (st) return st;
    if (sequence >= c->cfg.sequences) return fail(MF_OUT_OF_BOUNDS, "sequence exceeds the paged cache's sequences");
    if (length > c->length[sequence]) return fail(MF_OUT_OF_BOUNDS, "truncation exceeds the sequence's length");
    c->in_pass = false;
    try {
        for (uint64_t p = c->pages_of(length); p < c->pages_of(c->length[sequence]); ++p) {
            c->drop((uint32_t)c->page(sequence, p));
            c->page(sequence, p) = -1;
        }
    } catch (const std::bad_alloc &) {  // the free list had room for every page when it was made
        return fail(MF_RESOURCE_LIMIT, "host allocation failed");
    }
    c->length[sequence] = length;
    return MF_OK;  // the device's table keeps the old ids: none lies within a length
}

int32_t mf_paged_compact(mf_paged_cache *c) {
    int32_t st = check_cache(c);
    if (st) return st;
    try {
        const uint32_t live = (uint32_t)(c->cfg.pages - c->free.size());
        std::vector<uint32_t> from, to;
        for (uint32_t p = 0; p < c->cfg.pages; ++p) {
            if (p < live && !c->refs[p]) to.push_back(p);
            if (p >= live && c->refs[p]) from.push_back(p);
        }
        if (from.empty()) {  // (as many free pages below as live ones above)
            c->in_pass = false;
            return MF_OK;
        }
        std::vector<int32_t> moved(c->cfg.pages, -1);
        for (size_t i = 0; i < from.size(); ++i) moved[from[i]] = (int32_t)to[i];
        std::vector<uint32_t> ids;
        ids.reserve(c->cfg.pages);  // room to return every page
        for (uint32_t p = live; p < c->cfg.pages; ++p) ids.push_back(p);
        decltype(c->free) free(std::greater<uint32_t>(), std::move(ids));
        c->in_pass = false;
        c->free.swap(free);
        for (size_t i = 0; i < from.size(); ++i) std::swap(c->refs[from[i]], c->refs[to[i]]);
        for (int32_t &p : c->table)
            if (p >= 0 && moved[p] >= 0) p = moved[p];
        if ((st = copy_all(c, from, to))) return st;
        return send_rows(c, 0, c->cfg.sequences - 1);
    } catch (const std::bad_alloc &) {
        return fail(MF_RESOURCE_LIMIT, "host allocation failed");
    }
}

int32_t mf_paged_sequence(const mf_paged_cache *c, uint32_t sequence, uint64_t *length, int32_t *pages, uint64_t capacity) {
    int32_t st = check_cache(c);
    if (st) return st;
    if (sequence >= c->cfg.sequences) return fail(MF_OUT_OF_BOUNDS, "sequence exceeds the paged cache's sequences");
    if (!length || (capacity && !pages)) return fail(MF_INVALID_ARGUMENT, "null argument");
    *length = c->length[sequence];
    const uint64_t n = std::min(capacity, c->pages_of(*length));
    for (uint64_t p = 0; p < n; ++p) pages[p] = c->table[(uint64_t)sequence * c->cfg.max_pages + p];
    return MF_OK;
}

int32_t mf_paged_free_pages(const mf_paged_cache *c, uint64_t *free_pages) {
    int32_t st = check_cache(c);
    if (st) return st;
    if (!free_pages) return fail(MF_INVALID_ARGUMENT, "null argument");
    *free_pages = c->free.size();
    return MF_OK;
}

int32_t mf_paged_pages(const mf_paged_cache *c, uint32_t layer, void **key_pages, void **value_pages) {
    int32_t st = check_cache(c);
    if (st) return st;
    if (layer >= c->cfg.layers) return fail(MF_OUT_OF_BOUNDS, "layer exceeds the paged cache's layers");
    if (!key_pages || !value_pages) return fail(MF_INVALID_ARGUMENT, "null argument");
    *key_pages = c->pools[2 * layer], *value_pages = c->pools[2 * layer + 1];
    return MF_OK;
}

}  // extern "C"
