"""Paged cache on a GPU: rows into pages, one-token attention, page copies.

Appended rows and copies are compared bit for bit; attention with the 64-bit
form, element by element within the bound that tests/paged_ref.py derives.
"""
import numpy as np
import pytest
import torch

from paged_ref import PAGE_DTYPES, WORKSPACE, attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from runtime_b200 import _lib

    return _lib.load()


def dev(values, dtype=torch.int32):
    return torch.as_tensor(np.asarray(values), dtype=dtype).cuda()


class Cache:
    """Random pages and a table whose pages lie in no order."""

    def __init__(self, lengths, kv_heads, dim, page, dtype, seed=0, max_pages=None, fill=0.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.code, self.dtype = PAGE_DTYPES[dtype]
        self.page, self.kv_heads, self.dim = page, kv_heads, dim
        need = [-(-n // page) for n in lengths]
        self.pages = sum(need) + 2
        order = np.random.default_rng(seed).permutation(self.pages).astype(np.int32)
        self.table = np.full((len(lengths), max_pages or max(1, max(need))), -1, np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at : at + n]
            at += n
        self.keys, self.values = (torch.randn(self.pages, kv_heads, page, dim, generator=g, device="cuda").to(self.dtype)
                                  for _ in range(2))
        # Whatever no token owns is NaN: it must not reach a result.
        seen = torch.zeros(self.pages, page, dtype=torch.bool)
        for i, n in enumerate(lengths):
            for pos in range(n):
                seen[self.table[i, pos // page], pos % page] = True
        for p in (self.keys, self.values):
            p.masked_fill_(~seen.cuda()[:, None, :, None], float("nan"))
        self.device_table = dev(self.table)

    def attend(self, lib, q, lengths, slots=None, workspace=None, stream=None, out=None):
        n = q.shape[0]
        out = torch.full_like(q, 7.0) if out is None else out
        ws = torch.zeros(WORKSPACE, dtype=torch.uint8, device="cuda") if workspace is None else workspace
        lens = lengths if isinstance(lengths, torch.Tensor) else dev(lengths)
        ids = None if slots is None else dev(slots)
        st = lib.mfk_paged_gqa(out.data_ptr(), q.data_ptr(), self.keys.data_ptr(), self.values.data_ptr(), self.code,
                               self.pages, self.page, self.device_table.data_ptr(), self.table.shape[0],
                               self.table.shape[1], lens.data_ptr(), None if ids is None else ids.data_ptr(), n,
                               q.shape[1], self.kv_heads, self.dim, ws.data_ptr(), WORKSPACE,
                               torch.cuda.current_stream().cuda_stream if stream is None else stream)
        assert st == 0, lib.mf_last_error()
        torch.cuda.synchronize()
        return out

    def check(self, out, q, lengths, slots=None):
        ref, bound = attention(q.cpu(), self.keys.cpu(), self.values.cpu(), self.table, lengths,
                               range(len(lengths)) if slots is None else slots, self.page)
        off = (out.cpu().double() - ref).abs()
        assert torch.isfinite(out).all()
        assert (off <= bound).all(), (off - bound).max().item()


def queries(n, heads, dim, seed=1):
    return torch.randn(n, heads, dim, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * 2


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("q_heads,kv_heads,dim,page", [
    (32, 8, 64, 16), (16, 8, 64, 32), (8, 1, 128, 16), (3, 3, 64, 5), (24, 2, 64, 16), (6, 2, 80, 24), (20, 1, 8, 1),
    (8, 2, 120, 7), (5, 1, 104, 64),
])
def test_attention_over_ragged_sequences(lib, dtype, q_heads, kv_heads, dim, page):
    lengths = [1, 0, page - 1, page, page + 1, 2 * page, 63, 64, 65, 129, 300]
    cache = Cache(lengths, kv_heads, dim, page, dtype)
    q = queries(len(lengths), q_heads, dim)
    out = cache.attend(lib, q, lengths)
    cache.check(out, q, lengths)
    for i, n in enumerate(lengths):
        assert n or not out[i].any()  # no tokens: a row of zeros


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("lengths,heads", [([5000], (8, 2)), ([1, 4097, 0, 2500, 700], (32, 8)), ([1], (1, 1))])
def test_attention_split_over_long_sequences(lib, dtype, lengths, heads):
    cache = Cache(lengths, heads[1], 64, 16, dtype, seed=3)
    q = queries(len(lengths), heads[0], 64)
    ws = torch.zeros(WORKSPACE, dtype=torch.uint8, device="cuda")
    out = cache.attend(lib, q, lengths, workspace=ws)
    cache.check(out, q, lengths)
    for _ in range(3):  # the workspace is ready again, and the join has one order
        assert torch.equal(cache.attend(lib, q, lengths, workspace=ws), out)


def test_more_sequences_than_a_block_scans(lib):
    rng = np.random.default_rng(8)
    lengths = [int(v) for v in rng.integers(0, 9, 1500)]
    cache = Cache(lengths, 1, 16, 4, "f32", seed=5)
    q = queries(len(lengths), 2, 16)
    out = cache.attend(lib, q, lengths)
    cache.check(out, q, lengths)


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
def test_slot_ids_repeat_and_lengths_differ(lib, dtype):
    cache = Cache([40, 77, 12], 2, 64, 16, dtype, seed=2)
    slots, lengths = [2, 0, 1, 1, 0, 1], [12, 40, 77, 3, 0, 50]
    q = queries(len(slots), 8, 64)
    out = cache.attend(lib, q, lengths, slots)
    cache.check(out, q, lengths, slots)


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
def test_bad_pages_slots_and_lengths_stay_in_bounds(lib, dtype):
    """Pages outside the pool hold no tokens, slots outside the table no
    sequence, lengths end at the table."""
    cache = Cache([64, 64, 64, 64], 2, 64, 16, dtype, seed=4)
    cache.table[0, 1], cache.table[1, :], cache.table[2, 3] = -7, cache.pages, 1 << 30
    cache.device_table = dev(cache.table)
    q = queries(6, 4, 64)
    lengths, slots = [64, 64, 64, 1 << 30, 5, -3], [0, 1, 2, 3, 3, 0]
    out = cache.attend(lib, q, lengths, slots)
    cache.check(out, q, [max(0, min(n, 64)) for n in lengths], slots)
    assert not out[1].any() and not out[5].any()
    wild = cache.attend(lib, q, [64] * 6, [-1, 4, 1 << 30, -(1 << 31), 0, 3])
    assert not wild[:4].any() and wild[4:].any()


def test_a_nan_stays_in_its_sequence_and_head(lib):
    cache = Cache([20, 20, 20], 2, 64, 16, "f32", seed=6)
    cache.keys[int(cache.table[1, 0]), 1, 3] = float("nan")
    out = cache.attend(lib, queries(3, 4, 64), [20, 20, 20])
    nan = torch.isnan(out)
    assert nan[1, 2:].all() and not nan[1, :2].any() and not nan[0].any() and not nan[2].any()


@pytest.mark.parametrize("dtype,scale", [("f16", 2.0**-20), ("f16", 2.0**14), ("bf16", 2.0**-60), ("f32", 2.0**-70)])
def test_queries_of_any_size(lib, dtype, scale):
    """Keys of the inverse size: the scores are ordinary ones."""
    lengths = [50]
    cache = Cache(lengths, 2, 64, 16, dtype, seed=7)
    kscale = 1.0 if dtype == "f16" else 1 / scale
    cache.keys = (cache.keys.float() * kscale).to(cache.dtype)
    q = queries(1, 8, 64) * scale
    cache.check(cache.attend(lib, q, lengths), q, lengths)


def test_peaked_scores(lib):
    """One key far above the others, and the same score everywhere."""
    lengths = [200, 200]
    cache = Cache(lengths, 1, 64, 16, "bf16", seed=9)
    q = queries(2, 4, 64)
    cache.keys[int(cache.table[0, 5]), 0, 2] = 40.0 * q[0, 0].sign()
    q[1] = 0.0
    cache.check(cache.attend(lib, q, lengths), q, lengths)


def test_attention_captured_and_replayed_with_other_lengths(lib):
    lengths = [1000, 31, 512, 0]
    cache = Cache(lengths, 2, 64, 16, "bf16", seed=11)
    q, lens = queries(4, 8, 64), dev([3, 1, 2, 0])
    ws = torch.zeros(WORKSPACE, dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(q)
    cache.attend(lib, q, lens, workspace=ws, out=out)
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        st = lib.mfk_paged_gqa(out.data_ptr(), q.data_ptr(), cache.keys.data_ptr(), cache.values.data_ptr(), cache.code,
                               cache.pages, cache.page, cache.device_table.data_ptr(), 4, cache.table.shape[1],
                               lens.data_ptr(), None, 4, 8, 2, 64, ws.data_ptr(), WORKSPACE, stream.cuda_stream)
        assert st == 0
    for now in ([1, 1, 1, 0], [1000, 31, 512, 0], [7, 0, 300, 0]):
        lens.copy_(dev(now))
        graph.replay()
        torch.cuda.synchronize()
        cache.check(out, q, now)


def test_offsets_past_32_bits(lib):
    """Pages whose elements lie past 2^32 (values are made only where used)."""
    page, heads, dim = 64, 8, 128
    pages = (1 << 32) // (page * heads * dim) + 40
    keys, values = (torch.empty(pages, heads, page, dim, dtype=torch.float16, device="cuda") for _ in range(2))
    small = Cache([200], heads, dim, page, "f16", seed=12)
    where = np.array([[pages - 1, 3, pages - 17, pages - 30]], np.int32)
    for p in range(4):
        keys[int(where[0, p])] = small.keys[int(small.table[0, p])]
        values[int(where[0, p])] = small.values[int(small.table[0, p])]
    q, out = queries(1, 16, dim), None
    expected = small.attend(lib, q, [200])
    small.check(expected, q, [200])
    small.keys, small.values, small.pages, small.table = keys, values, pages, where
    small.device_table = dev(where)
    assert torch.equal(small.attend(lib, q, [200]), expected)
    k, v = (torch.randn(1, heads * dim, device="cuda") for _ in range(2))
    start = dev([199])
    assert lib.mfk_paged_append(keys.data_ptr(), values.data_ptr(), 1, pages, page, small.device_table.data_ptr(), 1, 4,
                                k.data_ptr(), v.data_ptr(), 1, start.data_ptr(), None, None, 1, heads, dim,
                                torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(keys[pages - 30, :, 7], k.half().view(heads, dim))
    assert torch.equal(values[pages - 30, :, 7], v.half().view(heads, dim))
    pools = np.array([keys.data_ptr(), values.data_ptr()], np.uint64)
    s, d = np.array([pages - 30], np.uint32), np.array([5], np.uint32)
    assert lib.mfk_copy_pages(pools.ctypes.data, 2, pages, page * heads * dim * 2, s.ctypes.data, d.ctypes.data, 1,
                              torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(keys[5, :, :8], keys[pages - 30, :, :8])


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("counts,starts,page,heads,dim", [
    ([1, 1, 1], [0, 15, 16], 16, 8, 64), ([5, 0, 40, 1], [3, 9, 0, 63], 16, 2, 64), ([200], [1], 7, 3, 40), ([0, 3], [0, 0], 1, 1, 8),
])
def test_append_rows(lib, dtype, counts, starts, page, heads, dim):
    total = [s + c for s, c in zip(starts, counts)]
    cache = Cache(total, heads, dim, page, dtype, seed=13)
    rows = sum(counts) + 2  # two rows behind the last sequence
    k, v = (torch.randn(rows, heads * dim, device="cuda") * 3 for _ in range(2))
    k[0, :3] = torch.tensor([float("inf"), float("nan"), -0.0], device="cuda")
    offsets = np.concatenate(([0], np.cumsum(counts)))
    expected = [cache.keys.clone(), cache.values.clone()]
    for i, c in enumerate(counts):
        for t in range(c):
            pos = starts[i] + t
            for pages, x in zip(expected, (k, v)):
                pages[int(cache.table[i, pos // page]), :, pos % page] = x[offsets[i] + t].view(heads, dim).to(pages.dtype)
    do, ds = dev(offsets), dev(starts)
    st = lib.mfk_paged_append(cache.keys.data_ptr(), cache.values.data_ptr(), cache.code, cache.pages, page,
                              cache.device_table.data_ptr(), len(counts), cache.table.shape[1], k.data_ptr(), v.data_ptr(),
                              rows, ds.data_ptr(), do.data_ptr(), None, len(counts), heads, dim,
                              torch.cuda.current_stream().cuda_stream)
    assert st == 0
    for got, want in zip((cache.keys, cache.values), expected):
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got, nan=0.5), torch.nan_to_num(want, nan=0.5))


def test_append_out_of_bounds_rows_are_dropped(lib):
    cache = Cache([32] * 5, 2, 64, 16, "bf16", seed=14)
    cache.table[1, 0], cache.table[2, 0] = -1, cache.pages
    cache.device_table = dev(cache.table)
    before = cache.keys.clone(), cache.values.clone()
    k = torch.randn(6, 128, device="cuda")
    starts, slots = dev([-1, 0, 3, 32, 5, 2]), dev([0, 1, 2, 3, 5, -1])
    assert lib.mfk_paged_append(cache.keys.data_ptr(), cache.values.data_ptr(), cache.code, cache.pages, 16,
                                cache.device_table.data_ptr(), 5, 2, k.data_ptr(), k.data_ptr(), 6, starts.data_ptr(),
                                None, slots.data_ptr(), 6, 2, 64, torch.cuda.current_stream().cuda_stream) == 0
    for got, want in zip((cache.keys, cache.values), before):
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


@pytest.mark.parametrize("page_bytes,pages,count,pools", [(16, 9, 4, 1), (16384, 300, 130, 3), (4112, 9000, 4100, 2), (48, 5, 2, 70)])
def test_copy_pages(lib, page_bytes, pages, count, pools):
    rng = np.random.default_rng(pages)
    data = torch.randint(0, 256, (pools, pages, page_bytes), dtype=torch.uint8, device="cuda")
    order = rng.permutation(pages).astype(np.uint32)
    targets, sources = order[:count].copy(), rng.choice(order[count:], count).astype(np.uint32)  # sources repeat
    expected = data.clone()
    expected[:, targets.astype(np.int64)] = data[:, sources.astype(np.int64)]
    bases = np.array([data[i].data_ptr() for i in range(pools)], np.uint64)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    assert lib.mfk_copy_pages(bases.ctypes.data, pools, pages, page_bytes, sources.ctypes.data, targets.ctypes.data, count,
                              stream.cuda_stream) == 0
    targets[:], sources[:] = 0, 0  # the lists were read before the call returned
    stream.synchronize()
    assert torch.equal(data, expected)


def test_two_streams_with_a_workspace_each(lib):
    lengths = [3000, 50, 800, 1]
    cache = Cache(lengths, 2, 64, 16, "bf16", seed=15)
    qs = [queries(4, 8, 64, seed=20 + i) for i in range(2)]
    alone = [cache.attend(lib, q, lengths) for q in qs]
    ws = [torch.zeros(WORKSPACE, dtype=torch.uint8, device="cuda") for _ in qs]
    outs, lens = [torch.zeros_like(q) for q in qs], dev(lengths)
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, q in enumerate(qs):
            assert lib.mfk_paged_gqa(outs[i].data_ptr(), q.data_ptr(), cache.keys.data_ptr(), cache.values.data_ptr(),
                                     cache.code, cache.pages, cache.page, cache.device_table.data_ptr(), 4,
                                     cache.table.shape[1], lens.data_ptr(), None, 4, 8, 2, 64, ws[i].data_ptr(), WORKSPACE,
                                     streams[i].cuda_stream) == 0
    torch.cuda.synchronize()
    for got, want in zip(outs, alone):
        assert torch.equal(got, want)


def test_append_then_attend_in_one_stream(lib):
    """A new token's row is seen by the attention that follows it at once."""
    lengths = [33, 16, 1]
    cache = Cache(lengths, 2, 64, 16, "f16", seed=16)
    stream = torch.cuda.current_stream().cuda_stream
    for step in range(4):
        k, v = (torch.randn(3, 128, device="cuda") for _ in range(2))
        q = queries(3, 4, 64, seed=30 + step)
        starts = dev([n - 1 for n in lengths])
        assert lib.mfk_paged_append(cache.keys.data_ptr(), cache.values.data_ptr(), cache.code, cache.pages, 16,
                                    cache.device_table.data_ptr(), 3, cache.table.shape[1], k.data_ptr(), v.data_ptr(), 3,
                                    starts.data_ptr(), None, None, 3, 2, 64, stream) == 0
        cache.check(cache.attend(lib, q, lengths), q, lengths)


@pytest.mark.parametrize("sequences", [129, 300, 4097])
def test_append_finds_each_row_among_many_sequences(lib, sequences):
    rng = np.random.default_rng(sequences)
    counts = rng.integers(0, 4, sequences)
    counts[0], counts[-1] = 0, 2
    rows = int(counts.sum())
    offsets = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    pages = sequences
    keys, values = (torch.zeros(pages, 1, 4, 8, device="cuda") for _ in range(2))
    table = dev(rng.permutation(sequences)[:, None])
    k = torch.arange(rows, device="cuda", dtype=torch.float32)[:, None].repeat(1, 8) + 1
    do, ds = dev(offsets), dev(np.zeros(sequences))
    assert lib.mfk_paged_append(keys.data_ptr(), values.data_ptr(), 0, pages, 4, table.data_ptr(), sequences, 1,
                                k.data_ptr(), (-k).data_ptr(), rows, ds.data_ptr(), do.data_ptr(), None, sequences, 1, 8,
                                torch.cuda.current_stream().cuda_stream) == 0
    want = torch.zeros(pages, 4)
    for i, c in enumerate(counts):
        for t in range(c):
            want[int(table[i, 0]), t] = offsets[i] + t + 1
    assert torch.equal(keys[:, 0, :, 0].cpu(), want) and torch.equal(values[:, 0, :, 3].cpu(), -want)


@pytest.mark.parametrize("dtype,dim", [("f16", 8), ("f32", 16), ("f32", 128), ("bf16", 128)])
def test_lengths_up_to_the_last_position(lib, dtype, dim):
    """A table of 2^31 - 16 positions of which three pages exist, at both ends
    and in the middle: the tokens there are found whatever the lengths."""
    page, most = 16, (1 << 27) - 1
    small = Cache([48], 1, dim, page, dtype, seed=17)
    table = torch.full((1, most), -1, dtype=torch.int32, device="cuda")
    for nth, i in zip((0, 1 << 26, most - 1), range(3)):
        table[0, nth] = int(small.table[0, i])
    ends = [most * page, most * page - 1, most * page - 15, (1 << 30) + 5, 7, (1 << 31) - 1]
    here = [48, 47, 33, 21, 7, 48]  # of them exist
    q, lens, slots = queries(len(ends), 2, dim), dev(ends), dev([0] * len(ends))
    out, ws = torch.full_like(q, 7.0), torch.zeros(WORKSPACE, dtype=torch.uint8, device="cuda")
    st = lib.mfk_paged_gqa(out.data_ptr(), q.data_ptr(), small.keys.data_ptr(), small.values.data_ptr(), small.code,
                           small.pages, page, table.data_ptr(), 1, most, lens.data_ptr(), slots.data_ptr(), len(ends),
                           2, 1, dim, ws.data_ptr(), WORKSPACE, torch.cuda.current_stream().cuda_stream)
    assert st == 0, lib.mf_last_error()
    torch.cuda.synchronize()
    small.check(out, q, here, [0] * len(ends))
