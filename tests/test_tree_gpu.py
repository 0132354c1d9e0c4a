"""Drafted trees on a GPU: rotated appends, attention, the convolution along
branches, acceptance.  Compared with 64-bit forms within bounds that
tests/tree_ref.py derives, moved rows and whole numbers exactly."""
import numpy as np
import pytest
import torch

import tree_ref
from paged_ref import PAGE_DTYPES
from tree_ref import TREE_WORKSPACE, U

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from runtime_b200 import _lib

    return _lib.load()


def dev(values, dtype=torch.int32):
    return torch.as_tensor(np.asarray(values), dtype=dtype).cuda()


def at(x):
    return None if x is None else x.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


class Draft:
    """Sequences of `lengths` tokens, the last rows[i] of them drafted, over pages in no order."""

    def __init__(self, lengths, rows, shape="tree", seed=0, gap=0, behind=0):
        rng = np.random.default_rng(seed)
        self.lengths, self.rows = list(lengths), list(rows)
        self.offsets = gap + np.concatenate([[0], np.cumsum(rows)])
        self.tokens = int(self.offsets[-1]) + behind
        self.parents = None
        if shape != "chain":
            self.parents = np.full(self.tokens, -7)
            for i, n in enumerate(rows):
                tree = tree_ref.random_tree(n, rng)
                if shape == "garbage":  # what is no earlier row counts as none
                    tree = [p if rng.random() < 0.6 else int(rng.choice([r, r + 1, n, n + 9, -1, -2**31, 2**31 - 1])) for r, p in enumerate(tree)]
                self.parents[self.offsets[i] : self.offsets[i] + n] = tree
        self.device = {n: None if v is None else dev(v) for n, v in
                       (("lengths", self.lengths), ("offsets", self.offsets), ("parents", self.parents),
                        ("starts", [n - r for n, r in zip(self.lengths, self.rows)]))}

    def owned(self):
        """Rows that belong to a sequence."""
        inside = np.zeros(self.tokens, bool)
        inside[self.offsets[0] : self.offsets[-1]] = True
        return torch.from_numpy(inside)


class Cache:
    def __init__(self, lengths, kv_heads, dim, page, dtype, seed=0, max_pages=None, fill=True):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.code, self.dtype = PAGE_DTYPES[dtype]
        self.page, self.kv_heads, self.dim = page, kv_heads, dim
        need = [-(-n // page) for n in lengths]
        self.pages = sum(need) + 2
        order = np.random.default_rng(seed).permutation(self.pages).astype(np.int32)
        self.table = np.full((len(lengths), max_pages or max(1, max(need))), -1, np.int32)
        done = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[done : done + n]
            done += n
        self.keys, self.values = (torch.randn(self.pages, kv_heads, page, dim, generator=g, device="cuda").to(self.dtype) for _ in range(2))
        if fill:  # whatever no token owns is NaN: it must not reach a result
            seen = torch.zeros(self.pages, page, dtype=torch.bool)
            for i, n in enumerate(lengths):
                pos = np.arange(n)
                seen[self.table[i, pos // page], pos % page] = True
            for p in (self.keys, self.values):
                p.masked_fill_(~seen.cuda()[:, None, :, None], float("nan"))
        self.device_table = dev(self.table)

    def args(self):
        return (self.keys.data_ptr(), self.values.data_ptr(), self.code, self.pages, self.page, self.device_table.data_ptr(),
                self.table.shape[0], self.table.shape[1])


def workspace():
    return torch.zeros(TREE_WORKSPACE, dtype=torch.uint8, device="cuda")


def attend(lib, cache, draft, q, slots=None, ws=None, out=None, wait=True):
    out = torch.full_like(q, 7.0) if out is None else out
    ws = workspace() if ws is None else ws
    d = draft.device
    st = lib.mfk_paged_tree_gqa(out.data_ptr(), q.data_ptr(), *cache.args(), q.shape[0], at(d["lengths"]), at(d["offsets"]),
                                at(d["parents"]), at(slots), len(draft.rows), q.shape[1], cache.kv_heads, cache.dim,
                                ws.data_ptr(), TREE_WORKSPACE, stream())
    assert st == 0, lib.mf_last_error()
    if wait:
        torch.cuda.synchronize()
    return out


def check(out, cache, draft, q, slots=None):
    ref, bound = tree_ref.attention(q.cpu(), cache.keys.cpu(), cache.values.cpu(), cache.table, draft.lengths, draft.offsets,
                                    draft.parents, range(len(draft.rows)) if slots is None else slots, cache.page)
    own = draft.owned()
    out = out.cpu()
    assert (out[~own] == 7.0).all()  # rows of no sequence: as they were
    assert torch.isfinite(out[own]).all()
    off = (out.double() - ref).abs()[own]
    assert (off <= bound[own]).all(), ((off / bound[own].clamp_min(1e-300)).max().item(), off.max().item())


def queries(n, heads, dim, seed=1):
    return torch.randn(n, heads, dim, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * 2


LENGTHS = [1, 9, 0, 17, 64, 65, 130, 12, 200, 40]
ROWS = [1, 9, 0, 1, 7, 33, 16, 0, 64, 40]


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("shape", ["tree", "chain", "garbage"])
@pytest.mark.parametrize("q_heads,kv_heads,dim,page", [
    (8, 2, 64, 16), (16, 8, 64, 32), (8, 1, 128, 16), (3, 3, 64, 5), (6, 2, 80, 24), (5, 1, 8, 1), (8, 2, 120, 7), (12, 1, 104, 64),
])
def test_attention_over_ragged_drafts(lib, dtype, shape, q_heads, kv_heads, dim, page):
    cache = Cache(LENGTHS, kv_heads, dim, page, dtype)
    draft = Draft(LENGTHS, ROWS, shape, gap=3, behind=5)
    q = queries(draft.tokens, q_heads, dim)
    check(attend(lib, cache, draft, q), cache, draft, q)


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("heads,dim", [((8, 2), 64), ((8, 8), 64), ((16, 2), 128)])
@pytest.mark.parametrize("lengths,rows", [([5000], [11]), ([1, 4097, 0, 2500, 700], [1, 40, 0, 3, 130])])
def test_attention_split_over_long_sequences(lib, dtype, heads, dim, lengths, rows):
    cache = Cache(lengths, heads[1], dim, 16, dtype, seed=3)
    draft = Draft(lengths, rows, seed=2)
    q = queries(draft.tokens, heads[0], dim)
    ws = workspace()
    out = attend(lib, cache, draft, q, ws=ws)
    check(out, cache, draft, q)
    for _ in range(3):  # the workspace is ready again, and the join has one order
        assert torch.equal(attend(lib, cache, draft, q, ws=ws), out)


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_one_head_split_over_every_processor(lib, dtype, dim):
    lengths, rows = [20011], [9]  # hundreds of tiles of one item: a run of them for each CTA, all joined
    cache = Cache(lengths, 1, dim, 24, dtype, seed=9)
    draft = Draft(lengths, rows, seed=8)
    q = queries(9, 3, dim)
    ws = workspace()
    out = attend(lib, cache, draft, q, ws=ws)
    check(out, cache, draft, q)
    assert torch.equal(attend(lib, cache, draft, q, ws=ws), out)


def test_captured_graphs_that_share_a_workspace_take_turns(lib):
    cases = []
    ws = workspace()
    for lengths, rows, dim, dtype in (([3000, 40], [8, 3], 64, "bf16"), ([700], [30], 128, "f32")):
        cache, draft = Cache(lengths, 2, dim, 16, dtype), Draft(lengths, rows)
        q = queries(sum(rows), 8, dim)
        out = torch.full_like(q, 7.0)
        attend(lib, cache, draft, q, ws=ws, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            attend(lib, cache, draft, q, ws=ws, out=out, wait=False)
        cases.append((cache, draft, q, out, graph))
    for _ in range(3):
        for *_, out, graph in cases:
            out.fill_(7.0)
            graph.replay()
    torch.cuda.synchronize()
    for cache, draft, q, out, _ in cases:
        check(out, cache, draft, q)


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_scores_that_grow_and_fall_along_a_sequence(lib, dtype, dim):
    """Maxima that change with every tile, up to scores of thousands: only a few tokens count."""
    lengths, rows = [1500, 700], [10, 25]
    cache = Cache(lengths, 2, dim, 16, dtype, seed=5, fill=False)
    for i, n in enumerate(lengths):
        pos = np.arange(n)
        page, slot = (torch.from_numpy(x).cuda().long() for x in (cache.table[i, pos // 16], pos % 16))
        size = torch.from_numpy(10.0 ** (2.0 * np.sin(pos / 90.0 + i))).cuda()
        cache.keys[page, :, slot] = (cache.keys[page, :, slot].double() * size[:, None, None]).to(cache.dtype)
    draft = Draft(lengths, rows)
    q = queries(draft.tokens, 8, dim)
    check(attend(lib, cache, draft, q), cache, draft, q)


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("group", [1, 5, 64, 130, 256, 300])
def test_groups_of_query_heads(lib, dtype, group):
    lengths, rows = [70, 133], [5, 3]
    cache = Cache(lengths, 2, 64, 16, dtype, seed=4)
    draft = Draft(lengths, rows, seed=3)
    q = queries(draft.tokens, 2 * group, 64)
    check(attend(lib, cache, draft, q), cache, draft, q)


@pytest.mark.parametrize("shape", ["tree", "chain"])
def test_large_drafts(lib, shape):
    """Rows of many tiles: a deep tree, a prompt in one chunk."""
    lengths, rows = [700, 450], [700, 333]
    cache = Cache(lengths, 2, 64, 16, "bf16", seed=4)
    draft = Draft(lengths, rows, shape, seed=5)
    if shape == "tree":  # one sequence as a single long branch
        draft.parents[:700] = np.arange(-1, 699)
        draft.device["parents"] = dev(draft.parents)
    q = queries(draft.tokens, 6, 64)
    check(attend(lib, cache, draft, q), cache, draft, q)


def test_a_chain_is_the_tree_of_a_single_branch(lib):
    lengths, rows = [300, 80], [70, 80]
    cache = Cache(lengths, 2, 64, 16, "f16")
    chain, tree = Draft(lengths, rows, "chain"), Draft(lengths, rows)
    tree.device["parents"] = dev(np.concatenate([np.arange(-1, n - 1) for n in rows]))
    q = queries(150, 8, 64)
    assert torch.equal(attend(lib, cache, chain, q), attend(lib, cache, tree, q))


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
def test_rows_at_places_that_do_not_exist(lib, dtype):
    """Lengths below the rows or past the table, missing pages, bad slots: rows that
    see nothing are zeros."""
    lengths = [40, 40, 40, 40, 40, 40]
    cache = Cache(lengths, 2, 64, 16, dtype, fill=False)
    cache.table[0, 1] = -1
    cache.table[1, 0] = cache.pages
    cache.table[2, :] = -1
    cache.device_table = dev(cache.table)
    draft = Draft([40, 40, 40, 3, 48, 60], [5, 30, 4, 8, 48, 20], seed=1)
    q = queries(draft.tokens, 4, 64)
    check(attend(lib, cache, draft, q), cache, draft, q)
    slots = [5, -1, 6, 0, 2**31 - 1, 3]
    check(attend(lib, cache, draft, q, slots=dev(slots)), cache, draft, q, slots=slots)
    out = attend(lib, cache, Draft([-5, -2**31, 0, 1, 2, 3], [5, 30, 4, 8, 48, 20]), q)
    assert not out[:39].any()


def test_one_row_per_sequence_without_offsets(lib):
    lengths = [5, 0, 70, 129]
    cache = Cache(lengths, 2, 64, 16, "bf16")
    draft = Draft(lengths, [1] * 4, "chain")
    q = queries(4, 8, 64)
    full = attend(lib, cache, draft, q)
    draft.device["offsets"] = None
    assert torch.equal(attend(lib, cache, draft, q), full)
    ref, bound = tree_ref.attention(q.cpu(), cache.keys.cpu(), cache.values.cpu(), cache.table, lengths, range(5), None, range(4), 16)
    assert ((full.cpu().double() - ref).abs() <= bound).all()


def test_no_table_at_all_is_rows_of_zeros(lib):
    q, out = queries(3, 2, 64), torch.full((3, 2, 64), 7.0, device="cuda")
    one, offsets, ws = dev([3]), dev([0, 3]), workspace()
    st = lib.mfk_paged_tree_gqa(out.data_ptr(), q.data_ptr(), None, None, 0, 0, 16, None, 1, 0, 3, one.data_ptr(),
                                offsets.data_ptr(), None, None, 1, 2, 1, 64, ws.data_ptr(), TREE_WORKSPACE, stream())
    assert st == 0
    torch.cuda.synchronize()
    assert not out.any()


def test_offsets_past_the_rows_are_cut(lib):
    lengths = [30, 30]
    cache = Cache(lengths, 1, 64, 16, "f32")
    draft = Draft(lengths, [4, 6])
    q = queries(10, 2, 64)
    whole = attend(lib, cache, draft, q)
    cut = queries(10, 2, 64)[:8].contiguous()
    draft.device["offsets"] = dev([0, 4, 8])  # what the cut makes of [0, 4, 10]
    draft.device["lengths"] = dev([30, 30])
    short = attend(lib, cache, draft, cut)
    draft.device["offsets"] = dev([0, 4, 10])
    assert torch.equal(attend(lib, cache, draft, cut), short) and torch.equal(short[:4], whole[:4])
    for bad in ([0, 4, -3], [-5, 4, 2**31 - 1], [9, 4, 2], [2**31 - 1, -2**31, 5]):
        draft.device["offsets"] = dev(bad)
        attend(lib, cache, draft, q)


def test_many_sequences(lib):
    rng = np.random.default_rng(8)
    lengths = [int(v) for v in rng.integers(0, 12, 1500)]
    rows = [int(rng.integers(0, n + 1)) for n in lengths]
    cache = Cache(lengths, 1, 16, 4, "f32", seed=5)
    draft = Draft(lengths, rows, seed=6)
    q = queries(draft.tokens, 2, 16)
    check(attend(lib, cache, draft, q), cache, draft, q)


def test_a_captured_call_follows_its_arrays(lib):
    cap = [200, 90, 300]
    cache = Cache(cap, 2, 64, 16, "bf16", fill=False)
    draft = Draft(cap, [8, 8, 8])
    q, out, ws = queries(24, 8, 64), torch.full((24, 8, 64), 7.0, device="cuda"), workspace()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attend(lib, cache, draft, q, ws=ws, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend(lib, cache, draft, q, ws=ws, out=out, wait=False)
    for lengths, rows, seed in (([200, 90, 300], [8, 8, 8], 1), ([24, 60, 8], [20, 1, 3], 2), ([0, 17, 299], [0, 17, 7], 3)):
        now = Draft(lengths, rows, seed=seed, behind=24 - sum(rows))
        for n in ("lengths", "offsets", "parents"):
            draft.device[n].copy_(now.device[n])
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        check(out, cache, now, q)


def test_calls_on_two_streams_with_a_workspace_each(lib):
    lengths, rows = [3000, 2000], [20, 30]
    cache = Cache(lengths, 2, 64, 16, "f16")
    draft = Draft(lengths, rows)
    q = queries(50, 8, 64)
    want = attend(lib, cache, draft, q)
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [torch.full_like(q, 7.0) for _ in range(2)]
    spaces = [workspace() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, o, w in zip(streams, outs, spaces):
            with torch.cuda.stream(s):
                attend(lib, cache, draft, q, ws=w, out=o, wait=False)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("dim,rows", [(64, 3), (64, 60), (128, 20)])
@pytest.mark.parametrize("length", [100, 5000, 60000])
def test_error_of_the_whole_output(lib, dtype, dim, rows, length):
    """At most 16 U of the output's norm (tests/test_paged_accuracy.py derives it)."""
    kv, heads, page = 2, 8, 16
    cache = Cache([length], kv, dim, page, dtype, seed=length + dim, fill=False)
    draft = Draft([length], [rows], "chain")
    q = queries(rows, heads, dim)
    got = attend(lib, cache, draft, q).double()
    where = torch.from_numpy(cache.table[0]).cuda().long()
    k, v = (x[where].double().transpose(1, 2).reshape(-1, kv, dim)[:length].repeat_interleave(heads // kv, 1) for x in (cache.keys, cache.values))
    s = torch.einsum("rhd,nhd->rhn", q.double(), k) / dim**0.5
    hidden = torch.arange(length, device="cuda") > length - rows + torch.arange(rows, device="cuda")[:, None]
    p = torch.softmax(s.masked_fill(hidden[:, None], -np.inf), 2)
    want = torch.einsum("rhn,nhd->rhd", p, v)
    assert ((got - want).norm() / want.norm()).item() <= 16 * U


# ---------------------------------------------------------------------
# Rotated appends
# ---------------------------------------------------------------------

def append(lib, cache, draft, q, k, v, weights, positions=None, slots=None, q_out=None, epsilon=1e-5, theta=1e6):
    q_out = (torch.full_like(q, 7.0) if q is not None else None) if q_out is None else q_out
    d = draft.device
    st = lib.mfk_paged_append_rope(*cache.args(), at(q_out), at(q), k.data_ptr(), v.data_ptr(), k.shape[0], at(weights[0]),
                                   at(weights[1]), epsilon, theta, at(positions), at(d["starts"]), at(d["offsets"]), at(slots),
                                   len(draft.rows), 0 if q is None else q.shape[1], cache.kv_heads, cache.dim, stream())
    assert st == 0, lib.mf_last_error()
    torch.cuda.synchronize()
    return q_out


def rounding(value, dtype):
    """Half a step of a page's type at `value`: relative, and below the smallest normal value absolute."""
    info = torch.finfo(dtype)
    return value.abs() * (info.eps / 2) * 1.01 + info.smallest_normal * info.eps / 2 if dtype != torch.float32 else 0.0


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("q_heads,kv_heads,dim,page", [(8, 2, 64, 16), (16, 8, 64, 32), (8, 1, 128, 16), (3, 3, 40, 5), (6, 2, 80, 24), (5, 1, 8, 1), (1, 2, 120, 7)])
def test_rotated_append(lib, dtype, norm, q_heads, kv_heads, dim, page):
    cache = Cache(LENGTHS, kv_heads, dim, page, dtype, fill=False)
    draft = Draft(LENGTHS, ROWS, gap=2, behind=4)
    g = torch.Generator(device="cuda").manual_seed(3)
    n = draft.tokens
    q, k, v = (torch.randn(n, h, dim, generator=g, device="cuda") for h in (q_heads, kv_heads, kv_heads))
    weights = [torch.randn(dim, generator=g, device="cuda") if norm else None for _ in range(2)]
    positions = np.random.default_rng(1).integers(0, 131071, n)
    before = [cache.keys.cpu().double(), cache.values.cpu().double()]
    out = append(lib, cache, draft, q, k, v, weights, dev(positions)).cpu()
    own = draft.owned()
    want, bound = tree_ref.rotated(q.cpu(), None if not norm else weights[0].cpu(), 1e-5, 1e6, positions)
    assert (out[~own] == 7.0).all()
    assert ((out.double() - want).abs() <= bound)[own].all()
    key, key_bound = tree_ref.rotated(k.cpu(), None if not norm else weights[1].cpu(), 1e-5, 1e6, positions)
    value, value_bound = v.cpu().double(), torch.zeros(n, kv_heads, dim).double()
    for pages, new, slack, old in ((cache.keys, key, key_bound, before[0]), (cache.values, value, value_bound, before[1])):
        allowed = torch.zeros_like(old)
        for i, rows in enumerate(draft.rows):
            for r in range(rows):
                pos = draft.lengths[i] - rows + r
                where = (int(cache.table[i, pos // page]), slice(None), pos % page)
                old[where] = new[draft.offsets[i] + r]
                allowed[where] = slack[draft.offsets[i] + r] + rounding(new[draft.offsets[i] + r], cache.dtype)
        assert ((pages.cpu().double() - old).abs() <= allowed).all()


def test_positions_default_to_places(lib):
    lengths, rows = [40, 9], [12, 9]
    draft = Draft(lengths, rows)
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(21, h, 64, generator=g, device="cuda") for h in (4, 2, 2))
    caches = [Cache(lengths, 2, 64, 16, "f32", fill=False) for _ in range(2)]
    places = np.concatenate([np.arange(n - r, n) for n, r in zip(lengths, rows)])
    outs = [append(lib, c, draft, q, k, v, (None, None), p) for c, p in zip(caches, (None, dev(places)))]
    assert torch.equal(*outs) and torch.equal(caches[0].keys, caches[1].keys)
    inplace = q.clone()
    append(lib, caches[0], draft, inplace, k, v, (None, None), q_out=inplace)
    assert torch.equal(inplace, outs[0])
    keys = caches[0].keys.clone()
    append(lib, caches[0], draft, None, k, v, (None, None))  # without queries
    assert torch.equal(caches[0].keys, keys)


@pytest.mark.parametrize("page_dtype", PAGE_DTYPES)
def test_rotated_append_writes_what_norm_rotation_and_append_write(lib, page_dtype):
    """With heads of 64 a cache may be written by either, bit for bit."""
    from runtime_b200.backend import CudaBackend

    tokens, heads, kv, dim = 37, 8, 4, 64
    rng = np.random.default_rng(5)
    q, k, v = (rng.standard_normal((tokens, h * dim)).astype(np.float32) for h in (heads, kv, kv))
    wq, wk = (rng.standard_normal(dim).astype(np.float32) for _ in range(2))
    positions = rng.integers(0, 131071, tokens)
    with CudaBackend(0) as be:
        qo, ko = be.allocate_f32((tokens, heads * dim)), be.allocate_f32((tokens, kv * dim))
        be.qk_norm_rope(qo, ko, be.upload_f32(q), be.upload_f32(k), be.upload_f32(wq), be.upload_f32(wk), positions,
                        (heads, dim, 1e6), (kv, dim), 1e-5)
        q_want, k_want = (torch.from_numpy(np.array(be.read_f32(x))).cuda().view(tokens, -1, dim) for x in (qo, ko))
    draft = Draft([50], [tokens], "chain")
    here, there = (Cache([50], kv, dim, 16, page_dtype, fill=False) for _ in range(2))
    t = lambda x: torch.from_numpy(x).cuda().view(tokens, -1, dim)  # noqa: E731
    out = append(lib, here, draft, t(q), t(k), t(v), (torch.from_numpy(wq).cuda(), torch.from_numpy(wk).cuda()), dev(positions))
    assert torch.equal(out, q_want)
    st = lib.mfk_paged_append(*there.args(), k_want.contiguous().data_ptr(), t(v).data_ptr(), tokens, at(draft.device["starts"]),
                              at(draft.device["offsets"]), None, 1, kv, dim, stream())
    assert st == 0
    torch.cuda.synchronize()
    assert torch.equal(here.keys, there.keys) and torch.equal(here.values, there.values)


def test_append_at_places_that_do_not_exist(lib):
    """Bad slots and pages, negative starts, positions past the table: nothing is written, queries are rotated."""
    lengths = [40] * 5
    cache = Cache(lengths, 2, 64, 16, "f32", fill=False)
    cache.table[0, 2], cache.table[1, 2] = -1, cache.pages
    cache.device_table = dev(cache.table)
    draft = Draft(lengths, [4] * 5, "chain")
    draft.device["starts"] = dev([36, 36, -1, 46, 36])
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(20, h, 64, generator=g, device="cuda") for h in (2, 2, 2))
    keys = cache.keys.clone()
    out = append(lib, cache, draft, q, k, v, (None, None), dev(np.zeros(20)), slots=dev([0, 1, 2, 3, 5]))
    assert torch.equal(out, q)  # position 0 turns nothing
    keys[cache.table[3, 2], :, 14:16] = k[12:14].transpose(0, 1)
    assert torch.equal(cache.keys, keys)


# ---------------------------------------------------------------------
# Convolution
# ---------------------------------------------------------------------

def convolve(lib, draft, projection, kernel, history, slots=None):
    hidden, width = kernel.shape
    out = torch.full((projection.shape[0], hidden), 7.0, device="cuda")
    d = draft.device
    st = lib.mfk_tree_convolution(out.data_ptr(), projection.data_ptr(), kernel.data_ptr(), at(history), history.shape[0],
                                  projection.shape[0], at(d["offsets"]), at(d["parents"]), at(slots), len(draft.rows), hidden,
                                  width, stream())
    assert st == 0, lib.mf_last_error()
    torch.cuda.synchronize()
    return out


def convolution_inputs(draft, hidden, width, slots, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(draft.tokens, 3 * hidden, generator=g, device="cuda"), torch.randn(hidden, width, generator=g, device="cuda"),
            torch.randn(slots, width - 1, hidden, generator=g, device="cuda"))


@pytest.mark.parametrize("shape", ["tree", "chain", "garbage"])
@pytest.mark.parametrize("hidden,width", [(64, 3), (1024, 3), (130, 4), (7, 1), (1, 2), (516, 16), (2049, 5)])
def test_convolution_along_branches(lib, shape, hidden, width):
    draft = Draft(LENGTHS, ROWS, shape, gap=3, behind=6)
    projection, kernel, history = convolution_inputs(draft, hidden, width, len(ROWS))
    out = convolve(lib, draft, projection, kernel, history).cpu()
    want, bound = tree_ref.convolution(projection.cpu(), kernel.cpu(), history.cpu(), draft.offsets, draft.parents, range(len(ROWS)))
    own = draft.owned()
    assert (out[~own] == 7.0).all()
    assert ((out.double() - want).abs() <= bound)[own].all()


def test_convolution_slots(lib):
    draft = Draft(LENGTHS, ROWS)
    projection, kernel, history = convolution_inputs(draft, 64, 3, 4)
    slots = [3, -1, 2, 1, 4, 0, 2**31 - 1, 0, -2**31, 3]
    out = convolve(lib, draft, projection, kernel, history, dev(slots)).cpu()
    want, bound = tree_ref.convolution(projection.cpu(), kernel.cpu(), history.cpu(), draft.offsets, draft.parents, slots)
    assert ((out.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("hidden,width,tokens", [(64, 3, 1), (64, 3, 40), (2048, 3, 17), (30, 5, 3), (8, 16, 20)])
def test_convolution_of_a_chain_is_the_short_convolution(lib, hidden, width, tokens):
    """Output and history, bit for bit."""
    from runtime_b200.backend import CudaBackend

    draft = Draft([tokens], [tokens], "chain")
    projection, kernel, history = convolution_inputs(draft, hidden, width, 1)
    out = convolve(lib, draft, projection, kernel, history)
    after = torch.empty_like(history)
    paths, counts = dev(np.arange(tokens)), dev([tokens])
    st = lib.mfk_tree_convolution_keep(after.data_ptr(), history.data_ptr(), 1, projection.data_ptr(), tokens, paths.data_ptr(),
                                       counts.data_ptr(), None if tokens == 1 else at(draft.device["offsets"]), None, 1, hidden, width, stream())
    assert st == 0
    torch.cuda.synchronize()
    with CudaBackend(0) as be:
        y, h = be.allocate_f32((tokens, hidden)), be.upload_f32(history[0].cpu().numpy())
        be.gated_short_convolution(y, be.upload_f32(projection.cpu().numpy()), be.upload_f32(kernel.cpu().numpy()), h, (hidden, width))
        assert np.array_equal(be.read_f32(y), out.cpu().numpy())
        assert np.array_equal(be.read_f32(h), after[0].cpu().numpy())


@pytest.mark.parametrize("hidden,width", [(64, 3), (130, 4), (1, 2), (33, 16)])
@pytest.mark.parametrize("in_place", [True, False])
def test_histories_move_on(lib, hidden, width, in_place):
    rows = [1, 9, 0, 5, 30, 20, 3]
    draft = Draft(rows, rows, gap=2, behind=3)
    slots = [4, 7, 0, 1, 2, -1, 5]
    projection, _, history = convolution_inputs(draft, hidden, width, 8)
    rng = np.random.default_rng(3)
    paths, counts = np.full(draft.tokens, -1), np.zeros(len(rows), int)
    want = history.cpu().double()
    u = projection[:, :hidden] * projection[:, 2 * hidden :]
    for i, n in enumerate(rows):
        count = int(rng.integers(0, n + 1))
        path = np.sort(rng.choice(n, count, replace=False))
        paths[draft.offsets[i] : draft.offsets[i] + count], counts[i] = path, count
        if slots[i] >= 0:
            kept = torch.cat([want[slots[i]], u[draft.offsets[i] + torch.from_numpy(path).cuda().long()].cpu().double()])
            want[slots[i]] = kept[len(kept) - (width - 1) :]
    out = history if in_place else torch.full_like(history, 7.0)
    if not in_place:  # slots that no sequence names stay
        for s in (3, 6):
            want[s] = 7.0
    paths, counts, slots = dev(paths), dev(counts), dev(slots)
    st = lib.mfk_tree_convolution_keep(out.data_ptr(), history.data_ptr(), 8, projection.data_ptr(), draft.tokens, paths.data_ptr(),
                                       counts.data_ptr(), at(draft.device["offsets"]), slots.data_ptr(), len(rows), hidden, width, stream())
    assert st == 0
    torch.cuda.synchronize()
    assert torch.equal(out.cpu().double(), want)


# ---------------------------------------------------------------------
# Acceptance
# ---------------------------------------------------------------------

def accept(lib, cache, draft, drafted, sampled, pools, slots=None, n_pools=None):
    n = len(draft.rows)
    paths, counts = (torch.full((m,), 7, dtype=torch.int32, device="cuda") for m in (draft.tokens, n))
    nexts = torch.full((n,), 7.0, device="cuda")
    addresses = np.array([p.data_ptr() for p in pools], np.uint64)
    d = draft.device
    drafted, sampled = (dev(x, torch.float32) for x in (drafted, sampled))
    st = lib.mfk_paged_accept(paths.data_ptr(), counts.data_ptr(), nexts.data_ptr(), addresses.ctypes.data, len(pools), *cache.args()[2:],
                              drafted.data_ptr(), sampled.data_ptr(), draft.tokens, at(d["starts"]), at(d["offsets"]),
                              at(d["parents"]), at(slots), n, cache.kv_heads, cache.dim, stream())
    assert st == 0, lib.mf_last_error()
    torch.cuda.synchronize()
    return paths.cpu().numpy(), counts.cpu().numpy(), nexts.cpu().numpy()


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("shape", ["tree", "chain", "garbage"])
@pytest.mark.parametrize("kv_heads,dim,page,pools", [(2, 64, 16, 4), (1, 8, 1, 1), (3, 120, 7, 70), (8, 128, 64, 12), (2, 64, 16, 0)])
def test_acceptance(lib, dtype, shape, kv_heads, dim, page, pools):
    lengths, rows = LENGTHS + [90, 100], ROWS + [80, 100]
    cache = Cache(lengths, kv_heads, dim, page, dtype, fill=False)
    draft = Draft(lengths, rows, shape, gap=3, behind=6, seed=2)
    rng = np.random.default_rng(7)
    drafted, sampled = (rng.integers(0, 2, draft.tokens) for _ in range(2))  # few ids: long paths, siblings that agree
    drafted[-6:], sampled[draft.offsets[-2] :] = 1, 1
    drafted[draft.offsets[-2] : draft.offsets[-1]] = 1  # the last sequence: as far as its branches go
    g = torch.Generator(device="cuda").manual_seed(1)
    stores = [torch.randn(cache.keys.shape, generator=g, device="cuda").to(cache.dtype) for _ in range(pools)]
    want = [s.clone().cpu() for s in stores]
    paths, counts, nexts = accept(lib, cache, draft, drafted, sampled, stores)
    expected = np.full(draft.tokens, 7)
    longest = 0
    for i, n in enumerate(rows):
        first = draft.offsets[i]
        if n == 0:
            assert counts[i] == 0 and np.isnan(nexts[i])
            continue
        path, last = tree_ref.accept(drafted, sampled, draft.parents, first, n)
        longest = max(longest, len(path))
        expected[first : first + n] = path + [-1] * (n - len(path))
        assert counts[i] == len(path) and nexts[i] == last
        start = lengths[i] - n
        for w in want:
            rows_at = [w[int(cache.table[i, (start + r) // page]), :, (start + r) % page].clone() for r in path]
            for j, x in enumerate(rows_at):
                w[int(cache.table[i, (start + j) // page]), :, (start + j) % page] = x
    assert np.array_equal(paths, expected)
    assert longest == 100 if shape == "chain" else longest > 3 or shape == "garbage"
    for s, w in zip(stores, want):
        assert torch.equal(s.cpu(), w)


def test_acceptance_of_ids_that_are_none(lib):
    """A NaN draw ends the path; -0 equals 0; the first of equal children is taken."""
    cache = Cache([8] * 3, 1, 64, 16, "f32", fill=False)
    draft = Draft([8] * 3, [5] * 3)
    draft.device["parents"] = dev([-1, 0, 0, 1, 2] * 3)
    nan = float("nan")
    drafted = [9, nan, 4, 5, 6] + [9, 0.0, 0.0, 5, 5] + [1, 2, 3, 4, 5]
    sampled = [nan, 4, 6, 1, 1] + [-0.0, 5, 5, 7, 8] + [3, 0, 5, 0, nan]
    paths, counts, nexts = accept(lib, cache, draft, drafted, sampled, [])
    assert counts.tolist() == [1, 3, 3]
    assert paths.tolist() == [0, -1, -1, -1, -1, 0, 1, 3, -1, -1, 0, 2, 4, -1, -1]
    assert np.isnan(nexts[0]) and nexts[1] == 7 and np.isnan(nexts[2])


def test_acceptance_moves_nothing_to_places_that_do_not_exist(lib):
    cache = Cache([40] * 4, 2, 64, 16, "bf16", fill=False)
    cache.table[0, 2], cache.table[1, 2] = -1, cache.pages
    cache.device_table = dev(cache.table)
    draft = Draft([40] * 4, [6] * 4)
    draft.device["parents"] = dev([-1, 0, 0, 1, 2, 4] * 4)
    draft.device["starts"] = dev([34, 34, -3, 34])
    before = cache.keys.clone()
    paths, counts, _ = accept(lib, cache, draft, [1, 0, 1, 0, 1, 1] * 4, [1] * 24, [cache.keys], slots=dev([0, 1, 2, -1]))
    assert counts.tolist() == [4] * 4 and paths[:6].tolist() == [0, 2, 4, 5, -1, -1]
    assert torch.equal(cache.keys, before)
