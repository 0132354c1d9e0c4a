"""Acceptance of more rows than a warp holds (128): chunks of prompts, large trees."""
import numpy as np
import pytest
import torch

import tree_ref
from paged_ref import PAGE_DTYPES
from test_tree_gpu import Cache, Draft, accept, lib  # noqa: F401

pytestmark = pytest.mark.gpu

ROWS = [129, 500, 2500, 128, 0, 160]
LENGTHS = [129, 517, 2600, 200, 30, 161]


def expected(draft, drafted, sampled):
    """paths, counts and next of every sequence."""
    paths, counts, nexts = np.full(draft.tokens, 7), [], []
    for i, n in enumerate(draft.rows):
        first = draft.offsets[i]
        path, last = tree_ref.accept(drafted, sampled, draft.parents, first, n) if n else ([], np.nan)
        paths[first : first + n] = path + [-1] * (n - len(path))
        counts.append(len(path)), nexts.append(last)
    return paths, np.array(counts), np.array(nexts, np.float32)


def check(lib, draft, drafted, sampled, dtype="f32", pools=2):  # noqa: F811
    cache = Cache(LENGTHS, 2, 64, 16, dtype, fill=False)
    g = torch.Generator(device="cuda").manual_seed(1)
    stores = [torch.randn(cache.keys.shape, generator=g, device="cuda").to(cache.dtype) for _ in range(pools)]
    want = [s.clone().cpu() for s in stores]
    paths, counts, nexts = accept(lib, cache, draft, drafted, sampled, stores)
    e_paths, e_counts, e_nexts = expected(draft, drafted, sampled)
    assert np.array_equal(counts, e_counts) and np.array_equal(paths, e_paths)
    assert np.array_equal(nexts, e_nexts, equal_nan=True)
    for i, n in enumerate(draft.rows):
        path = e_paths[draft.offsets[i] : draft.offsets[i] + e_counts[i]]
        start = LENGTHS[i] - n
        fro, to = start + path, start + np.arange(len(path))
        for w in want:
            w[cache.table[i, to // 16], :, to % 16] = w[cache.table[i, fro // 16], :, fro % 16]
    for s, w in zip(stores, want):
        assert torch.equal(s.cpu(), w)
    return e_counts


@pytest.mark.parametrize("parents", [True, False])
@pytest.mark.parametrize("end", [None, 0, 1, 31, 32, 127, 128, 129, 158])
def test_chains(lib, parents, end):  # noqa: F811
    """As prompts enter: all rows of the longest agree, or all up to one."""
    draft = Draft(LENGTHS, ROWS, "chain", gap=3, behind=6)
    if parents:
        draft.parents = np.full(draft.tokens, -1)
        for first, n in zip(draft.offsets, ROWS):
            draft.parents[first : first + n] = np.arange(-1, n - 1)
        draft.device["parents"] = torch.from_numpy(draft.parents.astype(np.int32)).cuda()
    rng = np.random.default_rng(3)
    drafted = rng.integers(0, 60000, draft.tokens)
    sampled = np.append(drafted[1:], 5)
    if end is not None:
        for first in draft.offsets[:-1]:
            sampled[first + end] = -1
    counts = check(lib, draft, drafted, sampled)
    # (An end past a short sequence's rows is one of the next sequence's.)
    assert counts[2] == (2500 if end is None else end + 1)


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("shape", ["far", "tree", "garbage"])
@pytest.mark.parametrize("seed", [1, 2, 3])
def test_trees(lib, dtype, shape, seed):  # noqa: F811
    draft = Draft(LENGTHS, ROWS, shape, gap=3, behind=6, seed=seed)
    if shape != "garbage":  # "far": a branch of the even rows, the odd ones leaves beside it
        for first, n in zip(draft.offsets, ROWS):
            draft.parents[first : first + n] = [max(-1, r - 1 - r % 3 if shape == "tree" else r - 2 - r % 2) for r in range(n)]
        draft.device["parents"] = torch.from_numpy(draft.parents.astype(np.int32)).cuda()
    rng = np.random.default_rng(seed)
    few = 1 if shape != "garbage" and seed == 1 else 2
    drafted, sampled = (rng.integers(0, few, draft.tokens) for _ in range(2))
    counts = check(lib, draft, drafted, sampled, dtype, pools=3)
    if shape == "far" and few == 1:  # all ids alike: a path that goes on to the end, and skips rows on the way
        assert 800 < counts.max() < 2500


@pytest.mark.parametrize("width", [2, 3])
def test_a_prompt_chunk_is_accepted_whole_and_moves_its_histories_on(width):
    """The handle tier: a chunk of 300 rows, all kept; a layer's histories are its last rows'."""
    from runtime_b200.backend import CudaBackend, PagedCache

    hidden, rows = 96, [300, 0, 140]
    rng = np.random.default_rng(2)
    with CudaBackend(0) as be:
        cache = PagedCache(be, 1, 2, 64, pages=60, sequences=4, max_pages=40)
        cache.begin([2, 0, 3], rows)
        n = sum(rows)
        ids = rng.integers(0, 60000, n).astype(np.float32)
        drawn = np.append(ids[1:], 9.0).astype(np.float32)
        drawn[299] = 11.0
        projection = rng.standard_normal((n, 3 * hidden)).astype(np.float32)
        before = rng.standard_normal((4, width - 1, hidden)).astype(np.float32)
        history, device = be.upload_f32(before), be.upload_f32(projection)
        kept = cache.accept(be.upload_f32(ids), be.upload_f32(drawn))
        assert [p for p, _ in kept] == [list(range(300)), [], list(range(140))]
        assert kept[0][1] == 11.0 and kept[2][1] == 9.0
        cache.convolution_keep(history, device, width)
        want = before.copy()
        u = projection[:, :hidden] * projection[:, 2 * hidden :]
        want[2], want[3] = u[300 - width + 1 : 300], u[n - width + 1 :]
        assert np.array_equal(be.read_f32(history), want)
        assert [cache.sequence(s)[0] for s in range(4)] == [0, 0, 300, 140]
        cache.close()
