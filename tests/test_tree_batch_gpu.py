"""Batches of so many rows that a CTA of the rotated append or of the convolution
takes several: rows of other sequences, of none, and a last CTA that is not full."""
import numpy as np
import pytest
import torch

import tree_ref
from paged_ref import PAGE_DTYPES
from test_tree_gpu import Cache, Draft, append, convolution_inputs, convolve, dev, lib, rounding, stream  # noqa: F401

pytestmark = pytest.mark.gpu


def batch(rows_in_all, shape, seed=1):
    """Ragged sequences, some without rows, of about so many rows; 3 rows before and 6 behind them."""
    rng = np.random.default_rng(seed)
    rows = []
    while sum(rows) < rows_in_all:
        rows.append(int(rng.choice([0, 1, 2, 3, int(rng.integers(4, 40))])))
    rows[-1] -= sum(rows) - rows_in_all
    lengths = [n + int(rng.integers(0, 30)) for n in rows]
    return lengths, Draft(lengths, rows, shape, seed=seed, gap=3, behind=6)


# A CTA takes two rows from 1,184 on, three from 1,776, four from 2,368.
@pytest.mark.parametrize("rows", [1290, 1801, 2377, 3601])
@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("q_heads,kv_heads,dim", [(8, 2, 64), (3, 1, 128), (5, 2, 40), (0, 3, 64), (33, 1, 64)])
def test_append_of_many_rows(lib, rows, dtype, q_heads, kv_heads, dim):  # noqa: F811
    lengths, draft = batch(rows, "tree")
    cache = Cache(lengths, kv_heads, dim, 16, dtype, fill=False)
    g = torch.Generator(device="cuda").manual_seed(3)
    n = draft.tokens
    q, k, v = (torch.randn(n, h, dim, generator=g, device="cuda") for h in (q_heads, kv_heads, kv_heads))
    weights = [torch.randn(dim, generator=g, device="cuda") for _ in range(2)]
    positions = np.random.default_rng(1).integers(0, 131071, n)
    before = [cache.keys.cpu().double(), cache.values.cpu().double()]
    out = append(lib, cache, draft, q if q_heads else None, k, v, weights, dev(positions))
    own = draft.owned()
    if q_heads:
        out = out.cpu()
        want, bound = tree_ref.rotated(q.cpu(), weights[0].cpu(), 1e-5, 1e6, positions)
        assert (out[~own] == 7.0).all()
        assert ((out.double() - want).abs() <= bound)[own].all()
    key, key_bound = tree_ref.rotated(k.cpu(), weights[1].cpu(), 1e-5, 1e6, positions)
    place = np.concatenate([np.arange(a - b, a) for a, b in zip(lengths, draft.rows)])
    seq = np.repeat(np.arange(len(lengths)), draft.rows)
    at, off = torch.from_numpy(cache.table[seq, place // 16]).long(), torch.from_numpy(place % 16)
    for pages, new, slack, old in ((cache.keys, key[own], key_bound[own], before[0]),
                                   (cache.values, v.cpu().double()[own], torch.zeros(int(own.sum()), kv_heads, dim).double(), before[1])):
        allowed = torch.zeros_like(old)
        old[at, :, off] = new
        allowed[at, :, off] = slack + rounding(new, cache.dtype)
        assert ((pages.cpu().double() - old).abs() <= allowed).all()


@pytest.mark.parametrize("rows", [1290, 2377, 3601])
@pytest.mark.parametrize("in_place", [True, False])
def test_append_of_many_rows_is_that_of_few(lib, rows, in_place):  # noqa: F811
    """Row by row the same bits as in calls of 100 rows, whose CTAs take one row each."""
    lengths, draft = batch(rows, "chain", seed=4)
    caches = [Cache(lengths, 2, 64, 16, "bf16", fill=False) for _ in range(2)]
    g = torch.Generator(device="cuda").manual_seed(5)
    n = draft.tokens
    q, k, v = (torch.randn(n, h, 64, generator=g, device="cuda") for h in (8, 2, 2))
    weights = [torch.randn(64, generator=g, device="cuda") for _ in range(2)]
    q_in = q.clone()
    whole = append(lib, caches[0], draft, q_in, k, v, weights, q_out=q_in if in_place else None)
    pieces = torch.full_like(q, 7.0)
    starts, offsets = draft.device["starts"].cpu().numpy(), draft.offsets
    for lo in range(0, n, 100):
        hi = min(n, lo + 100)
        cut = np.clip(offsets, lo, hi)
        part = Draft(lengths, np.diff(cut).tolist(), "chain")
        part.device["offsets"] = dev(cut - lo)
        part.device["starts"] = dev(starts + cut[:-1] - offsets[:-1])
        pieces[lo:hi] = append(lib, caches[1], part, q[lo:hi].contiguous(), k[lo:hi].contiguous(), v[lo:hi].contiguous(), weights)
    own = draft.owned().cuda()
    assert torch.equal(whole[own], pieces[own])
    assert torch.equal(whole[~own], q[~own] if in_place else torch.full_like(q[~own], 7.0))
    assert torch.equal(caches[0].keys, caches[1].keys) and torch.equal(caches[0].values, caches[1].values)


# Rows times parts of 512 channels (128 where they are no multiple of 4) over 888: rows of a CTA, eight at most.
@pytest.mark.parametrize("shape", ["tree", "chain", "garbage"])
@pytest.mark.parametrize("rows,hidden,width", [(1795, 2048, 3), (951, 1024, 3), (7201, 64, 3), (1795, 2052, 3), (1795, 2048, 4), (901, 1029, 3), (901, 1029, 2)])
def test_convolution_of_many_rows(lib, shape, rows, hidden, width):  # noqa: F811
    """Bit for bit the sums of the taps in order, each product and sum rounded to F32."""
    lengths, draft = batch(rows, shape, seed=2)
    projection, kernel, history = convolution_inputs(draft, hidden, width, len(lengths))
    out = convolve(lib, draft, projection, kernel, history)
    b, c, v = projection.split(hidden, 1)
    line = torch.cat([history.view(-1, hidden), b * v])  # every slot's entries, then the rows' products
    past, taps = len(lengths) * (width - 1), np.zeros((width, draft.tokens), np.int64)
    for i, n in enumerate(draft.rows):
        first = int(draft.offsets[i])
        for r in range(n):
            way = [past + first + a for a in tree_ref.ancestors(draft.parents, first, r)[:width]]
            way += [i * (width - 1) + width - 2 - j for j in range(width - len(way))]
            taps[:, first + r] = way[::-1]
    total = torch.zeros_like(out)
    for j in range(width):
        total = total + kernel[:, j] * line[torch.from_numpy(taps[j]).cuda()]
    want, own = total * c, draft.owned().cuda()
    assert torch.equal(out[own], want[own]) and (out[~own] == 7.0).all()
