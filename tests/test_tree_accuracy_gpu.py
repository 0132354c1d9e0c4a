"""How exact the tree attention's scores are, and its outputs where trees are
split over many CTAs."""
import numpy as np
import pytest
import torch

import tree_ref
from paged_ref import PAGE_DTYPES
from test_tree_gpu import Cache, Draft, attend, dev, lib, queries, stream, workspace  # noqa: F401
from tree_ref import TREE_WORKSPACE, U

pytestmark = pytest.mark.gpu


def excess_of_scores(lib, dtype, dim, size, single):  # noqa: F811
    """The relative excess of 4,096 scores of `size`, read off the weights of two tokens:
    the second has a key of zeros and alone a value, 1, so out = 1 / (1 + e^s)."""
    n, heads = 512, 8
    code, t = PAGE_DTYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(dim)
    k, q = (torch.randn(n, heads, dim, generator=g, device="cuda") for _ in range(2))
    if single:  # a score of one product
        k[..., 1:] = 0.0
        k[..., 0] = 1.0 + k[..., 0].abs() / 8
    k = k.to(t)
    kd = k.double()
    q = 2 * q.double() * (0.0 if single else 1.0)
    q = (q + ((size * dim**0.5 - (q * kd).sum(2)) / kd.square().sum(2))[..., None] * kd).float()
    s = (q.double() * kd).sum(2) / dim**0.5
    keys, values = (torch.zeros(n, heads, 2, dim, dtype=t, device="cuda") for _ in range(2))
    keys[:, :, 0], values[:, :, 1] = k, 1.0
    out, table, lengths, ws = torch.empty_like(q), dev(np.arange(n)[:, None]), dev([2] * n), workspace()
    st = lib.mfk_paged_tree_gqa(out.data_ptr(), q.data_ptr(), keys.data_ptr(), values.data_ptr(), code, n, 2, table.data_ptr(), n, 1,
                                n, lengths.data_ptr(), None, None, None, n, heads, heads, dim, ws.data_ptr(), TREE_WORKSPACE, stream())
    assert st == 0, lib.mf_last_error()
    torch.cuda.synchronize()
    o = out.double()[..., 0]
    return ((torch.log(1 - o) - torch.log(o) - s) / s).mean().item()


@pytest.mark.parametrize("dtype,size", [("f32", 9.0), ("f32", 40.0), ("f16", 9.0), ("bf16", 9.0), ("bf16", 40.0)])
@pytest.mark.parametrize("dim", [8, 16, 32, 64, 72, 80, 96, 112, 120, 128])
def test_scores_are_neither_too_small_nor_too_large(lib, dtype, dim, size):  # noqa: F811
    """The tensor core cuts sums, by some 0.4e-7 to 1.9e-7 of a score; the scale makes up for
    it.  What is left is within half a step of F32 on the average, at every head dimension and
    page type (the roundings of the queries times the scale add nothing to a mean of 4,096); the
    exponential may add its 2^-22, which is 2^-22 / size of a score."""
    assert abs(excess_of_scores(lib, dtype, dim, size, False)) <= U + 2.0**-22 / size


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("dim", [8, 64, 120, 128])
def test_scores_of_a_single_product(lib, dtype, dim):  # noqa: F811
    """Nothing is cut where one product is the sum: such a score comes out too large by what the
    scale holds more, 1.94e-7 at most, less than 4 U."""
    assert abs(excess_of_scores(lib, dtype, dim, 9.0, True)) <= 4 * U + 2.0**-22 / 9


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("shape", ["tree", "chain", "garbage"])
@pytest.mark.parametrize("length,rows,page,heads,dim", [
    (5000, 33, 24, (8, 2), 64), (20011, 9, 7, (3, 1), 128), (20011, 100, 24, (6, 2), 64), (5000, 70, 1, (4, 2), 80), (20011, 21, 64, (16, 1), 128),
])
def test_error_of_trees_that_are_split(lib, dtype, shape, length, rows, page, heads, dim):  # noqa: F811
    """At most 16 U of the output's norm (tests/test_paged_accuracy.py derives it).  A single
    token that a row sees and should not, or the other way round, moves the row by some 1e-2 to
    1e-3 of its norm: thousands of U."""
    cache = Cache([length], heads[1], dim, page, dtype, seed=length + rows)
    draft = Draft([length], [rows], shape, seed=rows)
    q = queries(rows, heads[0], dim)
    got = attend(lib, cache, draft, q).double()
    pos = torch.arange(length)
    where = torch.from_numpy(cache.table[0]).long()[pos // page].cuda(), (pos % page).cuda()
    k, v = (x[where[0], :, where[1]].double().repeat_interleave(heads[0] // heads[1], 1) for x in (cache.keys, cache.values))
    seen = torch.ones(rows, length, dtype=torch.bool)
    seen[:, length - rows :] = False
    for r in range(rows):
        seen[r, [length - rows + a for a in tree_ref.ancestors(draft.parents, 0, r)]] = True
    s = torch.einsum("rhd,nhd->rhn", q.double(), k) / dim**0.5
    p = torch.softmax(s.masked_fill(~seen.cuda()[:, None], -np.inf), 2)
    want = torch.einsum("rhn,nhd->rhd", p, v)
    assert ((got - want).norm() / want.norm()).item() <= 16 * U
    # The rows one by one: less is averaged, so each may be off by four times as much (its largest weight alone).
    assert ((got - want).norm(dim=2) / want.norm(dim=2)).max().item() <= 64 * U
