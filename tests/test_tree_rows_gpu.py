"""Which rows the operators over drafted trees take as a sequence's: offsets are
cut to [0, tokens), by all of them alike."""
import numpy as np
import pytest
import torch

from paged_ref import PAGE_DTYPES
from test_tree_gpu import Cache, Draft, accept, append, attend, convolution_inputs, convolve, dev, lib, queries, stream  # noqa: F401

pytestmark = pytest.mark.gpu

# (offsets, what the cut makes of them) of 12 rows.
CUTS = [
    ([-5, 4, 9], [0, 4, 9]),  # one sequence begins before the first row
    ([-9, -2, 7], [0, 0, 7]),  # one lies before it
    ([-2**31, 3, 2**31 - 1], [0, 3, 12]),
    ([2, 8, 40], [2, 8, 12]),
    ([3, 15, 40], [3, 12, 12]),
    ([-3, 0, 0], [0, 0, 0]),
]
TOKENS = 12


def drafts(cut):
    """The same sequences under both sets of offsets; the tree's rows name places among those that are left."""
    offsets, left = cut
    rows = np.diff(left).tolist()
    lengths = [30 + n for n in rows]
    pair = []
    for device in (offsets, left):
        d = Draft(lengths, rows, seed=3)
        d.tokens = TOKENS
        parents = np.full(TOKENS, -1)
        for first, n in zip(left, rows):
            parents[first : first + n] = [max(-1, r - 1 - r % 2) for r in range(n)]
        d.device["parents"], d.device["offsets"] = dev(parents), dev(device)
        pair.append(d)
    return lengths, left, pair


@pytest.mark.parametrize("cut", CUTS)
@pytest.mark.parametrize("dtype", PAGE_DTYPES)
def test_attention_and_append_take_the_same_rows(lib, cut, dtype):  # noqa: F811
    lengths, left, pair = drafts(cut)
    q = queries(TOKENS, 4, 64)
    cache = Cache(lengths, 2, 64, 16, dtype, fill=False)
    outs = [attend(lib, cache, d, q) for d in pair]
    assert torch.equal(*outs)
    own = torch.zeros(TOKENS, dtype=torch.bool)
    own[left[0] : left[-1]] = True
    assert (outs[0].cpu()[~own] == 7.0).all() and (outs[0].cpu()[own] != 7.0).any(2).all()
    k, v = queries(TOKENS, 2, 64, 5), queries(TOKENS, 2, 64, 6)
    caches = [Cache(lengths, 2, 64, 16, dtype, fill=False) for _ in pair]
    before = caches[0].keys.clone()
    turned = [append(lib, c, d, q, k, v, (None, None)) for c, d in zip(caches, pair)]
    assert torch.equal(*turned) and torch.equal(caches[0].keys, caches[1].keys) and torch.equal(caches[0].values, caches[1].values)
    assert (turned[0].cpu()[~own] == 7.0).all()
    # The rows written are those at the places that the attention takes for the sequence's last tokens.
    written = (caches[0].keys != before).any(3).any(1).cpu()
    places = torch.zeros_like(written)
    for i, n in enumerate(np.diff(left)):
        pos = np.arange(lengths[i] - n, lengths[i])
        places[cache.table[i, pos // 16], pos % 16] = True
    assert torch.equal(written, places)


@pytest.mark.parametrize("cut", CUTS)
@pytest.mark.parametrize("shape", ["tree", "chain"])
def test_convolution_and_acceptance_take_the_same_rows(lib, cut, shape):  # noqa: F811
    lengths, left, pair = drafts(cut)
    if shape == "chain":
        for d in pair:
            d.device["parents"] = None
    projection, kernel, history = convolution_inputs(pair[0], 64, 3, 2)
    outs = [convolve(lib, d, projection, kernel, history) for d in pair]
    assert torch.equal(*outs)
    inside = torch.zeros(TOKENS, dtype=torch.bool)
    inside[left[0] : left[-1]] = True
    assert (outs[0].cpu()[~inside] == 7.0).all() and (outs[0].cpu()[inside] != 7.0).any(1).all()
    cache = Cache(lengths, 2, 64, 16, "f32", fill=False)
    ids = np.zeros(TOKENS)
    results, stores, kept = [], [cache.keys.clone(), cache.keys.clone()], []
    for d, store in zip(pair, stores):
        results.append(accept(lib, cache, d, ids, ids, [store]))
        paths, counts, _ = results[-1]
        after = history.clone()
        device = [dev(paths), dev(counts)]
        assert lib.mfk_tree_convolution_keep(after.data_ptr(), after.data_ptr(), 2, projection.data_ptr(), TOKENS, device[0].data_ptr(),
                                             device[1].data_ptr(), d.device["offsets"].data_ptr(), None, 2, 64, 3, stream()) == 0
        torch.cuda.synchronize()
        kept.append(after)
    for a, b in zip(*results):
        assert np.array_equal(a, b, equal_nan=True)
    assert torch.equal(*stores) and torch.equal(*kept)
    for i, n in enumerate(np.diff(left)):
        assert (results[0][1][i] > 0) == (n > 0)
