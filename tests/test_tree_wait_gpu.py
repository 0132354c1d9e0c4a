"""Waits of the tree attention that run out: the call returns, what it could not
compute is NaN, the host reads the fault, and the next call is right again."""
import ctypes as C

import numpy as np
import pytest
import torch

from paged_ref import PAGE_DTYPES
from test_tree_gpu import Cache, Draft, attend, check, lib, queries, workspace  # noqa: F401

pytestmark = pytest.mark.gpu
MOST = 1 << 22


def faults(lib):  # noqa: F811
    v = C.c_uint32(7)
    assert lib.mf_device_faults(C.byref(v)) == 0
    return v.value


def limited(lib, tries, cache, draft, q, ws):  # noqa: F811
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    assert lib.mf_set_tree_wait(tries) == 0
    try:
        start.record()
        out = attend(lib, cache, draft, q, ws=ws)
        end.record()
    finally:
        assert lib.mf_set_tree_wait(MOST) == 0
    torch.cuda.synchronize()
    assert start.elapsed_time(end) < 1000  # (nothing waits for loads that were never issued: that takes seconds)
    return out.cpu().double()


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths,rows", [([2000], [8]), ([1, 1500, 0, 700, 90], [1, 30, 0, 3, 90])])
def test_calls_that_give_up_at_once(lib, dtype, dim, lengths, rows):  # noqa: F811
    cache = Cache(lengths, 2, dim, 16, dtype, seed=3)
    draft = Draft(lengths, rows, seed=2)
    q = queries(draft.tokens, 8, dim)
    ws = workspace()
    right = attend(lib, cache, draft, q, ws=ws)
    assert faults(lib) == 0
    assert limited(lib, 0, cache, draft, q, ws).isnan().all()
    assert faults(lib) == 1 and faults(lib) == 0
    again = attend(lib, cache, draft, q, ws=ws)
    assert torch.equal(again, right) and faults(lib) == 0
    check(again, cache, draft, q)


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_waits_of_a_single_try(lib, dtype, dim):  # noqa: F811
    """Whichever of them run out, loads and products under way: what is no NaN is right, and without a fault all is."""
    lengths, rows = [3000] * 24 + [40] * 8, [7] * 24 + [40] * 8
    cache = Cache(lengths, 4, dim, 16, dtype, seed=3)
    draft = Draft(lengths, rows, seed=2)
    q = queries(draft.tokens, 16, dim)
    ws = workspace()
    right = attend(lib, cache, draft, q, ws=ws)
    faults(lib)
    for _ in range(4):
        torch.empty(200 << 20, dtype=torch.uint8, device="cuda").zero_()  # (loads from memory, not from L2)
        out = limited(lib, 1, cache, draft, q, ws)
        assert out.isnan().any() == (faults(lib) == 1)
        assert (out.isnan() | (out == right.cpu().double())).all()
    assert torch.equal(attend(lib, cache, draft, q, ws=ws), right) and faults(lib) == 0


def test_no_wait_of_an_ordinary_call_runs_out(lib):  # noqa: F811
    faults(lib)
    rng = np.random.default_rng(4)
    for dtype in PAGE_DTYPES:
        for dim in (64, 128):
            lengths = [int(n) for n in rng.integers(1, 4000, 20)]
            rows = [int(rng.integers(0, min(n, 40) + 1)) for n in lengths]
            cache, draft = Cache(lengths, 2, dim, 16, dtype), Draft(lengths, rows)
            assert attend(lib, cache, draft, queries(draft.tokens, 8, dim)).isfinite().all()
    assert faults(lib) == 0
