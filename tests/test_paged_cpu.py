"""What the paged-cache and sampling entry points refuse: every check runs on
the host before any device call, so none of these needs a GPU."""
import ctypes as C
import os

import numpy as np
import pytest

from runtime_b200 import _lib

INVALID_ARGUMENT, INVALID_SHAPE, INVALID_LAYOUT, INVALID_DTYPE, OVERFLOW, OUT_OF_BOUNDS, UNSUPPORTED, RESOURCE = range(1, 9)
A, B = 1 << 20, 1 << 21  # stand-ins for device addresses: never read here


@pytest.fixture(scope="module")
def lib():
    from runtime_b200 import build

    build.build()
    return _lib.load()


def gqa(lib, **kw):
    a = dict(out=A, q=B, keys=A, values=B, dtype=0, pages=4, page_tokens=16, table=A, slots=2, max_pages=4, lengths=A,
             slot_ids=None, sequences=2, q_heads=8, kv_heads=2, head_dim=64, workspace=A, workspace_bytes=8 << 20,
             stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.mfk_paged_gqa(*a.values())


def append(lib, **kw):
    a = dict(keys=A, values=B, dtype=0, pages=4, page_tokens=16, table=A, slots=2, max_pages=4, k=A, v=A, tokens=2,
             starts=A, row_offsets=None, slot_ids=None, sequences=2, kv_heads=2, head_dim=64, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.mfk_paged_append(*a.values())


GEOMETRY = [
    (dict(dtype=3), INVALID_DTYPE), (dict(dtype=-1), INVALID_DTYPE), (dict(head_dim=0), INVALID_SHAPE),
    (dict(page_tokens=0), INVALID_SHAPE), (dict(kv_heads=0), INVALID_SHAPE), (dict(head_dim=60), UNSUPPORTED),
    (dict(head_dim=136), UNSUPPORTED), (dict(max_pages=1 << 28), OVERFLOW), (dict(pages=1 << 40), OVERFLOW), (dict(pages=1 << 28), OVERFLOW),
    (dict(sequences=3), OUT_OF_BOUNDS), (dict(sequences=(1 << 20) + 1, slots=1 << 21), RESOURCE),
    (dict(keys=None), INVALID_ARGUMENT), (dict(values=None), INVALID_ARGUMENT), (dict(table=None), INVALID_ARGUMENT),
    (dict(keys=A + 8), INVALID_LAYOUT), (dict(values=B + 2), INVALID_LAYOUT), (dict(table=A + 2), INVALID_LAYOUT),
]


@pytest.mark.parametrize("kw,status", GEOMETRY + [
    (dict(out=None), INVALID_ARGUMENT), (dict(q=None), INVALID_ARGUMENT), (dict(q=A), INVALID_ARGUMENT), (dict(lengths=None), INVALID_ARGUMENT),
    (dict(workspace=None), INVALID_ARGUMENT), (dict(workspace_bytes=(8 << 20) - 1), RESOURCE),
    (dict(q_heads=0), INVALID_SHAPE), (dict(q_heads=7), INVALID_SHAPE), (dict(out=A + 4), INVALID_LAYOUT),
    (dict(workspace=A + 4), INVALID_LAYOUT),
])
def test_paged_gqa_refuses(lib, kw, status):
    assert gqa(lib, **kw) == status
    assert lib.mf_last_error()


@pytest.mark.parametrize("kw,status", GEOMETRY[:-3] + [
    (dict(k=None), INVALID_ARGUMENT), (dict(starts=None), INVALID_ARGUMENT), (dict(v=A + 4), INVALID_LAYOUT),
    (dict(values=A), INVALID_ARGUMENT), (dict(tokens=1 << 31), OVERFLOW), (dict(row_offsets=A + 1), INVALID_LAYOUT),
])
def test_paged_append_refuses(lib, kw, status):
    assert append(lib, **kw) == status


def test_nothing_to_do_is_no_error_and_no_launch(lib):
    assert gqa(lib, sequences=0, out=None, q=None) == 0
    assert append(lib, tokens=0, k=None, v=None) == 0
    assert append(lib, sequences=0) == 0
    assert lib.mfk_copy_pages(None, 0, 4, 64, None, None, 0, None) == 0
    assert lib.mfk_sample(None, None, 0, 8, None, None, None, None, None, None) == 0


def copy(lib, sources, destinations, pages=8, page_bytes=64, pools=(A,), n=None):
    s, d = (np.array(x, np.uint32) for x in (sources, destinations))
    p = np.array(pools, np.uint64)
    return lib.mfk_copy_pages(p.ctypes.data, len(p), pages, page_bytes, s.ctypes.data, d.ctypes.data,
                              len(s) if n is None else n, None)


@pytest.mark.parametrize("kw,status", [
    (dict(sources=[8], destinations=[0]), OUT_OF_BOUNDS), (dict(sources=[0], destinations=[8]), OUT_OF_BOUNDS),
    (dict(sources=[0, 1], destinations=[2, 2]), INVALID_ARGUMENT),     # one destination twice
    (dict(sources=[0, 2], destinations=[2, 3]), INVALID_ARGUMENT),     # a chain
    (dict(sources=[0, 1], destinations=[1, 0]), INVALID_ARGUMENT),     # a swap
    (dict(sources=[5], destinations=[5]), INVALID_ARGUMENT),
    (dict(sources=[0] * 9, destinations=range(9)), INVALID_ARGUMENT),
    (dict(sources=[0], destinations=[1], page_bytes=24), INVALID_LAYOUT),
    (dict(sources=[0], destinations=[1], page_bytes=0), INVALID_LAYOUT),
    (dict(sources=[0], destinations=[1], pools=(A + 8,)), INVALID_LAYOUT),
    (dict(sources=[0], destinations=[1], pools=(A, 0)), INVALID_ARGUMENT),
    (dict(sources=[0], destinations=[1], pages=1 << 33), OVERFLOW),
])
def test_copy_pages_refuses(lib, kw, status):
    assert copy(lib, **kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(width=0), INVALID_SHAPE), (dict(width=(1 << 24) + 1), OVERFLOW), (dict(rows=1 << 31), OVERFLOW),
    (dict(out=None), INVALID_ARGUMENT), (dict(logits=None), INVALID_ARGUMENT), (dict(temperature=None), INVALID_ARGUMENT),
    (dict(uniform=None), INVALID_ARGUMENT), (dict(logits=A + 2), INVALID_LAYOUT), (dict(top_k=A + 1), INVALID_LAYOUT),
])
def test_sample_refuses(lib, kw, status):
    a = dict(out=A, logits=A, rows=2, width=16, temperature=A, top_k=None, top_p=None, min_p=None, uniform=A, stream=None)
    a.update(kw)
    assert lib.mfk_sample(*a.values()) == status


def test_reference_sampler_known_answers():
    """The plain sampler that the GPU tests compare with, on rows done by hand."""
    from paged_ref import sample

    x = np.log([0.1, 0.4, 0.2, 0.3])
    assert [sample(x, 1, 0, 1, 0, u) for u in (0.0, 0.05, 0.15, 0.55, 0.75)] == [0, 0, 1, 2, 3]
    assert [sample(x, 1, 2, 1, 0, u) for u in (0.0, 0.5, 0.6, 0.99)] == [1, 1, 3, 3]     # 0.4 and 0.3 stay
    assert [sample(x, 1, 0, 0.65, 0, u) for u in (0.1, 0.9)] == [1, 3]                    # 0.4 + 0.3 reach 0.65
    assert [sample(x, 1, 0, 1, 0.6, u) for u in (0.1, 0.9)] == [1, 3]                     # at least 0.24
    assert sample([1, 3, 3, 2], 0, 0, 1, 0, 0.9) == 1
    assert sample([2, 2, 2, 2], 1, 2, 1, 0, 0.99) == 1                                    # ties: the lowest indexes
    assert sample([-np.inf, 0, -np.inf], 1, 0, 1, 0, 0.5) == 1
    assert np.isnan(sample([np.nan, 0], 1, 0, 1, 0, 0.5)) and np.isnan(sample([-np.inf] * 2, 1, 0, 1, 0, 0.5))


def test_paged_gqa_refuses_a_capacity_past_its_work_list(lib):
    """The table's capacity, not the lengths, decides: those are on the device."""
    big = dict(sequences=1 << 20, slots=1 << 20, q_heads=8, kv_heads=8, page_tokens=1 << 20, max_pages=(1 << 11) - 1)
    assert gqa(lib, **big) == OVERFLOW
    assert gqa(lib, sequences=1 << 20, slots=1 << 20, q_heads=16, kv_heads=8) == OVERFLOW  # 2^24 query rows


def test_uniform_numbers_below_one_stay_below_one():
    from runtime_b200.backend import uniform_array

    below = 1.0 - 2.0**-24  # F32's largest
    got = uniform_array([0.0, 0.25, below, 1.0 - 2.0**-26, 1.0 - 2.0**-53, 1.0, 1.5, -0.5, np.nan])
    assert got.dtype == np.float32 and got.flags.c_contiguous
    np.testing.assert_array_equal(got, np.array([0.0, 0.25, below, below, below, 1.0, 1.5, -0.5, np.nan], np.float32))
    assert float(uniform_array(1.0 - 2.0**-53)) == below
    f = np.random.default_rng(0).random(1000).astype(np.float32)
    assert np.array_equal(uniform_array(f), f)


def test_the_largest_uniform_number_is_passed_on_below_one(monkeypatch):
    """A state's and a batch's draw hand over what uniform_array gives."""
    from runtime_b200 import lfm2
    from runtime_b200.backend import Sampling

    seen = []

    class Lib:
        @staticmethod
        def mf_lfm2_sample(model, state, params, uniform):
            seen.append(np.float32(uniform))
            return 0

        @staticmethod
        def mf_lfm2_batch_sample(batch, params, n, at):
            seen.extend(np.ctypeslib.as_array(C.cast(at, C.POINTER(C.c_float)), (2,)).copy())
            return 0

    class Model:
        handle = None

    monkeypatch.setattr(lfm2._lib, "load", lambda: Lib)
    lfm2.Lfm2State(Model, None).sample(Sampling(), 1.0 - 2.0**-53)
    lfm2.Lfm2Batch(Model, None, 2).sample(Sampling(), [0.5, 1.0 - 2.0**-30])
    below = np.float32(1.0 - 2.0**-24)
    assert seen == [below, np.float32(0.5), below]


@pytest.mark.parametrize("q", [A - 4096 + 16, A, A + 16, A + 4096 - 16])
def test_paged_gqa_refuses_a_query_that_its_output_overlaps(lib, q):
    assert gqa(lib, out=A, q=q, keys=B, values=B + 4096) == INVALID_ARGUMENT  # rows of 2 x 8 x 64 floats


@pytest.mark.parametrize("kw", [
    dict(logits=A), dict(logits=A - 4 * 31), dict(logits=A + 4), dict(top_k=A), dict(top_p=A), dict(top_k=A + 4), dict(top_p=A - 4),
    dict(temperature=A + 4), dict(min_p=A - 4), dict(uniform=A + 4),
])
def test_sample_refuses_an_output_that_overlaps_its_inputs(lib, kw):
    a = dict(out=A, logits=B, rows=2, width=16, temperature=B, top_k=None, top_p=None, min_p=None, uniform=B, stream=None)
    a.update(kw)
    assert lib.mfk_sample(*a.values()) == INVALID_ARGUMENT
