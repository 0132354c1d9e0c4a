"""What the entry points of drafted trees refuse: every check runs on the host
before any device call, so none of these needs a GPU."""
import ctypes as C

import numpy as np
import pytest

from runtime_b200 import _lib

INVALID_ARGUMENT, INVALID_SHAPE, INVALID_LAYOUT, INVALID_DTYPE, OVERFLOW, OUT_OF_BOUNDS, UNSUPPORTED, RESOURCE = range(1, 9)
A = [(i + 1) << 28 for i in range(24)]  # stand-ins for device addresses, far apart: never read here
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def lib():
    from runtime_b200 import build

    build.build()
    return _lib.load()


def call(entry, defaults, kw):
    assert set(kw) <= set(defaults), set(kw) - set(defaults)
    return entry(*{**defaults, **kw}.values())


def gqa(lib, **kw):
    return call(lib.mfk_paged_tree_gqa, dict(
        out=A[0], q=A[1], keys=A[2], values=A[3], dtype=0, pages=4, page_tokens=16, table=A[4], slots=2, max_pages=4,
        tokens=6, lengths=A[5], offsets=A[6], parents=A[7], slot_ids=None, sequences=2, q_heads=8, kv_heads=2,
        head_dim=64, workspace=A[8], workspace_bytes=32 << 20, stream=None), kw)


def append(lib, **kw):
    return call(lib.mfk_paged_append_rope, dict(
        keys=A[2], values=A[3], dtype=0, pages=4, page_tokens=16, table=A[4], slots=2, max_pages=4, q_out=A[0], q=A[1],
        k=A[9], v=A[10], tokens=6, q_weight=A[11], k_weight=A[12], epsilon=1e-5, theta=1e6, positions=A[13], starts=A[14],
        offsets=A[6], slot_ids=None, sequences=2, q_heads=8, kv_heads=2, head_dim=64, stream=None), kw)


def convolution(lib, **kw):
    return call(lib.mfk_tree_convolution, dict(
        out=A[0], projection=A[1], kernel=A[2], history=A[3], slots=2, tokens=6, offsets=A[4], parents=A[5], slot_ids=None,
        sequences=2, hidden=64, width=3, stream=None), kw)


def keep(lib, **kw):
    return call(lib.mfk_tree_convolution_keep, dict(
        out=A[0], history=A[1], slots=2, projection=A[2], tokens=6, paths=A[3], counts=A[4], offsets=A[5], slot_ids=None,
        sequences=2, hidden=64, width=3, stream=None), kw)


POOLS = np.array(A[15:17], np.uint64)


def accept(lib, **kw):
    return call(lib.mfk_paged_accept, dict(
        paths=A[0], counts=A[1], next=A[2], pools=POOLS.ctypes.data, n_pools=2, dtype=0, pages=4, page_tokens=16,
        table=A[4], slots=2, max_pages=4, drafted=A[5], sampled=A[6], tokens=6, starts=A[7], offsets=A[8], parents=A[9],
        slot_ids=None, sequences=2, kv_heads=2, head_dim=64, stream=None), kw)


GEOMETRY = [
    (dict(dtype=3), INVALID_DTYPE), (dict(dtype=-1), INVALID_DTYPE), (dict(head_dim=0), INVALID_SHAPE),
    (dict(page_tokens=0), INVALID_SHAPE), (dict(kv_heads=0), INVALID_SHAPE), (dict(head_dim=60), UNSUPPORTED),
    (dict(head_dim=136), UNSUPPORTED), (dict(max_pages=1 << 28), OVERFLOW), (dict(pages=1 << 40), OVERFLOW),
    (dict(sequences=3), OUT_OF_BOUNDS), (dict(sequences=(1 << 20) + 1, slots=1 << 21), RESOURCE),
    (dict(tokens=1 << 31), OVERFLOW), (dict(table=None), INVALID_ARGUMENT), (dict(table=A[4] + 2), INVALID_LAYOUT),
    (dict(offsets=A[6] + 1), INVALID_LAYOUT), (dict(slot_ids=A[20] + 2), INVALID_LAYOUT),
]


@pytest.mark.parametrize("kw,status", GEOMETRY + [
    (dict(out=None), INVALID_ARGUMENT), (dict(q=None), INVALID_ARGUMENT), (dict(keys=None), INVALID_ARGUMENT),
    (dict(values=None), INVALID_ARGUMENT), (dict(lengths=None), INVALID_ARGUMENT), (dict(workspace=None), INVALID_ARGUMENT),
    (dict(workspace_bytes=(32 << 20) - 1), RESOURCE), (dict(q_heads=0), INVALID_SHAPE), (dict(q_heads=7), INVALID_SHAPE),
    (dict(tokens=1 << 28, q_heads=16), OVERFLOW), (dict(out=A[0] + 4), INVALID_LAYOUT), (dict(q=A[1] + 8), INVALID_LAYOUT),
    (dict(keys=A[2] + 8), INVALID_LAYOUT), (dict(workspace=A[8] + 4), INVALID_LAYOUT), (dict(parents=A[7] + 2), INVALID_LAYOUT),
    (dict(out=A[1]), INVALID_ARGUMENT), (dict(out=A[1] + 64), INVALID_ARGUMENT), (dict(out=A[2]), INVALID_ARGUMENT),
    (dict(workspace=A[0]), INVALID_ARGUMENT), (dict(workspace=A[7] - 64), INVALID_ARGUMENT), (dict(out=A[5] - 16), INVALID_ARGUMENT),
])
def test_tree_gqa_refuses(lib, kw, status):
    assert gqa(lib, **kw) == status
    assert lib.mf_last_error()


@pytest.mark.parametrize("kw,status", GEOMETRY + [
    (dict(q_out=None), INVALID_ARGUMENT), (dict(q=None), INVALID_ARGUMENT), (dict(k=None), INVALID_ARGUMENT),
    (dict(v=None), INVALID_ARGUMENT), (dict(starts=None), INVALID_ARGUMENT), (dict(keys=None), INVALID_ARGUMENT),
    (dict(values=A[2]), INVALID_ARGUMENT), (dict(values=A[2] + 1024), INVALID_ARGUMENT), (dict(q_heads=1 << 17), OVERFLOW),
    (dict(theta=0.0), INVALID_ARGUMENT), (dict(theta=NAN), INVALID_ARGUMENT), (dict(theta=INF), INVALID_ARGUMENT),
    (dict(theta=-1.0), INVALID_ARGUMENT), (dict(epsilon=0.0), INVALID_ARGUMENT), (dict(epsilon=NAN), INVALID_ARGUMENT),
    (dict(epsilon=INF), INVALID_ARGUMENT), (dict(q_weight=None, epsilon=-1.0), INVALID_ARGUMENT),
    (dict(q=A[1] + 4), INVALID_LAYOUT), (dict(k_weight=A[12] + 4), INVALID_LAYOUT), (dict(positions=A[13] + 2), INVALID_LAYOUT),
    (dict(q_out=A[1] + 256), INVALID_ARGUMENT), (dict(q_out=A[9]), INVALID_ARGUMENT), (dict(q_out=A[2]), INVALID_ARGUMENT),
    (dict(k=A[2]), INVALID_ARGUMENT), (dict(q=A[3], q_out=A[3]), INVALID_ARGUMENT), (dict(positions=A[2]), INVALID_ARGUMENT),
])
def test_append_rope_refuses(lib, kw, status):
    assert append(lib, **kw) == status


CONVOLUTION = [
    (dict(hidden=0), INVALID_ARGUMENT), (dict(width=0), INVALID_ARGUMENT), (dict(width=17), UNSUPPORTED),
    (dict(hidden=(1 << 24) + 4), OVERFLOW), (dict(tokens=1 << 31), OVERFLOW), (dict(sequences=3), OUT_OF_BOUNDS),
    (dict(sequences=(1 << 20) + 1, slots=1 << 21), RESOURCE), (dict(out=None), INVALID_ARGUMENT),
    (dict(projection=None), INVALID_ARGUMENT), (dict(history=None), INVALID_ARGUMENT), (dict(out=A[0] + 2), INVALID_LAYOUT),
    (dict(offsets=A[4] + 2), INVALID_LAYOUT),
]


@pytest.mark.parametrize("kw,status", CONVOLUTION + [
    (dict(kernel=None), INVALID_ARGUMENT), (dict(out=A[0] + 4), INVALID_LAYOUT), (dict(out=A[1] + 16), INVALID_ARGUMENT),
    (dict(out=A[3]), INVALID_ARGUMENT), (dict(out=A[5] - 16), INVALID_ARGUMENT), (dict(parents=A[5] + 1), INVALID_LAYOUT),
])
def test_tree_convolution_refuses(lib, kw, status):
    assert convolution(lib, **kw) == status


@pytest.mark.parametrize("kw,status", CONVOLUTION + [
    (dict(paths=None), INVALID_ARGUMENT), (dict(counts=None), INVALID_ARGUMENT), (dict(out=A[1] + 16), INVALID_ARGUMENT),
    (dict(out=A[2]), INVALID_ARGUMENT), (dict(out=A[3] - 16), INVALID_ARGUMENT), (dict(paths=A[3] + 2), INVALID_LAYOUT),
])
def test_tree_convolution_keep_refuses(lib, kw, status):
    assert keep(lib, **kw) == status


@pytest.mark.parametrize("kw,status", [g for g in GEOMETRY if "offsets" not in g[0]] + [
    (dict(paths=None), INVALID_ARGUMENT), (dict(counts=None), INVALID_ARGUMENT), (dict(next=None), INVALID_ARGUMENT),
    (dict(pools=None), INVALID_ARGUMENT), (dict(drafted=None), INVALID_ARGUMENT), (dict(sampled=None), INVALID_ARGUMENT),
    (dict(starts=None), INVALID_ARGUMENT), (dict(paths=A[0] + 2), INVALID_LAYOUT), (dict(paths=A[5]), INVALID_ARGUMENT),
    (dict(counts=A[0]), INVALID_ARGUMENT), (dict(next=A[1]), INVALID_ARGUMENT), (dict(next=A[9]), INVALID_ARGUMENT),
    (dict(paths=A[15]), INVALID_ARGUMENT), (dict(drafted=A[16] + 16), INVALID_ARGUMENT), (dict(parents=A[9] + 1), INVALID_LAYOUT),
])
def test_accept_refuses(lib, kw, status):
    assert accept(lib, **kw) == status


def test_accept_refuses_bad_pools(lib):
    page = 2 * 16 * 64 * 4
    for bad, status in (([A[15], 0], INVALID_ARGUMENT), ([A[15] + 8, A[16]], INVALID_LAYOUT), ([A[16], A[16]], INVALID_ARGUMENT),
                        ([A[16], A[16] - 4 * page + 16], INVALID_ARGUMENT)):
        pools = np.array(bad, np.uint64)
        assert accept(lib, pools=pools.ctypes.data) == status


def test_nothing_to_do_is_no_error_and_no_launch(lib):
    for f in (gqa, append, convolution):
        assert f(lib, sequences=0) == 0
        assert f(lib, tokens=0) == 0
    assert gqa(lib, tokens=0, out=None, q=None, keys=None, values=None, table=None) == 0
    assert keep(lib, sequences=0) == 0
    assert keep(lib, width=1, history=None, out=None) == 0
    assert accept(lib, sequences=0, counts=None) == 0


def test_workspace_size_is_the_headers():
    import os

    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "mfcuda.h")).read()
    from tree_ref import TREE_WORKSPACE

    assert "#define MF_PAGED_TREE_WORKSPACE_BYTES (32u << 20)" in text and TREE_WORKSPACE == 32 << 20
    assert C.sizeof(C.c_float) == 4


def test_tree_gqa_refuses_pools_of_more_rows_than_it_can_name(lib):
    far = dict(keys=1 << 40, values=1 << 42, page_tokens=64, kv_heads=2, q_heads=8)
    assert gqa(lib, pages=(1 << 24), **far) == OVERFLOW  # 2^31 rows
    assert gqa(lib, pages=(1 << 24), tokens=0, **far) == 0
