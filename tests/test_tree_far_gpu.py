"""Pools of more than 2^32 bytes, and of more than 2^31 values: a pass whose pages lie
at their ends is the pass over a small pool, bit for bit."""
import numpy as np
import pytest
import torch

from paged_ref import PAGE_DTYPES
from test_tree_gpu import Cache, Draft, accept, append, attend, dev, lib, queries  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,pages", [("f32", 1_100_000), ("bf16", 2_200_000)])
@pytest.mark.parametrize("page", [16, 5])
def test_pages_past_32_bits(lib, dtype, pages, page):  # noqa: F811
    kv_heads, dim, lengths, rows = 2, 64, [400, 33, 150], [20, 33, 7]
    pages = pages * 16 // page
    near = Cache(lengths, kv_heads, dim, page, dtype, fill=False)
    far = Cache(lengths, kv_heads, dim, page, dtype, fill=False)
    if torch.cuda.mem_get_info()[0] < 4 * pages * kv_heads * page * dim * far.keys.element_size():
        pytest.skip("not enough memory")
    # The near pool's pages, in their order, are the far one's last.
    first = pages - near.pages
    far.pages, far.table = pages, np.where(near.table >= 0, near.table + first, -1).astype(np.int32)
    far.device_table = dev(far.table)
    for name in ("keys", "values"):
        pool = torch.empty(pages, kv_heads, page, dim, dtype=far.dtype, device="cuda")
        pool[first:] = getattr(near, name)
        pool[: near.pages] = float("nan")  # where the places cut to 32 bits would lie
        setattr(far, name, pool)
    assert far.keys.numel() > 2**31 and far.keys.numel() * far.keys.element_size() > 2**32
    draft = Draft(lengths, rows)
    q, k, v = queries(60, 8, dim), queries(60, kv_heads, dim, 2), queries(60, kv_heads, dim, 3)
    rng = np.random.default_rng(1)
    drafted, sampled = (rng.integers(0, 2, 60) for _ in range(2))
    results = []
    for cache in (near, far):
        turned = append(lib, cache, draft, q, k, v, (None, None))
        out = attend(lib, cache, draft, turned)
        moved = accept(lib, cache, draft, drafted, sampled, [cache.keys, cache.values])
        results.append((turned, out, *(torch.from_numpy(x) for x in moved), cache.keys[-near.pages :], cache.values[-near.pages :]))
    assert max(results[0][3]) > 2  # (rows moved)
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert far.keys[: near.pages].isnan().all() and far.values[: near.pages].isnan().all()
