"""Sampling on a GPU against the plain 64-bit sampler, id by id."""
import numpy as np
import pytest
import torch

from paged_ref import sample

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    from runtime_b200 import _lib

    return _lib.load()


def draw(lib, logits, temperature, uniform, top_k=None, top_p=None, min_p=None):
    x = torch.as_tensor(np.asarray(logits, np.float32)).cuda()
    rows, width = x.shape
    f = lambda v, t=torch.float32: None if v is None else torch.as_tensor(np.asarray(v)).to(t).cuda()  # noqa: E731
    args = [f(temperature), f(top_k, torch.int32), f(top_p), f(min_p), f(uniform)]
    out = torch.full((rows,), -5.0, device="cuda")
    st = lib.mfk_sample(out.data_ptr(), x.data_ptr(), rows, width, *(None if a is None else a.data_ptr() for a in args),
                        torch.cuda.current_stream().cuda_stream)
    assert st == 0, lib.mf_last_error()
    return out.cpu().numpy()


def expect(logits, temperature, uniform, top_k=None, top_p=None, min_p=None):
    n = len(logits)
    off = lambda v, x: [x] * n if v is None else v  # noqa: E731
    return np.array([sample(*a) for a in zip(np.asarray(logits, np.float32), temperature, off(top_k, 0), off(top_p, 1.0),
                                             off(min_p, 0.0), uniform)], np.float64)


def same(got, want):
    np.testing.assert_array_equal(got.astype(np.float64), want)


@pytest.mark.parametrize("width", [1, 2, 3, 31, 33, 127, 1000, 1024, 1025, 4097, 32003, 65536, 65537, 131071, 200001])
@pytest.mark.parametrize("filters", ["none", "top_k", "top_p", "min_p", "all"])
def test_every_filter_and_width(lib, width, filters):
    rng = np.random.default_rng(width)
    rows = 7
    logits = (rng.normal(size=(rows, width)) * 2.5).astype(np.float32)
    pick = lambda name, v: rng.choice(v, rows).astype(np.float32) if filters in (name, "all") else None  # noqa: E731
    t, u = rng.choice([0.2, 0.7, 1.0, 1.7], rows).astype(np.float32), rng.random(rows).astype(np.float32)
    k = rng.choice([1, 2, 17, 50, width, 0], rows) if filters in ("top_k", "all") else None
    p, m = pick("top_p", [0.05, 0.5, 0.9, 0.99, 1.0]), pick("min_p", [0.0, 0.01, 0.2])
    same(draw(lib, logits, t, u, k, p, m), expect(logits, t, u, k, p, m))


@pytest.mark.parametrize("width", [100, 5000, 65536])
def test_equal_logits_go_to_the_lowest_index(lib, width):
    """Few distinct values: the cuts of top-k and top-p fall among equals."""
    rng = np.random.default_rng(2)
    rows = 24
    logits = rng.integers(-3, 3, (rows, width)).astype(np.float32)
    logits[1] = 0.0
    logits[2, ::2] = -0.0
    t, u = np.full(rows, 1.0, np.float32), rng.random(rows).astype(np.float32)
    k = rng.integers(1, width, rows)
    same(draw(lib, logits, t, u, k), expect(logits, t, u, k))
    p = rng.choice([0.1, 0.3, 0.77], rows).astype(np.float32)
    same(draw(lib, logits, t, u, None, p), expect(logits, t, u, None, p))
    same(draw(lib, logits, t, u, k, p), expect(logits, t, u, k, p))


def test_values_that_decide_nothing_or_everything(lib):
    inf = np.inf
    rows = np.array([
        [-inf, 1.0, -inf, 0.5], [-inf, -inf, -inf, -2.0], [-3.4e38, -3.4e38, -3.4e38, -3.4e38], [3.4e38, -3.4e38, 0, 1],
        [-inf] * 4, [0, np.nan, 1, 2], [0, inf, 1, 2], [0, 0, 0, 0],
    ], np.float32)
    n = len(rows)
    for u in (0.0, 0.3, 1.0 - 2.0**-24):
        for t in (1e-30, 0.0, 1.0, 1e30):
            tt, uu = [t] * n, [u] * n
            same(draw(lib, rows, tt, uu), expect(rows, tt, uu))
            same(draw(lib, rows, tt, uu, [2] * n, [0.6] * n, [0.3] * n), expect(rows, tt, uu, [2] * n, [0.6] * n, [0.3] * n))


def test_settings_out_of_range(lib):
    x = np.tile(np.array([[0.0, 1.0, 2.0, 0.5]], np.float32), (9, 1))
    nan = np.nan
    t = np.array([-1, nan, np.inf, 1, 1, 1, 1, 1, 1], np.float32)
    p = np.array([0.9, 0.9, 0.9, nan, 0.9, 0.9, -2.0, 7.0, 0.0], np.float32)
    m = np.array([0, 0, 0, 0, nan, 0, 0, 5.0, -1.0], np.float32)
    u = np.array([0.5, 0.5, 0.5, 0.5, 0.5, nan, 0.9, 0.2, 0.9], np.float32)
    k = np.array([0, 0, 0, 0, 0, 0, -4, 9, 1 << 30])
    got = draw(lib, x, t, u, k, p, m)
    assert np.isnan(got[:6]).all()
    assert list(got[6:]) == [2.0, 2.0, 2.0]
    ends = draw(lib, x[:3], [1, 1, 1], [-0.5, 1.0, 2.0])
    assert list(ends) == [0.0, 3.0, 3.0]


def test_probabilities_come_out(lib):
    """Evenly spaced uniform numbers hit each token as often as its share."""
    width, n = 50, 4096
    rng = np.random.default_rng(4)
    x = rng.normal(size=width).astype(np.float32)
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    got = draw(lib, np.tile(x, (n, 1)), np.ones(n), u)
    share = np.exp(x.astype(np.float64) - x.max())
    share /= share.sum()
    counts = np.bincount(got.astype(int), minlength=width)
    assert np.all(np.abs(counts - share * n) <= 1.0 + 1e-6)


def test_captured_and_replayed(lib):
    rng = np.random.default_rng(5)
    x = torch.as_tensor(rng.normal(size=(3, 9000)).astype(np.float32)).cuda()
    t, u, out = torch.ones(3, device="cuda"), torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda")
    draw(lib, x.cpu().numpy(), [1, 1, 1], [0, 0, 0])
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        assert lib.mfk_sample(out.data_ptr(), x.data_ptr(), 3, 9000, t.data_ptr(), None, None, None, u.data_ptr(),
                              stream.cuda_stream) == 0
    for _ in range(3):
        now = rng.random(3).astype(np.float32)
        u.copy_(torch.as_tensor(now))
        graph.replay()
        torch.cuda.synchronize()
        same(out.cpu().numpy(), expect(x.cpu().numpy(), [1, 1, 1], now))


@pytest.mark.parametrize("width,rows", [(400003, 3), (1 << 20, 2), (2048, 700), (30000, 333)])
@pytest.mark.parametrize("filters", ["none", "flat", "all"])
def test_rows_too_wide_for_shared_memory_and_many_rows(lib, width, rows, filters):
    """Past the cluster's shared memory, and more rows than the SMs hold; flat
    rows with top-p alone go through the histogram."""
    rng = np.random.default_rng(width + rows)
    logits = (rng.normal(size=(rows, width)) * (0.3 if filters == "flat" else 2.0)).astype(np.float32)
    t, u = rng.choice([0.5, 1.0, 1.5], rows).astype(np.float32), rng.random(rows).astype(np.float32)
    k = p = m = None
    if filters == "flat":
        p = rng.choice([0.3, 0.9, 0.999], rows).astype(np.float32)
    if filters == "all":
        k = rng.choice([0, 3, 60, 300, 450, 2000], rows)
        p, m = rng.choice([1.0, 0.8], rows).astype(np.float32), rng.choice([0.0, 1e-3], rows).astype(np.float32)
    pick = rng.permutation(rows)[:12]
    got = draw(lib, logits, t, u, k, p, m)
    cut = lambda v: None if v is None else v[pick]  # noqa: E731
    same(got[pick], expect(logits[pick], t[pick], u[pick], cut(k), cut(p), cut(m)))
    assert ((got >= 0) & (got < width)).all()


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_logits_of_any_alignment(lib, offset):
    rng = np.random.default_rng(offset)
    width, rows = 9001, 5
    store = torch.zeros(rows * width + 8, device="cuda")
    x = (rng.normal(size=(rows, width)) * 2).astype(np.float32)
    view = store[offset : offset + rows * width]
    view.copy_(torch.as_tensor(x).reshape(-1))
    t, u, k = np.ones(rows, np.float32), rng.random(rows).astype(np.float32), np.array([0, 5, 50, 500, 1])
    args = [torch.as_tensor(v).cuda() for v in (t, k.astype(np.int32), u)]
    out = torch.zeros(rows, device="cuda")
    assert lib.mfk_sample(out.data_ptr(), view.data_ptr(), rows, width, args[0].data_ptr(), args[1].data_ptr(), None, None,
                          args[2].data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    same(out.cpu().numpy(), expect(x, t, u, k))


def test_two_streams_at_once(lib):
    """Calls share nothing: the same rows on two streams, together."""
    rng = np.random.default_rng(7)
    rows, width = 300, 20000
    x = torch.as_tensor((rng.normal(size=(rows, width)) * 2).astype(np.float32)).cuda()
    t = torch.ones(rows, device="cuda")
    u = [torch.as_tensor(rng.random(rows).astype(np.float32)).cuda() for _ in range(2)]
    p = torch.full((rows,), 0.9, device="cuda")
    outs = [torch.zeros(rows, device="cuda") for _ in range(4)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()

    def call(i, out, stream):
        assert lib.mfk_sample(out.data_ptr(), x.data_ptr(), rows, width, t.data_ptr(), None, p.data_ptr(), None,
                              u[i].data_ptr(), stream) == 0

    for _ in range(5):
        for i in range(2):
            call(i, outs[i], streams[i].cuda_stream)
    torch.cuda.synchronize()
    for i in range(2):
        call(i, outs[2 + i], torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])


@pytest.mark.parametrize("width", [1500, 20000, 65536])
@pytest.mark.parametrize("n", [1, 2, 31, 63, 64, 65, 128, 129, 511, 512, 513, 1200])
def test_rows_with_n_tokens_ahead_of_the_rest(lib, width, n):
    """Top-p, top-k and min-p over lists of every length that is dealt with in
    another way: compared in pairs, sorted, or too many to list."""
    rng = np.random.default_rng(n * 7 + width)
    rows = 16
    logits = (-40.0 + rng.random((rows, width))).astype(np.float32)
    for r in range(rows):
        logits[r, rng.choice(width, n, replace=False)] = (rng.random(n) * 5).astype(np.float32)
    logits[1][logits[1] > -1] = 2.5  # all of them equal
    t, u = np.ones(rows, np.float32), rng.random(rows).astype(np.float32)
    p = rng.choice([0.3, 0.9, 0.999], rows).astype(np.float32)
    m = rng.choice([0.0, 0.05, 0.4], rows).astype(np.float32)
    k = rng.choice([max(n // 2, 1), n, n + 1], rows)
    same(draw(lib, logits, t, u, None, p), expect(logits, t, u, None, p))
    same(draw(lib, logits, t, u, None, p, m), expect(logits, t, u, None, p, m))
    same(draw(lib, logits, t, u, k), expect(logits, t, u, k))
    same(draw(lib, logits, t, u, k, p, m), expect(logits, t, u, k, p, m))


@pytest.mark.parametrize("rows,width", [(296, 600), (297, 600), (300, 600), (1001, 40), (160, 33000)])
def test_every_row_is_drawn_whatever_their_order(lib, rows, width):
    """More rows than run at once are begun in an order by their settings."""
    rng = np.random.default_rng(rows)
    logits = rng.normal(size=(rows, width)).astype(np.float32)
    t, u = rng.choice([0.5, 1.0, 1.4], rows).astype(np.float32), rng.random(rows).astype(np.float32)
    k, p = rng.choice([0, 5, width], rows), rng.choice([0.7, 1.0, 1.0, 0.95], rows).astype(np.float32)
    same(draw(lib, logits, t, u, k, p), expect(logits, t, u, k, p))
    same(draw(lib, logits, t, u, None, p), expect(logits, t, u, None, p))
    same(draw(lib, logits, t, u, None, np.full(rows, 0.9)), expect(logits, t, u, None, np.full(rows, 0.9)))


@pytest.mark.parametrize("width", [4, 700, 30000, 400003])
@pytest.mark.parametrize("temperature", [1e36, 1e37, 6e37, 2e38, 3.4028234e38])
def test_temperatures_as_large_as_the_largest_logits(lib, width, temperature):
    """Logits over F32's whole range, whose differences pass it."""
    rng = np.random.default_rng(width)
    rows = 8
    logits = ((rng.random((rows, width)) * 2 - 1) * 3.4e38).astype(np.float32)
    logits[0, :4] = [3e38, 2.9e38, -3e38, -2.9e38]
    logits[1, 3:] = -3.4e38
    t, u = np.full(rows, temperature, np.float32), rng.random(rows).astype(np.float32)
    k = np.array([2, 3, 0, 50, 600, width, 1, 0])
    p = np.array([1.0, 0.9, 0.5, 0.95, 0.99, 0.7, 0.5, 0.2], np.float32)
    m = np.array([0.0, 0.3, 0.5, 0.0, 0.01, 0.9, 0.0, 1e-6], np.float32)
    same(draw(lib, logits, t, u), expect(logits, t, u))
    same(draw(lib, logits, t, u, k), expect(logits, t, u, k))
    same(draw(lib, logits, t, u, None, p), expect(logits, t, u, None, p))
    same(draw(lib, logits, t, u, None, None, m), expect(logits, t, u, None, None, m))
    same(draw(lib, logits, t, u, k, p, m), expect(logits, t, u, k, p, m))


@pytest.mark.parametrize("rows", [3, 700])
@pytest.mark.parametrize("which", ["temperature", "min_p", "uniform"])
def test_the_ids_may_replace_a_setting_of_their_own_row(lib, rows, which):
    rng = np.random.default_rng(rows)
    width = 3000
    logits = rng.normal(size=(rows, width)).astype(np.float32)
    a = dict(temperature=rng.choice([0.5, 1.0], rows), top_p=rng.choice([0.9, 1.0], rows), min_p=rng.choice([0.0, 0.1], rows),
             uniform=rng.random(rows))
    a = {n: v.astype(np.float32) for n, v in a.items()}
    x, dev = torch.as_tensor(logits).cuda(), {n: torch.as_tensor(v).cuda() for n, v in a.items()}
    assert lib.mfk_sample(dev[which].data_ptr(), x.data_ptr(), rows, width, dev["temperature"].data_ptr(), None,
                          dev["top_p"].data_ptr(), dev["min_p"].data_ptr(), dev["uniform"].data_ptr(),
                          torch.cuda.current_stream().cuda_stream) == 0
    same(dev[which].cpu().numpy(), expect(logits, a["temperature"], a["uniform"], None, a["top_p"], a["min_p"]))
