"""The paged cache and sampling of the handle tier: passes, forks, truncation
and compaction against contiguous copies kept in numpy, and a run of all of
them as a server would use them."""
import numpy as np
import pytest
import torch

from paged_ref import attention, sample
from runtime_b200.backend import PAGE_BF16, PAGE_F16, PAGE_F32, CudaBackend, ExecutorError, PagedCache, Sampling

pytestmark = pytest.mark.gpu

DTYPE = {PAGE_F32: torch.float32, PAGE_F16: torch.float16, PAGE_BF16: torch.bfloat16}


def kinds(fn):
    with pytest.raises(ExecutorError) as e:
        fn()
    return e.value.kind


@pytest.fixture(scope="module")
def be():
    b = CudaBackend(0)
    yield b
    b.close()


class Mirror:
    """Every sequence's K and V rows per layer, contiguous, on the host."""

    def __init__(self, be, layers, kv_heads, dim, sequences, seed=0, dtype=PAGE_F32, **kw):
        self.be, self.layers, self.kv, self.dim, self.dtype = be, layers, kv_heads, dim, dtype
        self.cache = PagedCache(be, layers, kv_heads, dim, sequences=sequences, page_dtype=dtype, **kw)
        self.rng = np.random.default_rng(seed)
        self.rows = [[[np.zeros((0, kv_heads * dim), np.float32) for _ in range(2)] for _ in range(layers)]
                     for _ in range(sequences)]

    def step(self, seqs, tokens, q_heads=None):
        """One pass: random rows in, and (with q_heads) every layer's attention checked."""
        self.cache.begin(seqs, tokens)
        for layer in range(self.layers):
            new = [[self.rng.normal(size=(n, self.kv * self.dim)).astype(np.float32) for n in tokens] for _ in range(2)]
            key, value = (self.be.upload_f32(np.concatenate(x) if sum(tokens) else np.zeros((0, self.kv * self.dim)))
                          for x in new)
            self.cache.write(layer, key, value)
            for i, s in enumerate(seqs):
                for w in range(2):
                    self.rows[s][layer][w] = np.concatenate([self.rows[s][layer][w], new[w][i]])
            if q_heads:
                self.check(layer, seqs, q_heads)

    def check(self, layer, seqs, q_heads):
        q = self.rng.normal(size=(len(seqs), q_heads * self.dim)).astype(np.float32)
        query, out = self.be.upload_f32(q), self.be.allocate_f32(q.shape)
        self.cache.gqa(layer, out, query, q_heads)
        got = torch.from_numpy(self.be.read_f32(out)).view(len(seqs), q_heads, self.dim)
        # The contiguous copies as one-page pools, a page per sequence.
        lengths = [len(self.rows[s][layer][0]) for s in seqs]
        page = max(1, max(lengths))
        pools = []
        for w in range(2):
            pool = torch.zeros(len(seqs), self.kv, page, self.dim, dtype=DTYPE[self.dtype])
            for i, s in enumerate(seqs):
                r = torch.from_numpy(self.rows[s][layer][w]).view(-1, self.kv, self.dim).transpose(0, 1)
                pool[i, :, : r.shape[1]] = r.to(pool.dtype)
            pools.append(pool)
        table = np.arange(len(seqs))[:, None]
        ref, bound = attention(torch.from_numpy(q).view(len(seqs), q_heads, self.dim), *pools, table, lengths,
                               range(len(seqs)), page)
        assert ((got.double() - ref).abs() <= bound).all()

    def fork(self, a, b):
        self.cache.fork(a, b)
        self.rows[b] = [[x.copy() for x in layer] for layer in self.rows[a]]

    def truncate(self, s, n):
        self.cache.truncate(s, n)
        self.rows[s] = [[x[:n] for x in layer] for layer in self.rows[s]]


@pytest.mark.parametrize("dtype", [PAGE_F32, PAGE_F16, PAGE_BF16])
def test_passes_forks_truncation_and_compaction(be, dtype):
    m = Mirror(be, layers=2, kv_heads=2, dim=64, sequences=6, seed=1, dtype=dtype, pages=40, max_pages=12, page_tokens=8)
    m.step([0, 3], [20, 7], q_heads=8)
    m.step([3, 0], [1, 1], q_heads=8)
    m.fork(0, 1)
    m.fork(0, 2)
    free = m.cache.free_pages
    assert m.cache.sequence(1) == m.cache.sequence(0)
    m.step([1, 2, 0, 3], [1, 1, 1, 1], q_heads=8)      # three owners of a shared last page: two copies
    assert m.cache.free_pages == free - 2 - 1           # and one page that sequence 3 begins
    pages = [m.cache.sequence(s)[1] for s in (0, 1, 2)]
    assert pages[0][:2] == pages[1][:2] == pages[2][:2] and len({p[2] for p in pages}) == 3
    m.truncate(0, 9)
    m.truncate(3, 0)
    assert m.cache.sequence(3) == (0, [])
    m.step([0, 4, 1], [3, 0, 30], q_heads=8)            # a shared page is cut and written: copied again; one empty
    before = m.cache.free_pages
    m.cache.compact()
    assert m.cache.free_pages == before
    used = sorted({p for s in range(6) for p in m.cache.sequence(s)[1]})
    assert used == list(range(len(used)))
    m.step([0, 1, 2, 5], [0, 1, 2, 40], q_heads=8)
    for s in range(6):
        m.truncate(s, 0)
    assert m.cache.free_pages == 40
    m.step([5], [96], q_heads=4)                        # every page of a sequence
    m.cache.close()


def test_pages_hold_the_rows(be):
    m = Mirror(be, layers=1, kv_heads=2, dim=8, sequences=2, seed=2, pages=6, max_pages=4, page_tokens=4)
    m.step([1], [10])
    assert m.cache.sequence(1) == (10, [0, 1, 2])       # the lowest free pages
    m.step([0], [1])
    m.truncate(1, 4)
    m.step([0], [7])
    assert m.cache.sequence(0) == (8, [3, 1]) and m.cache.free_pages == 3
    assert len(set(m.cache.pages(0))) == 2
    m.cache.close()


def test_refusals_change_nothing(be):
    c = PagedCache(be, 2, 2, 64, pages=4, sequences=3, max_pages=3, page_tokens=4)
    row = be.upload_f32(np.ones((2, 128)))
    q = be.upload_f32(np.ones((1, 256)))
    out = be.allocate_f32((1, 256))
    assert kinds(lambda: c.write(0, row, row)) == "InvalidArgument"          # no pass
    assert kinds(lambda: c.gqa(0, out, q, 4)) == "InvalidArgument"
    assert kinds(lambda: c.begin([3], [1])) == "OutOfBounds"
    assert kinds(lambda: c.begin([0, 0], [1, 1])) == "InvalidArgument"
    assert kinds(lambda: c.begin([0], [13])) == "OutOfBounds"                # a sequence's pages
    assert kinds(lambda: c.begin([0, 1], [12, 8])) == "ResourceLimit"        # 5 of 4 pages
    assert c.free_pages == 4 and c.sequence(0) == (0, [])
    c.begin([0], [2])
    assert kinds(lambda: c.write(2, row, row)) == "OutOfBounds"
    assert kinds(lambda: c.write(0, q, row)) == "InvalidShape"
    assert kinds(lambda: c.gqa(0, out, q, 3)) == "InvalidShape"
    assert kinds(lambda: c.gqa(0, out, out, 4)) == "InvalidArgument"
    assert kinds(lambda: c.gqa(0, out, q, 8)) == "InvalidShape"
    c.write(0, row, row)
    c.gqa(0, out, q, 4)
    assert np.allclose(be.read_f32(out), 1.0, atol=2.0**-18)
    assert kinds(lambda: c.fork(0, 0)) == "InvalidArgument"
    assert kinds(lambda: c.fork(0, 7)) == "OutOfBounds"
    c.fork(0, 1)
    assert kinds(lambda: c.write(0, row, row)) == "InvalidArgument"          # a fork ends the pass
    assert kinds(lambda: c.fork(0, 1)) == "InvalidArgument"                  # not empty
    assert kinds(lambda: c.truncate(0, 3)) == "OutOfBounds"
    c.begin([0, 1], [1, 1])                                                  # the shared page, copied once
    assert c.free_pages == 2
    with CudaBackend(0) as other:
        assert kinds(lambda: c.write(0, other.upload_f32(np.ones((2, 128))), row)) == "WrongBackend"
    c.close()


@pytest.mark.parametrize("kw,kind", [
    (dict(head_dim=60), "Unsupported"), (dict(head_dim=256), "Unsupported"), (dict(layers=0), "InvalidShape"),
    (dict(pages=0), "InvalidShape"), (dict(page_dtype=3), "InvalidDType"), (dict(pages=1 << 40), "Overflow"),
    (dict(max_pages=1 << 30), "Overflow"),
])
def test_geometry_refusals(be, kw, kind):
    a = dict(layers=1, kv_heads=2, head_dim=64, pages=4, sequences=2, max_pages=2, page_tokens=4, page_dtype=PAGE_F32)
    a.update(kw)
    assert kinds(lambda: PagedCache(be, **a)) == kind


def test_pages_are_accounted_and_limited():
    page = 2 * 4 * 64 * 4
    with CudaBackend(0, limits=dict(max_total_bytes=(8 << 20) + (1 << 20))) as b:
        before = b.resource_report()
        c = PagedCache(b, 3, 2, 64, pages=10, sequences=2, max_pages=2, page_tokens=4)
        now = b.resource_report()
        assert now["cache_bytes"] - before["cache_bytes"] == 6 * 10 * page + (2 * (2 + 4) + 1) * 4
        c.close()
        assert b.resource_report() == before
        assert kinds(lambda: PagedCache(b, 3, 2, 64, pages=1000, sequences=2, max_pages=2, page_tokens=4)) == "ResourceLimit"
        assert b.resource_report() == before


def test_a_stale_cache_is_refused():
    with CudaBackend(0) as b:
        c = PagedCache(b, 1, 1, 8, pages=2, sequences=1, max_pages=2)
        b.advance_generation()
        assert kinds(lambda: c.begin([0], [1])) == "StaleBuffer"


def test_sample_handles(be):
    rng = np.random.default_rng(6)
    x = (rng.normal(size=(5, 3000)) * 3).astype(np.float32)
    u = rng.random(5).astype(np.float32)
    logits, uniform, out = be.upload_f32(x), be.upload_f32(u), be.allocate_f32((5,))
    params = [Sampling(0.7, 40, 0.9, 0.01), Sampling(), Sampling(0.0), Sampling(1.3, 0, 0.5), Sampling(1.0, 7)]
    be.sample(out, logits, params, uniform)
    expect = [sample(x[i], p.temperature, p.top_k, p.top_p, p.min_p, u[i]) for i, p in enumerate(params)]
    assert list(be.read_f32(out)) == expect
    be.sample(out, logits, Sampling(0.7, 40), uniform)
    assert list(be.read_f32(out)) == [sample(x[i], 0.7, 40, 1, 0, u[i]) for i in range(5)]
    greedy = be.allocate_f32((5,))
    be.argmax(greedy, logits)
    be.sample(out, logits, Sampling(0.0), uniform)
    assert np.array_equal(be.read_f32(out), be.read_f32(greedy))
    for bad in (Sampling(-1.0), Sampling(float("nan")), Sampling(float("inf")), Sampling(1.0, 0, -0.1),
                Sampling(1.0, 0, float("nan")), Sampling(1.0, 0, 1.0, 1.5)):
        assert kinds(lambda: be.sample(out, logits, bad, uniform)) == "InvalidArgument"
    assert kinds(lambda: be.sample(out, logits, [Sampling()] * 2, uniform)) == "InvalidShape"
    assert kinds(lambda: be.sample(be.allocate_f32((4,)), logits, Sampling(), uniform)) == "InvalidShape"
    assert kinds(lambda: be.sample(out, uniform, Sampling(), uniform)) == "InvalidShape"
    assert kinds(lambda: be.sample(out, logits, Sampling(), be.allocate_f32((5, 1)))) == "InvalidShape"


def test_a_state_samples_and_goes_on(be, oracle):
    """A sampled generation with the model's own loop, against the oracle's
    logits and the plain sampler."""
    from runtime_b200 import lfm2 as M

    cfg = M.tiny_config()
    w = M.synthetic_weights(cfg, 0)
    model = M.Lfm2Model(be, cfg, w)
    ref = oracle.Lfm2Oracle(cfg, w, threads=4)
    rng = np.random.default_rng(3)
    prompt = rng.integers(0, cfg.vocab, size=12)
    st = model.new_state()
    assert kinds(lambda: st.sample(Sampling(), 0.5)) == "InvalidArgument"    # no logits yet
    st.append(prompt)
    ref_logits = ref.append(prompt)
    p = Sampling(0.9, 30, 0.95, 0.0)
    for _ in range(6):
        u = float(np.float32(rng.random()))
        st.sample(p, u)
        got = st.read_sampled()
        assert got == sample(st.logits(), p.temperature, p.top_k, p.top_p, p.min_p, u)
        assert np.max(np.abs(st.logits() - ref_logits)) <= 1e-2
        st.append_argmax()                                                   # appends the sampled id
        _, ref_logits = ref.append_argmax(int(got))
    st.sample(Sampling(0.0), 0.5)
    assert st.read_sampled() == float(np.argmax(st.logits()))
    assert kinds(lambda: st.sample(Sampling(-1.0), 0.5)) == "InvalidArgument"
    for u in (-0.1, 1.0, float("nan")):
        assert kinds(lambda: st.sample(Sampling(), u)) == "InvalidArgument"

    batch = model.new_batch(4)
    assert kinds(lambda: batch.sample(Sampling(), [0.5] * 4)) == "InvalidArgument"
    batch.fork(st)
    batch.append_argmax(rng.integers(0, cfg.vocab, size=(4, 3)))
    u = rng.random(4).astype(np.float32)
    params = [Sampling(0.8, 20), Sampling(0.0), Sampling(1.2, 0, 0.9), Sampling()]
    batch.sample(params, u)
    ids, logits = batch.read()
    assert list(ids) == [sample(logits[i], q.temperature, q.top_k, q.top_p, q.min_p, u[i]) for i, q in enumerate(params)]
    single = model.new_state()
    single.copy_from(st)
    batch.decode(1)
    assert kinds(lambda: batch.sample([Sampling()] * 3, u)) == "InvalidShape"
    for x in (batch, single, st, model):
        x.close()


def test_a_server_runs_them_together(be):
    """Two prompts enter, one is forked into three, all decode at different
    lengths and sample their next tokens; one ends, the cache is compacted and
    the rest goes on."""
    vocab, q_heads, kv, dim, layers = 500, 4, 2, 64, 2
    rng = np.random.default_rng(9)
    m = Mirror(be, layers=layers, kv_heads=kv, dim=dim, sequences=5, seed=10, dtype=PAGE_BF16, pages=30, max_pages=8,
               page_tokens=16)
    head = be.upload_f32(rng.normal(size=(vocab, q_heads * dim)).astype(np.float32))
    m.step([0, 4], [37, 60])
    m.fork(0, 1)
    m.fork(0, 2)
    live = [0, 1, 2, 4]
    for step in range(6):
        m.step(live, [1] * len(live), q_heads=q_heads)
        hidden = be.upload_f32(rng.normal(size=(len(live), q_heads * dim)).astype(np.float32))
        out = be.allocate_f32(hidden.shape)
        m.cache.gqa(layers - 1, out, hidden, q_heads)
        logits = be.allocate_f32((len(live), vocab))
        be.linear(logits, out, head)
        ids, u = be.allocate_f32((len(live),)), rng.random(len(live)).astype(np.float32)
        params = [Sampling(0.8, 40, 0.9, 0.02) if s % 2 else Sampling(1.0) for s in live]
        be.sample(ids, logits, params, be.upload_f32(u))
        x = be.read_f32(logits)
        assert list(be.read_f32(ids)) == [sample(x[i], p.temperature, p.top_k, p.top_p, p.min_p, u[i])
                                          for i, p in enumerate(params)]
        if step == 2:
            m.truncate(0, 0)
            live.remove(0)
            m.cache.compact()
            used = {p for s in live for p in m.cache.sequence(s)[1]}
            assert used == set(range(len(used)))
    m.cache.close()


@pytest.mark.parametrize("tokens", [[1, 9000, 5], [64, 0, 1], [65, 3, 0]])
def test_passes_that_change_few_and_many_entries_of_a_wide_table(be, tokens):
    m = Mirror(be, 1, 1, 8, sequences=3, pages=20000, max_pages=20000, page_tokens=1)
    m.step([0, 1, 2], tokens, q_heads=2)
    m.step([2, 0], [2, 1], q_heads=2)
    m.step([1], [70], q_heads=2)
    m.cache.close()


@pytest.mark.parametrize("cut,pages", [(8, [2, 3, 4]), (4, [2, 3, 1]), (0, [2, 1, 0])])
def test_compaction_ends_the_pass_whether_or_not_pages_move(be, cut, pages):
    """(The appended token takes the lowest free page; only the last case then moves one.)"""
    c = PagedCache(be, 1, 1, 8, pages=6, sequences=2, max_pages=3, page_tokens=4)
    c.begin([0, 1], [8, 8])
    c.truncate(0, cut)
    c.begin([1], [1])
    row = be.upload_f32(np.ones((1, 8)))
    c.write(0, row, row)
    c.compact()
    assert kinds(lambda: c.write(0, row, row)) == "InvalidArgument"
    assert kinds(lambda: c.gqa(0, row, row, 1)) == "InvalidArgument"
    assert c.sequence(1) == (9, pages)
    c.close()
