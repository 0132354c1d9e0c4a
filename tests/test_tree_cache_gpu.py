"""Drafted trees through the paged cache of the handle tier: bookkeeping and
refusals, and a small LFM2 that generates by verifying drafted trees, token for
token what its own greedy steps give."""
import numpy as np
import pytest

from runtime_b200 import lfm2
from runtime_b200.backend import PAGE_BF16, PAGE_F16, PAGE_F32, CudaBackend, ExecutorError, PagedCache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    b = CudaBackend(0)
    yield b
    b.close()


def kinds(fn):
    with pytest.raises(ExecutorError) as e:
        fn()
    return e.value.kind


class Verifier:
    """The operations of an LFM2 over a paged cache, every row of a pass at once."""

    def __init__(self, be, cfg, weights, sequences, **kw):
        self.be, self.cfg, self.sequences = be, cfg, sequences
        attention = [i for i, k in enumerate(cfg.layer_types) if k == "attention"]
        self.layer = {i: n for n, i in enumerate(attention)}
        self.cache = PagedCache(be, len(attention), cfg.kv_heads, cfg.head_dim, sequences=sequences, **kw)

        def up(w):
            return be.upload_f32(w["value"] if isinstance(w, dict) else w)

        self.w = [{n: up(v) for n, v in layer.items()} for layer in weights["layers"]]
        self.embedding, self.norm = up(weights["embedding"]), up(weights["embedding_norm"])
        shape = (sequences, cfg.conv_width - 1, cfg.hidden)
        self.history = {i: be.allocate_f32(shape) for i, k in enumerate(cfg.layer_types) if k == "conv"}

    def run(self, seqs, drafts, parents=None):
        """One pass; drafts: each sequence's ids, parents: of its rows.  Returns (accepted, logits)."""
        be, cfg = self.be, self.cfg
        n = sum(len(d) for d in drafts)
        ids = np.concatenate(drafts)
        self.cache.begin(seqs, [len(d) for d in drafts])
        if parents is not None:
            self.cache.tree(np.concatenate(parents))
        new = lambda width: be.allocate_f32((n, width))  # noqa: E731
        x = new(cfg.hidden)
        be.gather_rows(x, self.embedding, ids)
        projections = {}
        for i, (kind, w) in enumerate(zip(cfg.layer_types, self.w)):
            u, op = new(cfg.hidden), new(cfg.hidden)
            be.row_rms_norm(u, x, w["operator_norm"], cfg.block_eps)
            if kind == "conv":
                projections[i], y = new(3 * cfg.hidden), new(cfg.hidden)
                be.linear(projections[i], u, w["in_proj"])
                self.cache.convolution(y, projections[i], w["conv_kernel"], self.history[i], cfg.conv_width)
                be.linear(op, y, w["out_proj"])
            else:
                q, k, v, y = new(cfg.hidden), new(cfg.kv_width), new(cfg.kv_width), new(cfg.hidden)
                for out, name in ((q, "q"), (k, "k"), (v, "v")):
                    be.linear(out, u, w[name])
                self.cache.write_rotated(self.layer[i], q, q, k, v, (cfg.q_heads, cfg.rope_theta), (w["q_norm"], w["k_norm"]), cfg.block_eps)
                self.cache.tree_gqa(self.layer[i], y, q, cfg.q_heads)
                be.linear(op, y, w["o"])
            residual, f, gate, up, h, down, after = new(cfg.hidden), new(cfg.hidden), new(cfg.intermediate), new(cfg.intermediate), new(cfg.intermediate), new(cfg.hidden), new(cfg.hidden)
            be.add_row_rms_norm(residual, f, x, op, w["ffn_norm"], cfg.block_eps)
            be.linear(gate, f, w["w1"])
            be.linear(up, f, w["w3"])
            be.swiglu(h, gate, up)
            be.linear(down, h, w["w2"])
            be.add(after, residual, down)
            x = after
        u, logits, sampled = new(cfg.hidden), new(cfg.vocab), be.allocate_f32((n,))
        be.row_rms_norm(u, x, self.norm, cfg.norm_eps)
        be.linear(logits, u, self.embedding)
        be.argmax(sampled, logits)
        accepted = self.cache.accept(be.upload_f32(ids.astype(np.float32)), sampled)
        for i, projection in projections.items():
            self.cache.convolution_keep(self.history[i], projection, cfg.conv_width)
        return accepted, be.read_f32(logits), be.read_f32(sampled)


def small_model():
    cfg = lfm2.tiny_config({r: "dense" for r in lfm2.ROLES}, hidden=256, intermediate=256, vocab=512)
    return cfg, lfm2.synthetic_weights(cfg, seed=3)


@pytest.mark.parametrize("page_dtype,tolerance", [(PAGE_F32, 1e-4), (PAGE_F16, None), (PAGE_BF16, None)])
def test_generation_by_drafted_trees(be, page_dtype, tolerance):
    """Prompts of different lengths enter in chunks; then every step verifies a tree whose
    branches are right for some tokens.  With F32 pages ids and logits are those
    of the executor's greedy steps (other orders of F32 sums over 256 terms move
    logits of size 1 by some 1e-6, and the ids' margins are looked at); with
    16-bit pages what is accepted is what the pass itself drew."""
    cfg, weights = small_model()
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, cfg.vocab, n) for n in (37, 5, 18)]
    steps = 24
    greedy, logits_of = [], []
    model = lfm2.Lfm2Model(be, cfg, weights)
    for p in prompts:
        state = model.new_state()
        state.append(p)
        ids, rows = [], []
        for _ in range(steps):
            rows.append(np.array(state.logits()).ravel())
            ids.append(int(np.argmax(rows[-1])))
            state.append([ids[-1]])
        greedy.append(ids), logits_of.append(rows)
        state.close()
    model.close()
    if tolerance is not None:
        margin = min(float(np.diff(np.sort(r)[-2:])[0]) for rows in logits_of for r in rows)
        assert margin > 2 * tolerance
    v = Verifier(be, cfg, weights, 4, pages=64, max_pages=16, page_tokens=16, page_dtype=page_dtype)
    seqs = [2, 0, 3]
    # Prompts, in two chunks; the ids that follow a row count as drawn: all are accepted.
    produced = [[] for _ in seqs]
    for lo, hi in ((0, 9), (9, 64)):
        chunk = [(s, p[lo:hi]) for s, p in zip(range(3), prompts) if len(p) > lo]
        accepted, _, _ = v_prompt(v, [seqs[s] for s, _ in chunk], [c for _, c in chunk])
        for (s, c), (path, nxt) in zip(chunk, accepted):
            assert path == list(range(len(c)))
            produced[s] = [int(nxt)]
    taken = []
    while min(len(p) for p in produced) < steps:
        drafts, parents = [], []
        for s in range(3):
            at = len(produced[s])
            right = (greedy[s] + [0] * 8)[at : at + 6] if tolerance is not None else rng.integers(0, cfg.vocab, 6).tolist()
            # Row 0 is certain.  A wrong branch first, then one right for 0 to 5 tokens, its
            # rows among those of others.
            good = int(rng.integers(0, 6))
            ids, up = [produced[s][-1], (right[0] + 1) % cfg.vocab], [-1, 0]
            last = 0
            for d in range(good):
                ids.append(right[d]), up.append(last)
                last = len(ids) - 1
                ids.append((right[d] + 7) % cfg.vocab), up.append(int(rng.integers(0, len(ids) - 1)))
            ids.append((right[good] + 3) % cfg.vocab), up.append(last)
            drafts.append(np.array(ids)), parents.append(np.array(up))
        accepted, logits, sampled = v.run(seqs, drafts, parents)
        first = 0
        for s, (path, nxt) in enumerate(accepted):
            at = len(produced[s])
            for j, r in enumerate(path):  # every accepted row's id is what the row before drew
                if j:
                    assert drafts[s][r] == sampled[first + path[j - 1]]
            assert nxt == sampled[first + path[-1]]
            if tolerance is not None:
                for j, r in enumerate(path):
                    if at + j < steps:
                        assert np.abs(logits[first + r] - logits_of[s][at + j]).max() <= tolerance
            produced[s] += [int(drafts[s][r]) for r in path[1:]] + [int(nxt)]
            taken.append(len(path))
            assert v.cache.sequence(seqs[s])[0] == len(prompts[s]) + len(produced[s]) - 1
            first += len(drafts[s])
    if tolerance is not None:
        for s in range(3):
            assert produced[s][:steps] == greedy[s]
        assert max(taken) > 3
    v.cache.close()


def v_prompt(v, seqs, chunks):
    """A chunk of prompts as chains, all of whose rows are kept."""
    real = v.cache.accept

    def accept(drafted, sampled):
        drawn = v.be.read_f32(sampled).copy()
        first = 0
        for c in chunks:  # the row's next id, but for the last
            drawn[first : first + len(c) - 1] = c[1:]
            first += len(c)
        return real(drafted, v.be.upload_f32(drawn))

    v.cache.accept = accept
    try:
        return v.run(seqs, chunks)
    finally:
        v.cache.accept = real


def cache_of(be, **kw):
    return PagedCache(be, 2, 2, 64, **{**dict(pages=12, sequences=4, max_pages=4, page_tokens=4), **kw})


def rows_of(be, n, width, seed=0):
    return be.upload_f32(np.random.default_rng(seed).normal(size=(n, width)))


def test_accepting_cuts_the_sequence_and_frees_pages(be):
    cache = cache_of(be)
    cache.begin([1, 0], [10, 0])
    assert cache.free_pages == 9
    cache.tree([-1, 0, 0, 1, 2, 4, 5, 5, 7, 8])
    for layer in range(2):
        cache.write(layer, rows_of(be, 10, 128), rows_of(be, 10, 128, 1))
    drafted = be.upload_f32(np.arange(10))
    sampled = be.upload_f32([2, 0, 4, 0, 5, 99, 0, 0, 0, 0])
    assert cache.accept(drafted, sampled) == [([0, 2, 4, 5], 99.0), ([], pytest.approx(float("nan"), nan_ok=True))]
    assert cache.sequence(1)[0] == 4 and cache.free_pages == 11
    # What is left are the path's rows: they equal those of a chain of the same values.
    both = []
    for seed in (0, 1):
        both.append(np.random.default_rng(seed).normal(size=(10, 128)).astype(np.float32)[[0, 2, 4, 5]])
    other = cache_of(be)
    other.begin([0], [4])
    q, outs = rows_of(be, 1, 256, 7), []
    for c, s in ((cache, 1), (other, 0)):
        if c is other:
            for layer in range(2):
                c.write(layer, be.upload_f32(both[0]), be.upload_f32(both[1]))
        else:
            c.begin([s], [0])
        for layer in range(2):
            out = be.allocate_f32((1, 256))
            c.gqa(layer, out, q, 4)
            outs.append(be.read_f32(out).copy())
    assert np.array_equal(outs[0], outs[2]) and np.array_equal(outs[1], outs[3])
    cache.close(), other.close()


def test_forks_keep_their_rows_when_one_accepts(be):
    """A shared last page is copied when a draft enters: the other sequence's attention stays."""
    cache = cache_of(be)
    cache.begin([0], [6])
    for layer in range(2):
        cache.write(layer, rows_of(be, 6, 128, layer), rows_of(be, 6, 128, layer + 5))
    cache.fork(0, 3)
    q = rows_of(be, 1, 256, 9)

    def look(s):
        cache.begin([s], [0])
        out = be.allocate_f32((1, 256))
        cache.gqa(1, out, q, 4)
        return be.read_f32(out).copy()

    before = look(3)
    cache.begin([0], [5])
    cache.tree([-1, 0, 0, 2, 3])
    for layer in range(2):
        cache.write(layer, rows_of(be, 5, 128, 20), rows_of(be, 5, 128, 21))
    assert cache.accept(be.upload_f32([1, 2, 3, 4, 5]), be.upload_f32([3, 0, 4, 0, 0]))[0][0] == [0, 2, 3]
    assert np.array_equal(look(3), before)
    assert cache.sequence(0)[0] == 9 and cache.sequence(3)[0] == 6
    cache.close()


def test_tree_refusals(be):
    cache = cache_of(be)
    q, kv, hist = rows_of(be, 3, 256), rows_of(be, 3, 128), be.allocate_f32((4, 2, 32))
    proj, kern, out, ids = rows_of(be, 3, 96), rows_of(be, 32, 3), be.allocate_f32((3, 32)), be.upload_f32([1, 2, 3])
    o = be.allocate_f32((3, 256))
    rope = (4, 1e6)
    calls = [lambda: cache.tree([-1, 0, 0]), lambda: cache.write_rotated(0, q, q, kv, rows_of(be, 3, 128), rope),
             lambda: cache.tree_gqa(0, o, q, 4), lambda: cache.convolution(out, proj, kern, hist, 3), lambda: cache.accept(ids, ids),
             lambda: cache.convolution_keep(hist, proj, 3)]
    for call in calls:  # outside of a pass
        assert kinds(call) == "InvalidArgument"
    cache.begin([2], [3])
    cases = [
        (lambda: cache.tree([-1, 0]), "InvalidShape"), (lambda: cache.tree([-1, 1, 0]), "InvalidArgument"),
        (lambda: cache.tree([-1, -2, 0]), "InvalidArgument"), (lambda: cache.tree([0, 0, 0]), "InvalidArgument"),
        (lambda: cache.write_rotated(2, q, q, kv, rows_of(be, 3, 128), rope), "OutOfBounds"),
        (lambda: cache.write_rotated(0, q, q, kv, rows_of(be, 2, 128), rope), "InvalidShape"),
        (lambda: cache.write_rotated(0, kv, q, kv, kv, rope), "InvalidShape"),
        (lambda: cache.write_rotated(0, q, q, kv, rows_of(be, 3, 128), (4, 0.0)), "InvalidArgument"),
        (lambda: cache.write_rotated(0, q, q, kv, rows_of(be, 3, 128), rope, (be.upload_f32(np.ones(32)), None)), "InvalidShape"),
        (lambda: cache.write_rotated(0, kv, kv, kv, rows_of(be, 3, 128), (2, 1e6)), "InvalidArgument"),
        (lambda: cache.tree_gqa(0, q, q, 4), "InvalidArgument"), (lambda: cache.tree_gqa(0, o, q, 3), "InvalidShape"),
        (lambda: cache.tree_gqa(2, o, q, 4), "OutOfBounds"), (lambda: cache.tree_gqa(0, o, kv, 4), "InvalidShape"),
        (lambda: cache.convolution(out, proj, kern, hist, 4), "InvalidShape"), (lambda: cache.convolution(out, proj, kern, hist, 17), "Unsupported"),
        (lambda: cache.convolution(out, proj, kern, be.allocate_f32((3, 2, 32)), 3), "InvalidShape"),
        (lambda: cache.convolution(out, kv, kern, hist, 3), "InvalidShape"),
        (lambda: cache.accept(ids, be.upload_f32([1, 2])), "InvalidShape"),
        (lambda: cache.convolution_keep(hist, proj, 3), "InvalidArgument"),
    ]
    for i, (call, kind) in enumerate(cases):
        assert kinds(call) == kind, i
    assert cache.accept(ids, ids)[0][0] == [0]
    cache.convolution_keep(hist, proj, 3)
    assert kinds(lambda: cache.accept(ids, ids)) == "InvalidArgument"
    cache.begin([2], [1])
    assert kinds(lambda: cache.convolution_keep(hist, rows_of(be, 1, 96), 3)) == "InvalidArgument"
    cache.close()


def test_a_pass_of_nothing(be):
    cache = cache_of(be)
    cache.begin([1, 2], [0, 0])
    cache.tree(None)
    empty = be.allocate_f32((0, 256))
    cache.tree_gqa(0, empty, be.allocate_f32((0, 256)), 4)
    cache.write_rotated(0, empty, empty, be.allocate_f32((0, 128)), be.allocate_f32((0, 128)), (4, 1e6))
    assert [p for p, _ in cache.accept(be.allocate_f32((0,)), be.allocate_f32((0,)))] == [[], []]
    cache.close()


def test_growing_trees_and_changing_sequences(be):
    """Passes of 1 to 14 rows of sequences in changing order: lengths follow the paths."""
    cache = cache_of(be, pages=40, sequences=5, max_pages=8, page_tokens=5)
    rng, length = np.random.default_rng(2), [0] * 5
    for step in range(12):
        seqs = rng.permutation(5)[: rng.integers(1, 6)]
        rows = [int(rng.integers(0, 4 + step // 2)) for _ in seqs]
        if any(length[s] + n > 40 for s, n in zip(seqs, rows)):
            for s in seqs:
                cache.truncate(int(s), 3 if length[s] > 3 else length[s])
                length[s] = min(length[s], 3)
        cache.begin(seqs, rows)
        parents = np.concatenate([[-1 if r == 0 else int(rng.integers(0, r)) for r in range(n)] for n in rows]).astype(int)
        cache.tree(parents)
        total = sum(rows)
        key, value, query = rows_of(be, total, 128), rows_of(be, total, 128), rows_of(be, total, 256)
        cache.write_rotated(0, query, query, key, value, (4, 1e4))
        cache.tree_gqa(0, be.allocate_f32((total, 256)), query, 4)
        drafted, sampled = (rng.integers(0, 2, total) for _ in range(2))
        for s, n, (path, _) in zip(seqs, rows, cache.accept(be.upload_f32(drafted), be.upload_f32(sampled))):
            assert (len(path) > 0) == (n > 0)
            length[s] += len(path)
            assert cache.sequence(int(s))[0] == length[s]
        assert 40 - cache.free_pages == sum(-(-n // 5) for n in length)
    cache.close()
