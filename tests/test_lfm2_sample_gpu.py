"""Sampling of states and batches: from which logits a call draws, and when it
has none to draw from."""
import numpy as np
import pytest

from paged_ref import sample
from runtime_b200 import lfm2 as M
from runtime_b200.backend import CudaBackend, ExecutorError, Sampling

pytestmark = pytest.mark.gpu

PARAMS = [Sampling(0.9, 30, 0.95), Sampling(), Sampling(0.0), Sampling(1.4, 0, 0.9, 0.01), Sampling(2.0), Sampling(0.7, 5)]


@pytest.fixture(scope="module")
def be():
    b = CudaBackend(0)
    yield b
    b.close()


@pytest.fixture(scope="module")
def model(be):
    cfg = M.tiny_config()
    m = M.Lfm2Model(be, cfg, M.synthetic_weights(cfg, 0))
    yield m
    m.close()


def refused(fn):
    with pytest.raises(ExecutorError) as e:
        fn()
    return e.value.kind == "InvalidArgument"


def tokens(model, n, seed):
    return np.random.default_rng(seed).integers(0, model.cfg.vocab, size=n)


def check_draws(batch, logits, seed):
    """The batch's ids are drawn from `logits`, the same row for every sequence."""
    u = np.random.default_rng(seed).random(len(PARAMS)).astype(np.float32)
    batch.sample(PARAMS, u)
    ids, rows = batch.read()
    assert all(np.array_equal(row, logits) for row in rows)
    assert list(ids) == [sample(logits, p.temperature, p.top_k, p.top_p, p.min_p, x) for p, x in zip(PARAMS, u)]


def test_a_forked_batch_samples_from_its_prefix(model):
    """Several continuations of one prompt: fork, then sample, for a new batch
    and for one that has run something else."""
    st, other = model.new_state(), model.new_state()
    st.append(tokens(model, 12, 1))
    other.append(tokens(model, 5, 2))
    batch = model.new_batch(len(PARAMS))
    batch.fork(st)
    check_draws(batch, st.logits(), 3)
    batch.append_argmax(tokens(model, (len(PARAMS), 4), 4))
    batch.fork(other)
    check_draws(batch, other.logits(), 5)
    other.append_argmax(3)
    batch.fork(other)
    check_draws(batch, other.logits(), 6)
    empty = model.new_state()
    batch.fork(empty)
    assert refused(lambda: batch.sample(Sampling(), [0.5] * len(PARAMS)))
    for x in (batch, st, other, empty):
        x.close()


def test_a_state_without_logits_of_its_last_token_is_refused(model):
    """An append that wants no logits leaves none, whatever was there before;
    copies of such a state have none either."""
    fresh, used, good = (model.new_state() for _ in range(3))
    fresh.append(tokens(model, 6, 7), want_logits=False)
    assert refused(lambda: fresh.sample(Sampling(), 0.5))
    used.append(tokens(model, 6, 8))
    used.sample(Sampling(), 0.5)
    before = used.read_sampled()
    used.append(tokens(model, 2, 9), want_logits=False)
    assert refused(lambda: used.sample(Sampling(), 0.9))
    assert used.read_sampled() == before
    fork = used.fork()
    assert refused(lambda: fork.sample(Sampling(), 0.5))
    good.append(tokens(model, 4, 10))
    copy = model.new_state()
    copy.copy_from(good)
    copy.sample(Sampling(), 0.5)
    copy.copy_from(used)
    assert refused(lambda: copy.sample(Sampling(), 0.5))
    batch = model.new_batch(2)
    batch.fork(used)
    assert refused(lambda: batch.sample(Sampling(), [0.5, 0.5]))
    batch.append_argmax([[1], [2]])
    batch.sample(Sampling(), [0.5, 0.5])
    batch.fork(used)
    assert refused(lambda: batch.sample(Sampling(), [0.5, 0.5]))
    used.append([3])  # and now it has them
    used.sample(Sampling(0.0), 0.5)
    assert used.read_sampled() == float(np.argmax(used.logits()))
    for x in (batch, fresh, used, good, fork, copy):
        x.close()


@pytest.mark.parametrize("path", ["fused", "op by op", "persistent"])
def test_every_kind_of_step_leaves_logits(be, path):
    cfg = M.tiny_config()
    m = M.Lfm2Model(be, cfg, M.synthetic_weights(cfg, 0))
    m.set_fused(path != "op by op")
    m.set_persistent(path == "persistent")
    steps = [lambda s: s.append_argmax(5), lambda s: s.append_argmax(), lambda s: s.decode(1), lambda s: s.decode(9),
             lambda s: s.decode_host(4), lambda s: s.generate(3), lambda s: s.generate(3, stop_ids=range(65, 130)),
             lambda s: s.time_step(), lambda s: s.profile_step()]
    for step in steps:
        st = m.new_state()
        st.append(tokens(m, 3, 11))
        first = int(np.argmax(st.logits()))
        st.sample(Sampling(0.0), 0.0)
        assert st.read_sampled() == first
        st.append(tokens(m, 3, 12), want_logits=False)
        step(st)
        x = st.logits()
        st.sample(Sampling(1.5), 0.37)
        assert st.read_sampled() == sample(x, 1.5, 0, 1.0, 0.0, np.float32(0.37))
        st.close()
    m.close()


def test_the_next_step_appends_the_drawn_ids(model):
    """What is drawn is what goes on: of a batch and of a state, each against
    a state that is given the drawn ids."""
    st = model.new_state()
    st.append(tokens(model, 12, 13))
    n = len(PARAMS)
    u = np.random.default_rng(14).random(n).astype(np.float32)
    params = [Sampling(3.0)] * n
    batch = model.new_batch(n)
    batch.fork(st)
    given = [model.new_state() for _ in range(n)]
    for g in given:
        g.copy_from(st)
    for _ in range(3):
        batch.sample(params, u)
        ids, _ = batch.read()
        assert len(set(ids)) > 1
        batch.decode(1)
        _, rows = batch.read()
        for g, token, row in zip(given, ids, rows):
            g.append([int(token)])
            assert np.max(np.abs(g.logits() - row)) <= 1e-2       # as the batch's other tests
        assert np.max(np.abs(rows - rows[np.argmax(ids != ids[0])])) > 0.1
        u = (u + 0.37) % 1
    alone = model.new_state()
    alone.copy_from(st)
    alone.sample(Sampling(3.0), 0.9)
    token = int(alone.read_sampled())
    assert token != int(np.argmax(st.logits()))
    alone.append_argmax()
    given[0].copy_from(st)
    given[0].append([token])
    assert np.max(np.abs(alone.logits() - given[0].logits())) <= 1e-2
    for x in (batch, st, alone, *given):
        x.close()
