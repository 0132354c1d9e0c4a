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
