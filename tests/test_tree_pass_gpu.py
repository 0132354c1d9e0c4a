"""A whole pass of drafted trees on device pointers, captured once and replayed
with other lengths, trees, positions, ids and slots."""
import numpy as np
import pytest
import torch

import tree_ref
from paged_ref import PAGE_DTYPES
from test_tree_gpu import Cache, dev, lib, stream, workspace  # noqa: F401
from tree_ref import TREE_WORKSPACE

pytestmark = pytest.mark.gpu
SLOTS, PAGE, MAX_PAGES, TOKENS, HIDDEN, WIDTH = 6, 16, 20, 96, 128, 3


class Pass:
    """The arrays of a pass and its calls; everything that changes lies in device memory."""

    def __init__(self, lib, dtype, sequences, q_heads=8, kv_heads=2, dim=64):  # noqa: F811
        self.lib, self.n, self.heads = lib, sequences, (q_heads, kv_heads, dim)
        self.cache = Cache([PAGE * MAX_PAGES] * SLOTS, kv_heads, dim, PAGE, dtype, fill=False)
        g = torch.Generator(device="cuda").manual_seed(1)
        new = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.q, self.k, self.v = new(TOKENS, q_heads, dim), new(TOKENS, kv_heads, dim), new(TOKENS, kv_heads, dim)
        self.weights, self.projection, self.kernel = (new(dim), new(dim)), new(TOKENS, 3 * HIDDEN), new(HIDDEN, WIDTH)
        self.history = new(SLOTS, WIDTH - 1, HIDDEN)
        self.start_of = [x.clone() for x in (self.q, self.k, self.v, self.projection, self.history, self.cache.keys, self.cache.values)]
        self.turned, self.out, self.convolved = torch.empty_like(self.q), torch.empty_like(self.q), torch.empty(TOKENS, HIDDEN, device="cuda")
        self.ints = {name: dev(np.zeros(size)) for name, size in (
            ("starts", sequences), ("lengths", sequences), ("slots", sequences), ("offsets", sequences + 1), ("parents", TOKENS),
            ("positions", TOKENS), ("paths", TOKENS), ("counts", sequences))}
        self.drafted, self.sampled, self.next = (torch.zeros(m, device="cuda") for m in (TOKENS, TOKENS, sequences))
        self.pools = np.array([self.cache.keys.data_ptr(), self.cache.values.data_ptr()], np.uint64)
        self.ws = workspace()

    def reset(self):
        for x, y in zip((self.q, self.k, self.v, self.projection, self.history, self.cache.keys, self.cache.values), self.start_of):
            x.copy_(y)
        for x in (self.turned, self.out, self.convolved, self.next, self.ints["paths"], self.ints["counts"]):
            x.fill_(7)

    def set(self, step):
        for name, values in step.items():
            to = self.ints.get(name, getattr(self, name, None))
            to.copy_(torch.as_tensor(np.asarray(values), dtype=to.dtype))

    def run(self):
        lib, i, (qh, kvh, dim) = self.lib, {k: v.data_ptr() for k, v in self.ints.items()}, self.heads  # noqa: F811
        p, s = self.cache.args(), stream()
        status = [
            lib.mfk_paged_append_rope(*p, self.turned.data_ptr(), self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), TOKENS,
                                      self.weights[0].data_ptr(), self.weights[1].data_ptr(), 1e-5, 1e6, i["positions"], i["starts"],
                                      i["offsets"], i["slots"], self.n, qh, kvh, dim, s),
            lib.mfk_paged_tree_gqa(self.out.data_ptr(), self.turned.data_ptr(), *p, TOKENS, i["lengths"], i["offsets"], i["parents"],
                                   i["slots"], self.n, qh, kvh, dim, self.ws.data_ptr(), TREE_WORKSPACE, s),
            lib.mfk_tree_convolution(self.convolved.data_ptr(), self.projection.data_ptr(), self.kernel.data_ptr(), self.history.data_ptr(),
                                     SLOTS, TOKENS, i["offsets"], i["parents"], i["slots"], self.n, HIDDEN, WIDTH, s),
            lib.mfk_paged_accept(i["paths"], i["counts"], self.next.data_ptr(), self.pools.ctypes.data, 2, *p[2:], self.drafted.data_ptr(),
                                 self.sampled.data_ptr(), TOKENS, i["starts"], i["offsets"], i["parents"], i["slots"], self.n, kvh, dim, s),
            lib.mfk_tree_convolution_keep(self.history.data_ptr(), self.history.data_ptr(), SLOTS, self.projection.data_ptr(), TOKENS,
                                          i["paths"], i["counts"], i["offsets"], i["slots"], self.n, HIDDEN, WIDTH, s),
        ]
        assert status == [0] * 5, lib.mf_last_error()

    def results(self):
        return [x.clone() for x in (self.turned, self.out, self.convolved, self.next, self.history, self.cache.keys, self.cache.values,
                                    self.ints["paths"], self.ints["counts"])]


def steps(sequences):
    """Ragged, empty, full and single-row passes with trees of every kind."""
    rng = np.random.default_rng(9)
    made = []
    for rows in ([8] * sequences, [1] * sequences, [0, TOKENS - 3] + [1] * (sequences - 2), [30, 0, 20, 7][:sequences], [0] * sequences):
        starts = rng.integers(0, PAGE * MAX_PAGES - TOKENS, sequences)
        offsets = np.concatenate([[0], np.cumsum(rows)])
        parents, positions = np.full(TOKENS, -1), np.zeros(TOKENS, int)
        for f, n, start in zip(offsets, rows, starts):
            parents[f : f + n] = tree_ref.random_tree(n, rng)
            for r in range(n):
                positions[f + r] = start if parents[f + r] < 0 else positions[f + parents[f + r]] + 1
        made.append(dict(starts=starts, lengths=starts + rows, slots=rng.permutation(SLOTS)[:sequences], offsets=offsets, parents=parents,
                         positions=positions, drafted=rng.integers(0, 3, TOKENS), sampled=rng.integers(0, 3, TOKENS)))
    return made


@pytest.mark.parametrize("dtype", PAGE_DTYPES)
@pytest.mark.parametrize("sequences", [2, 4])
def test_a_captured_pass_follows_its_arrays(lib, dtype, sequences):  # noqa: F811
    p = Pass(lib, dtype, sequences)
    want = []
    for step in steps(sequences):
        p.reset(), p.set(step), p.run()
        torch.cuda.synchronize()
        want.append(p.results())
    paths = [w[7].cpu().numpy() for w in want]
    for step, path, w in zip(steps(sequences), paths, want):  # (the passes are themselves those of the plain form)
        for i in range(sequences):
            first, n = step["offsets"][i], step["offsets"][i + 1] - step["offsets"][i]
            expected = tree_ref.accept(step["drafted"], step["sampled"], step["parents"], first, n)[0] if n else []
            assert path[first : first + len(expected)].tolist() == expected and w[8][i] == len(expected)
    p.reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.run()
    p.pools[:] = 0  # (the list is read when the call is made)
    for order in (range(len(want)), reversed(range(len(want)))):
        for j in order:
            p.reset(), p.set(steps(sequences)[j])
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(p.results(), want[j]):
                assert torch.equal(a.nan_to_num(99.0) if a.is_floating_point() else a, b.nan_to_num(99.0) if b.is_floating_point() else b)


def test_passes_on_two_streams(lib):  # noqa: F811
    """A pass of its own on each stream, with its own workspace: neither sees the other."""
    passes = [Pass(lib, "bf16", 4) for _ in range(2)]
    todo = steps(4)[:2]
    want = []
    for p, step in zip(passes, todo):
        p.reset(), p.set(step), p.run()
        torch.cuda.synchronize()
        want.append(p.results())
    streams = [torch.cuda.Stream() for _ in passes]
    for _ in range(5):
        for p, step in zip(passes, todo):
            p.reset(), p.set(step)
        torch.cuda.synchronize()
        for p, s in zip(passes, streams):
            with torch.cuda.stream(s):
                p.run()
        torch.cuda.synchronize()
        for p, w in zip(passes, want):
            assert all(torch.equal(a, b) for a, b in zip(p.results(), w))
