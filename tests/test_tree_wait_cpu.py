"""The limit of the tree attention's waits: what is refused."""
from runtime_b200 import _lib, build


def test_limits_that_are_none_are_refused():
    build.build()
    lib = _lib.load()
    for tries in ((1 << 22) + 1, 2**32 - 1):
        assert lib.mf_set_tree_wait(tries) == 1 and lib.mf_last_error()
    for tries in (0, 1, 1 << 22):
        assert lib.mf_set_tree_wait(tries) == 0
