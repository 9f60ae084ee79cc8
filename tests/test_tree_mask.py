"""tf_tree_mask (host): a node sees itself and its ancestors; bad trees are refused."""
import numpy as np
import pytest

from tinferno_b200 import native


def call(parents, T):
    p = np.ascontiguousarray(parents, np.int32)
    m = np.full((T, (T + 63) // 64), 5, np.uint64)
    d = np.full(T, 5, np.int32)
    native.check(native.lib().tf_tree_mask(p.ctypes.data_as(native.i32p), len(p), T, m.ctypes.data_as(native.u64p),
                                           d.ctypes.data_as(native.i32p)))
    return m, d


@pytest.mark.parametrize("n,T", [(0, 1), (1, 1), (5, 5), (64, 64), (65, 65), (40, 130), (256, 256)])
def test_mask_is_ancestors_and_self(n, T):
    rng = np.random.default_rng(n)
    parents = ([-1] + [int(rng.integers(0, i)) for i in range(1, n)])[:n]
    m, d = call(parents, T)
    for t in range(T):
        want, x, depth = set(), t, -1
        while t < n and x >= 0:
            want.add(x)
            x, depth = parents[x], depth + 1
        got = {j for j in range(T) if int(m[t, j // 64]) >> (j % 64) & 1}
        assert got == want
        assert d[t] == max(depth, 0)


def test_bad_trees_are_refused():
    for parents, T in (([0], 1), ([-1, 1], 2), ([-1, -1], 2), ([-1, 0, 5], 3), ([-1, 0], 1), ([-1], 257)):
        with pytest.raises(native.TFError):
            call(parents, T)
