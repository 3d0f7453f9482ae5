"""The choice of experts where keys with a bias lie too near for 32 bits: a few candidates, and more than a wavefront holds (nanollama_amd.ops.route)."""
import numpy as np
import pytest

from test_gpu_ops import check_route

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E, k", [(2, 1), (8, 8), (64, 6), (96, 32), (256, 8), (500, 12), (1024, 32)])
def test_neighbours_a_rounding_apart(E, k):
    rng = np.random.default_rng(E + k)
    for alike in (2, 5, min(E, 60), min(E, 63), min(E, 64), min(E, 65), min(E, 66), E):      # that many lie around the border
        l = rng.uniform(-3, 0, (9, E)).astype(np.float32)
        b = np.zeros(E, np.float32)
        for t in range(9):
            at = rng.permutation(E)[:alike]
            l[t, at] = np.float32(1.5) + rng.integers(-3, 4, len(at)).astype(np.float32) * np.float32(2 ** -22)
        check_route(l, k, score="sigmoid", bias=b)
        check_route(l, k, score="sigmoid", bias=b + np.float32(0.37), renorm=False, scale=2.5)
        b[:: 2] = np.float32(1e-6)
        check_route(l, k, score="sigmoid", bias=b)


def test_neighbours_with_large_biases_and_places_without_an_expert():
    rng = np.random.default_rng(7)
    l = rng.standard_normal((20, 100)).astype(np.float32)
    for size in (1e3, 1e7, 1e30):                          # the sigmoids are lost in 32 bits, not in 64; at 1e30 in both: the lower number
        check_route(l, 9, score="sigmoid", bias=np.full(100, size, np.float32))
        check_route(l, 9, score="sigmoid", bias=np.full(100, -size, np.float32))
    l[:, 4:] = -np.inf
    check_route(l, 9, score="sigmoid", bias=np.full(100, 1e7, np.float32))
    b = np.full(100, -np.inf, np.float32)
    b[50] = 1.0
    check_route(rng.standard_normal((5, 100)).astype(np.float32), 9, score="sigmoid", bias=b)
    b[:] = np.inf
    check_route(rng.standard_normal((5, 100)).astype(np.float32), 9, score="sigmoid", bias=b)
