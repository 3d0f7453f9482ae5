"""The choice of experts with biases of very different sizes: every key has an error of its own (nanollama_amd.ops.route)."""
import time

import numpy as np
import pytest

from hip_arrays import DeviceArray, sync
from nanollama_amd import ops
from test_gpu_ops import check_route

pytestmark = pytest.mark.gpu
SIZES = [0.0, 1.0, 1e3, 1e5, 2.0 ** 20, 2.0 ** 21, 2.0 ** 23, 2.0 ** 24, 2.0 ** 24 + 2, 2.0 ** 25, 2.0 ** 26, 1e9, 1e30, 3.4e38, np.inf]


def neighbours(rng, n, E):
    """Logits a few steps apart in pairs and crowds, others anywhere."""
    l = rng.uniform(-4, 4, (n, E)).astype(np.float32)
    for t in range(n):
        at = rng.permutation(E)[:max(1, E // 2)]
        l[t, at] = np.float32(0.8) + rng.integers(-3, 4, len(at)).astype(np.float32) * np.float32(2.0 ** -22)
    return l


@pytest.mark.parametrize("E, k", [(2, 1), (9, 4), (64, 8), (100, 32), (256, 8), (500, 12), (1024, 32)])
def test_biases_of_very_different_sizes(E, k):
    rng = np.random.default_rng(E + k)
    for _ in range(6):
        b = rng.choice(SIZES, E) * rng.choice([-1.0, 1.0], E) + rng.integers(-1, 2, E)
        check_route(neighbours(rng, 7, E), k, score="sigmoid", bias=b.astype(np.float32))
    for some in (1, 3, E // 2, E - k - 1):                # kept out by their bias, the others near one another
        for size in (-1e3, -1e9, float(np.finfo(np.float32).min)):
            b = (0.1 * rng.standard_normal(E)).astype(np.float32)
            b[rng.permutation(E)[:max(0, some)]] = size
            check_route(neighbours(rng, 5, E), k, score="sigmoid", bias=b, renorm=False)
            check_route(rng.standard_normal((5, E)).astype(np.float32), k, score="sigmoid", bias=b)


@pytest.mark.parametrize("size", SIZES)
def test_one_size_a_step_or_two_apart(size):
    rng = np.random.default_rng(int(np.log2(min(size, 1e30) + 1)))
    step = np.spacing(np.float32(min(size, 3e38)))
    for sign in (-1, 1):
        b = (sign * (np.float32(size) + step * rng.integers(0, 2, 130).astype(np.float32))).astype(np.float32)
        check_route(rng.uniform(-30, 30, (20, 130)).astype(np.float32), 6, score="sigmoid", bias=b)
        check_route(neighbours(rng, 20, 130), 6, score="sigmoid", bias=b)


def test_a_few_experts_kept_out_cost_nothing():
    """us of a call with biases of 0.1 and with some of -1e9 among them: the others are as far apart as before."""
    rng = np.random.default_rng(0)
    n, E, k = 8191, 1024, 32
    l, ids, w = DeviceArray(rng.standard_normal((n, E)).astype(np.float32)), DeviceArray(np.zeros((n, k), np.int32)), DeviceArray(np.zeros((n, k), np.float32))
    plain = (0.1 * rng.standard_normal(E)).astype(np.float32)
    mixed = plain.copy()
    mixed[::64] = -1e9
    took = []
    for b in (DeviceArray(plain), DeviceArray(mixed)):
        best = np.inf
        for _ in range(6):
            sync()
            start = time.perf_counter()
            for _ in range(20):
                ops.route(l, ids, w, score="sigmoid", bias=b)
            sync()
            best = min(best, time.perf_counter() - start)
        took.append(best)
    assert took[1] < 2 * took[0], took
