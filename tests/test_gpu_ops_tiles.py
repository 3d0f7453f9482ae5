"""The experts' products in every size of tile, and slot by slot, at the sizes where one ends (nanollama_amd.ops.experts)."""
import numpy as np
import pytest

import ops_reference as ref
from hip_arrays import Stream, sync
from test_gpu_ops import Experts

pytestmark = pytest.mark.gpu


def skewed(n, E, k, seed=0):
    """Experts asked for very differently, and places without one."""
    rng = np.random.default_rng(seed)
    ids = np.minimum(rng.geometric(3.0 / max(E, 3), (n, k)) - 1, E + 1).astype(np.int32)      # E and E + 1 are no experts
    ids[rng.random((n, k)) < 0.05] = -1
    return ids


# what is expected to be done first: 64 x 64 twice; 128 x 128 and 128 x 64; 128 x 64 and 128 x 128; 256 x 256 and 128 x 128; 128 x 128 and 64 x 64
@pytest.mark.parametrize("n, dim, ff, E, k", [(600, 264, 200, 64, 8), (1500, 520, 1032, 16, 4), (700, 776, 520, 64, 4), (1600, 1032, 2056, 4, 2), (1600, 520, 1544, 4, 2)])
def test_every_tile(n, dim, ff, E, k):
    Experts(n, dim, ff, E, k, "bfloat16", seed=n).run()
    Experts(n, dim, ff, E, k, "bfloat16", seed=n, ids=skewed(n, E, k), x_apart=dim + 8, y_apart=dim + 3).run()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("cols", [8, 24, 56, 64, 72, 120, 128, 136, 192, 200, 256])
def test_rows_that_end_within_a_stage(cols, dtype):
    Experts(70, cols, 64, 3, 2, dtype, seed=cols).run()
    Experts(70, 64, cols, 3, 2, dtype, seed=cols).run()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("n", [15, 16, 17, 31, 33, 47, 49, 63, 64, 65, 127, 128, 129, 255, 256, 257])
def test_groups_that_end_within_a_tile(n, dtype):
    Experts(n, 64, 72, 2, 1, dtype, seed=n, ids=np.zeros((n, 1), np.int32)).run()
    Experts(n, 64, 72, 3, 2, dtype, seed=n, ids=np.tile(np.array([[2, 0]], np.int32), (n, 1))).run()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("n, E, k", [(1, 1, 1), (1, 2, 2), (1, 40, 32), (1, 64, 8), (2, 8, 2), (2, 7, 2), (4, 64, 8), (5, 64, 8), (16, 1024, 32), (17, 1024, 32)])
@pytest.mark.parametrize("dim, ff", [(8, 8), (264, 136), (1032, 520)])
def test_a_few_tokens(n, E, k, dim, ff, dtype):
    if E * dim * ff > 1 << 25:
        dim, ff = 40, 24
    Experts(n, dim, ff, E, k, dtype, seed=n).run()
    Experts(n, dim, ff, E, k, dtype, seed=n, ids=np.random.default_rng(n).integers(-1, E + 1, (n, k))).run()
    m = Experts(n, dim, ff, E, k, dtype, ids=np.full((n, k), -1), y_apart=dim + 5)
    m.run()
    assert np.all(m.y.numpy() == 0)


def test_a_few_tokens_in_a_graph():
    s = Stream()
    m = Experts(2, 96, 64, 16, 4, "bfloat16")
    play = s.capture(lambda: m.queue(s.number))
    for i in range(4):
        m.ids = np.random.default_rng(i).integers(-1, 16, m.ids.shape).astype(np.int32)
        m.di.write(m.ids)
        sync()
        play()
        s.sync()
        m.check()
        m.queue()                                          # eager work between the replays
        sync()
        m.check()


def test_the_same_bits_every_time_with_every_tile():
    for n, dim, ff, E, k in ((1500, 520, 1032, 16, 4), (700, 776, 520, 64, 4), (300, 264, 200, 6, 2), (1, 264, 200, 6, 2)):
        m = Experts(n, dim, ff, E, k, "bfloat16", seed=n)
        m.queue()
        sync()
        first = m.y.bits()
        for _ in range(3):
            m.queue()
            sync()
            assert np.array_equal(first, m.y.bits())


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("n, dim, ff, E, k", [(1, 34, 18, 3, 2), (3, 2, 2, 2, 1), (40, 100, 50, 6, 2), (70, 62, 66, 3, 2), (70, 126, 130, 3, 1), (200, 90, 258, 2, 2), (333, 190, 102, 5, 2)])
def test_rows_on_four_byte_boundaries(n, dim, ff, E, k, dtype):
    Experts(n, dim, ff, E, k, dtype, seed=n).run()
    Experts(n, dim, ff, E, k, dtype, seed=n, ids=skewed(n, E, k), x_apart=dim + 6, y_apart=dim + 1).run()
    Experts(n, 64, 48, E, k, dtype, seed=n, shift=2, x_apart=66).run()


@pytest.mark.parametrize("cols", [2, 30, 32, 34, 62, 64, 66, 94, 130, 190, 194, 258])
def test_rows_that_end_within_a_four_byte_stage(cols):
    Experts(70, cols, 66, 3, 2, "bfloat16", seed=cols).run()
    Experts(70, 66, cols, 3, 2, "bfloat16", seed=cols).run()


# slot by slot and activations as pairs: nothing but the result is rounded to bfloat16.  What is left of a rounded activation is at most 2^-8 of it, and that
# is rounded by 2^-8 once more: 2^-16 of the activation; a result is off by half a step of its own beside that.
@pytest.mark.parametrize("n, dim, ff, E, k", [(1, 768, 512, 64, 8), (4, 264, 136, 64, 8), (9, 264, 200, 12, 3), (32, 768, 512, 64, 8), (64, 520, 264, 32, 4), (31, 136, 1032, 8, 2), (128, 264, 776, 128, 8), (33, 64, 72, 300, 32)])
def test_few_tokens_an_expert_keep_their_activations(n, dim, ff, E, k):
    for ids in (None, skewed(n, E, k)):
        m = Experts(n, dim, ff, E, k, "bfloat16", seed=n, ids=ids)
        m.queue()
        sync()
        want, bound = ref.experts(m.x, m.ids, m.w, m.gate, m.up, m.down, "silu", 2.0 ** -16)
        step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(want) + bound, 1e-30))) - 7)
        assert np.all(np.abs(m.y.numpy() - want) <= step / 2 + bound)
        assert m.y.untouched() and m.ws.untouched()


def test_activations_that_are_no_numbers_stay_with_their_tokens():
    for n in (1, 20, 200):
        m = Experts(n, 64, 40, 8, 2, "bfloat16", seed=n)
        m.x[0] = 1e38                                      # products past the largest number, in one token
        m.dx.write(m.x)
        m.queue()
        sync()
        got = m.y.numpy()
        assert not np.all(np.isfinite(got[0])) and np.all(np.isfinite(got[1:]))
        want, bound = ref.experts(m.x[1:], m.ids[1:], m.w[1:], m.gate, m.up, m.down, "silu", 2.0 ** -8)
        assert np.all(np.abs(got[1:] - want) <= bound)


def test_two_threads_at_once():
    import threading
    cases = [Experts(33, 264, 136, 8, 2, "bfloat16", seed=1), Experts(300, 136, 264, 8, 2, "bfloat16", seed=2), Experts(2, 264, 136, 16, 4, "bfloat16", seed=3)]
    failed = []

    def work(m):
        try:
            s = Stream()
            for _ in range(50):
                m.queue(s.number)
            s.sync()
            m.check()
        except BaseException as e:      # noqa: B036 (told by the thread that asks)
            failed.append(e)

    threads = [threading.Thread(target=work, args=(m,)) for m in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
