"""Every instance of the experts' products (nanollama_amd.ops.experts), and that it is the one which ran."""
import numpy as np
import pytest

import ops_reference as ref
from graph_kernels import product_forms, queued
from hip_arrays import DeviceArray, sync
from nanollama_amd import ops
from test_gpu_ops import HALF, Experts, as_type
from test_gpu_ops_far import Far
from test_gpu_ops_tiles import skewed

pytestmark = pytest.mark.gpu

# rows x tokens, stages, bytes a piece, activations in pairs
T64, T128x64, T128, T256 = (64, 64, 3, 16, False), (128, 64, 2, 16, False), (128, 128, 2, 16, False), (256, 256, 2, 16, False)
PAIR64, PAIR128 = (64, 32, 3, 16, True), (128, 32, 2, 16, True)
F32, BY4, F32_BY4 = (64, 32, 3, 16, False), (64, 64, 3, 4, False), (64, 32, 3, 4, False)


def check(m, forms):
    assert product_forms(queued(m.queue)) == forms
    m.queue()
    sync()
    if forms[1] in (PAIR64, PAIR128) or (forms[1] == "slots" and m.dtype == "bfloat16"):      # nothing but the result is rounded to 16 bits: what pairs leave is 2^-16 of an activation
        want, bound = ref.experts(m.x, m.ids, m.w, m.gate, m.up, m.down, m.act, 2.0 ** -16)
        step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(want) + bound, 1e-30))) - 7)
        assert np.all(np.abs(m.y.numpy() - want) <= step / 2 + bound)
        assert m.y.untouched() and m.ws.untouched()
    else:
        m.check()


@pytest.mark.parametrize("n, dim, ff, E, k, forms", [
    (600, 264, 200, 64, 8, (T64, T64)), (1500, 520, 1032, 16, 4, (T128, T128x64)), (700, 776, 520, 64, 4, (T128x64, T128)), (1600, 1032, 2056, 4, 2, (T256, T128)),
    (400, 1544, 136, 32, 8, (T64, T256)), (1000, 4104, 520, 8, 2, (T128, T256)),
    (40, 136, 72, 8, 1, (T64, PAIR64)), (100, 520, 264, 64, 5, (T64, PAIR64)), (64, 776, 72, 64, 1, (T64, PAIR128)), (64, 776, 520, 64, 6, (T128x64, PAIR128)),
    (200, 1544, 200, 64, 2, (T64, PAIR128)), (3, 264, 200, 64, 8, ("slots", "slots")), (1, 264, 200, 2, 2, ("slots", "slots"))])
def test_bfloat16(n, dim, ff, E, k, forms):
    check(Experts(n, dim, ff, E, k, "bfloat16", seed=n), forms)
    check(Experts(n, dim, ff, E, k, "bfloat16", seed=n, ids=skewed(n, E, k), x_apart=dim + 8, y_apart=dim + 3), forms)
    check(Experts(n, dim, ff, E, k, "bfloat16", seed=n, act="gelu_tanh", ids=np.full((n, k), E - 1)), forms)      # every token at one expert


@pytest.mark.parametrize("n, dim, ff, forms", [(70, 264, 200, (F32, F32)), (70, 265, 203, (F32_BY4, F32_BY4)), (2, 264, 200, ("slots", "slots")), (2, 265, 203, (F32_BY4, F32_BY4))])
def test_float32(n, dim, ff, forms):
    for act in ("silu", "gelu_tanh"):
        check(Experts(n, dim, ff, 8, 2, "float32", seed=n, act=act), forms)
        check(Experts(n, dim, ff, 8, 2, "float32", seed=n, act=act, ids=skewed(n, 8, 2), x_apart=dim + 8, y_apart=dim + 3), forms)


@pytest.mark.parametrize("n", [2, 70, 600])
@pytest.mark.parametrize("dim, ff, form", [(266, 202, BY4), (264, 203, "elements"), (265, 200, "elements")])
def test_rows_off_sixteen_bytes(n, dim, ff, form):
    for act in ("silu", "gelu_tanh"):
        check(Experts(n, dim, ff, 8, 2, "bfloat16", seed=n, act=act), (form, form))


# elements further than 32 bits reach: 1024 experts of 2.1e6 elements a matrix, and rows of x 2.2e9 elements from the first to the last
@pytest.mark.parametrize("dtype, F, D, forms", [("bfloat16", 2048, 1032, None), ("bfloat16", 2050, 1030, (BY4, BY4)), ("bfloat16", 2049, 1031, ("elements", "elements")),
                                                ("float32", 2048, 1032, (F32, F32)), ("float32", 2049, 1031, (F32_BY4, F32_BY4))])
def test_grouped_products_behind_32_bits(dtype, F, D, forms):
    E, n, ld = 1024, 1024 // 2 + 8, 1 << 22               # (half as many slots as experts go slot by slot)
    rng = np.random.default_rng(D)
    x, gate, up, down = as_type(rng.standard_normal((n, D)), dtype), *(as_type(rng.standard_normal(s) * s[1] ** -0.5, dtype) for s in ((F, D), (F, D), (D, F)))
    ids = np.full((n, 1), E - 1, np.int32)
    ids[1::2] = E - 2                                     # zeros
    w = rng.random((n, 1)).astype(np.float32)
    mats = [Far((E,) + m.shape, (F * D, m.shape[1], 1), dtype) for m in (gate, up, down)]
    for far, m in zip(mats, (gate, up, down)):
        far.write((E - 1) * F * D, m)
    far_x = Far((n, D), (ld, 1), dtype)
    for i in range(n):
        far_x.write(i * ld, x[i])
    y, di, dw = DeviceArray(np.full((n, D), 3.0), dtype), DeviceArray(ids), DeviceArray(w)
    ws = DeviceArray(np.zeros(ops.experts_workspace(n, 1, E, D, F, dtype), np.uint8))
    queue = lambda stream=0: ops.experts(far_x, di, dw, *mats, y, ws, stream=stream)  # noqa: E731
    ran = product_forms(queued(queue))
    assert ran == forms if forms else "slots" not in ran and ran[1][3] == 16, ran
    queue()
    sync()
    want, bound = ref.experts(x[::2], np.zeros((len(x[::2]), 1), np.int32), w[::2], gate[None], up[None], down[None], "silu", HALF[dtype])
    got = y.numpy()
    assert np.all(np.abs(got[::2] - want) <= bound) and np.all(got[1::2] == 0)
    assert y.untouched()
