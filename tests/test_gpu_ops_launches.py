"""More tokens than the threads of one launch are counted for (nanollama_amd.ops): the rows behind the first launch's are written too."""
import numpy as np
import pytest

import ops_reference as ref
from hip_arrays import DeviceArray, sync
from nanollama_amd import ops
from test_gpu_ops import HALF, Experts, as_type
from test_gpu_ops_far import Far

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_residual_norm_of_more_rows(dtype):
    n = (1 << 24) + 5                                     # 2^32 threads and more
    rng = np.random.default_rng(1)
    x, d, g = rng.standard_normal((n, 1)).astype(np.float32), as_type(rng.standard_normal((n, 1)), dtype), rng.standard_normal((n, 1)).astype(np.float32)
    pre, post = np.full(1, 1.25, np.float32), np.full(1, 0.75, np.float32)
    xo, h = DeviceArray(np.full((n, 1), 9, np.float32)), DeviceArray(np.full((n, 1), 4.0), dtype)
    ops.residual_norm(DeviceArray(x), DeviceArray(d, dtype), xo, h, pre=DeviceArray(pre), post=DeviceArray(post), gate=DeviceArray(g), scale=0.5)
    sync()
    wx, wh, bx, bh = ref.residual_norm(x, d, pre, post, g, 0.5, 1e-5, HALF[dtype])
    assert np.all(np.abs(xo.numpy() - wx) <= bx) and np.all(np.abs(h.numpy() - wh) <= bh)
    assert xo.untouched() and h.untouched()


def test_route_of_more_rows():
    n = (1 << 26) + 5                                     # a wavefront each
    out = np.random.default_rng(2).random(n) < 0.25
    ids, w = DeviceArray(np.full((n, 1), 77, np.int32)), DeviceArray(np.full((n, 1), 5, np.float32))
    ops.route(DeviceArray(np.where(out, np.float32(-np.inf), np.float32(0.5))[:, None]), ids, w, scale=2.5)
    sync()
    assert np.array_equal(ids.numpy()[:, 0], np.where(out, -1, 0)) and np.array_equal(w.numpy()[:, 0], np.where(out, np.float32(0), np.float32(2.5)))
    assert ids.untouched() and w.untouched()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_experts_of_more_rows(dtype):
    n = (1 << 24) + 5
    Experts(n, 1, 1, 2, 1, dtype, ids=np.random.default_rng(3).integers(-1, 2, (n, 1))).run()


def test_experts_of_more_workgroups():
    """1024 experts whose first product has 8193 blocks of rows each: more than 2^31 threads."""
    n, E, F, D = 1100, 1024, (1 << 18) + 24, 4
    rng = np.random.default_rng(4)
    ids = (np.arange(n, dtype=np.int32) % E)[:, None]
    x, w = rng.standard_normal((n, D)).astype(np.float32), rng.random((n, 1)).astype(np.float32)
    some = (5, 1023)                                      # the others are zeros
    mats = [Far((E,) + s, (F * D, s[1], 1), "float32") for s in ((F, D), (F, D), (D, F))]
    values = {e: [(rng.standard_normal(s) * s[1] ** -0.5).astype(np.float32) for s in ((F, D), (F, D), (D, F))] for e in some}
    for e, v in values.items():
        for far, m in zip(mats, v):
            far.write(e * F * D, m)
    y = DeviceArray(np.full((n, D), 3, np.float32))
    ws = Far((ops.experts_workspace(n, 1, E, D, F, "float32"),), (1,), "uint8")
    ws.numel = lambda: ws.shape[0]
    ops.experts(DeviceArray(x), DeviceArray(ids), DeviceArray(w), *mats, y, ws)
    sync()
    got = y.numpy()
    for e, v in values.items():
        t = np.nonzero(ids[:, 0] == e)[0]
        want, bound = ref.experts(x[t], np.zeros((len(t), 1), np.int32), w[t], *(m[None] for m in v), "silu", ref.U32)
        assert np.all(np.abs(got[t] - want) <= bound)
    assert np.all(got[~np.isin(ids[:, 0], some)] == 0) and y.untouched()
