"""Padded batches and rows in place (nanollama_amd.ops): what lies in rows that nobody asks for reaches no other row."""
import numpy as np
import pytest

import ops_reference as ref
from hip_arrays import DeviceArray, Stream, sync
from nanollama_amd import ops
from test_gpu_ops import HALF, Experts, close_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("dim, ff", [(64, 40), (66, 34), (65, 33)])
@pytest.mark.parametrize("n", [2, 30, 300])
def test_padded_tokens_of_anything(n, dim, ff, dtype):
    m = Experts(n, dim, ff, 8, 2, dtype, seed=n)
    pad = np.arange(n) % 3 == 1
    m.ids[pad], m.w[pad] = -1, np.nan
    m.x[pad] = np.where(np.arange(dim) % 2, np.nan, np.inf)
    m.di.write(m.ids)
    m.dw.write(m.w)
    m.dx.write(m.x)
    m.queue()
    sync()
    got = m.y.numpy()
    assert np.all(got[pad] == 0)
    want, bound = ref.experts(m.x[~pad], m.ids[~pad], m.w[~pad], m.gate, m.up, m.down, m.act, HALF[dtype])
    assert np.all(np.abs(got[~pad] - want) <= bound)
    assert m.y.untouched() and m.ws.untouched()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_padded_block(dtype):
    """Rows of logits that are all out, then experts and the close: eager and replayed."""
    n, E, k, dim = 50, 70, 6, 96
    m = Experts(n, dim, 48, E, k, dtype, seed=5)
    rng = np.random.default_rng(6)
    pad = rng.random(n) < 0.4
    logits, x = rng.standard_normal((n, E)).astype(np.float32), rng.standard_normal((n, dim)).astype(np.float32)
    logits[pad], x[pad], m.x[pad] = -np.inf, np.nan, np.nan
    m.dx.write(m.x)
    dl, dr, one = DeviceArray(logits), DeviceArray(x), DeviceArray(np.ones(dim, np.float32))
    xo, h = DeviceArray(np.zeros((n, dim), np.float32)), DeviceArray(np.zeros((n, dim)), dtype)
    s = Stream()

    def block():
        ops.route(dl, m.di, m.dw, stream=s.number)
        m.queue(s.number)
        ops.residual_norm(dr, m.y, xo, h, pre=one, post=one, stream=s.number)

    def check():
        ids, w = m.di.numpy(), m.dw.numpy()
        assert np.all(ids[pad] == -1) and np.all(w[pad] == 0) and np.all(m.y.numpy()[pad] == 0)
        want, bound = ref.experts(m.x[~pad], ids[~pad], w[~pad], m.gate, m.up, m.down, "silu", HALF[dtype])
        y = m.y.numpy()[~pad]
        assert np.all(np.abs(y - want) <= bound)
        wx, wh, bx, bh = ref.residual_norm(x[~pad], y, np.ones(dim), np.ones(dim), None, 1.0, 1e-5, HALF[dtype])
        assert np.all(np.abs(xo.numpy()[~pad] - wx) <= bx) and np.all(np.abs(h.numpy()[~pad] - wh) <= bh)
        assert np.all(np.isnan(xo.numpy()[pad]))

    block()
    s.sync()
    check()
    play = s.capture(block)
    for _ in range(3):
        play()
        s.sync()
        check()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("dim", [4096, 4097, 5120, 11009])
def test_wide_rows_in_place(dim, dtype):
    close_case(3, dim, dtype, in_place=True)
    close_case(3, dim, dtype, in_place=True, gate="token", apart=dim + 24)
    close_case(3, dim, dtype, in_place=True, post=False, gate="none", apart=dim + 3)
    close_case(3, dim, dtype, h=False, size=0.0)
