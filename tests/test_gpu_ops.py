"""Operators on device memory (nanollama_amd.ops) against 64-bit restatements, with bounds from the arithmetic (ops_reference.py)."""
import numpy as np
import pytest

from nanollama_amd import _lib, ops
from nanollama_amd.safetensors import from_bf16, to_bf16

import ops_reference as ref
from hip_arrays import DeviceArray, Stream, sync

pytestmark = pytest.mark.gpu
HALF = {"bfloat16": ref.U16, "float32": ref.U32}


def as_type(a, dtype):
    a = np.asarray(a, np.float32)
    return from_bf16(to_bf16(a)).reshape(a.shape) if dtype == "bfloat16" else a


# ---- route ----------------------------------------------------------------------------------------------------------------------

def run_route(logits, k, rows_apart=0, **kw):
    n = logits.shape[0]
    bias = kw.pop("bias", None)
    l = DeviceArray(logits, rows_apart=rows_apart, fill=9)
    ids, w = DeviceArray(np.full((n, k), 77, np.int32)), DeviceArray(np.full((n, k), 5, np.float32))
    ops.route(l, ids, w, bias=None if bias is None else DeviceArray(bias), **kw)
    sync()
    assert ids.untouched() and w.untouched() and l.untouched()
    return ids.numpy(), w.numpy()


def check_route(logits, k, rows_apart=0, **kw):
    ids, w = run_route(logits, k, rows_apart, **kw)
    want_ids, want_w, bound = ref.route(logits, k, **kw)
    assert np.array_equal(ids, want_ids)
    assert np.all(np.abs(w - want_w) <= bound), float(np.max(np.abs(w - want_w) / np.maximum(bound, 1e-300)))


@pytest.mark.parametrize("E, k", [(1, 1), (2, 1), (3, 3), (7, 2), (63, 8), (64, 8), (65, 6), (96, 6), (128, 32), (200, 12), (256, 8), (500, 5), (1024, 32)])
@pytest.mark.parametrize("score, bias", [("softmax", False), ("sigmoid", False), ("sigmoid", True)])
def test_route(E, k, score, bias):
    rng = np.random.default_rng(E * 40 + k)
    for n, renorm, scale in ((1, True, 1.0), (5, False, 1.0), (67, True, 2.5)):
        logits = (2 * rng.standard_normal((n, E))).astype(np.float32)
        b = (0.2 * rng.standard_normal(E)).astype(np.float32) if bias else None
        check_route(logits, k, score=score, renorm=renorm, scale=scale, bias=b, rows_apart=E + 3 if n > 1 else 0)


def test_route_equal_and_neighbouring_keys():
    rng = np.random.default_rng(3)
    # few different values: ties everywhere
    check_route(rng.integers(-2, 3, (40, 100)).astype(np.float32), 12, renorm=False)
    check_route(rng.integers(-2, 3, (40, 100)).astype(np.float32), 12, score="sigmoid", bias=(rng.integers(-1, 2, 100) / 4).astype(np.float32))
    check_route(np.zeros((3, 130), np.float32), 32)
    check_route(np.where(rng.random((20, 70)) < 0.5, 0.0, -0.0).astype(np.float32), 9)
    # one 32-bit step apart: the keys with a bias differ by less than 32 bits hold
    l = np.full((30, 64), 0.3, np.float32)
    for t in range(30):
        for e in range(64):
            for _ in range(int(rng.integers(0, 4))):
                l[t, e] = np.nextafter(l[t, e], np.float32(1))
    check_route(l, 8, score="sigmoid", bias=np.full(64, 0.11, np.float32))
    check_route(l + 3, 8, score="sigmoid", bias=np.full(64, -40.0, np.float32))
    check_route(-l * 30, 8, score="sigmoid", bias=np.zeros(64, np.float32))
    check_route(l, 8)


def test_route_masked_infinite_and_unknown_logits():
    rng = np.random.default_rng(4)
    l = rng.standard_normal((12, 70)).astype(np.float32)
    l[0] = -np.inf                                        # nobody
    l[1, 1:] = -np.inf                                    # one expert, of five asked for
    l[2] = np.nan
    l[3, ::2] = np.nan
    l[4, 5] = np.inf                                      # one for sure
    l[5, [7, 66, 3]] = np.inf                             # three share
    l[6] = np.finfo(np.float32).min
    l[7] = np.finfo(np.float32).max
    l[8, 10:] = np.finfo(np.float32).min                  # a mask of the type's lowest value, with places to spare and without
    l[9, 3:] = np.finfo(np.float32).min
    l[10] = -200.0                                        # sigmoids that are 0 in 32 bits
    b = rng.standard_normal(70).astype(np.float32)
    b[11], b[12], b[13] = np.nan, -np.inf, np.inf
    for renorm in (True, False):
        check_route(l, 5, renorm=renorm)
        check_route(l, 5, score="sigmoid", renorm=renorm)
        check_route(l, 5, score="sigmoid", renorm=renorm, bias=b)


# ---- experts --------------------------------------------------------------------------------------------------------------------

class Experts:
    def __init__(self, n, dim, ff, E, k, dtype, seed=0, ids=None, x_apart=0, y_apart=0, shift=0, act="silu"):
        rng = np.random.default_rng(seed)
        self.dtype, self.act, self.sizes = dtype, act, (n, k, E, dim, ff)
        t = lambda a: as_type(a, dtype)  # noqa: E731
        self.x = t(rng.standard_normal((n, dim)))
        self.gate, self.up = (t(rng.standard_normal((E, ff, dim)) * dim ** -0.5) for _ in range(2))
        self.down = t(rng.standard_normal((E, dim, ff)) * ff ** -0.5)
        self.ids = np.array([rng.permutation(E)[:k] for _ in range(n)], np.int32).reshape(n, k) if ids is None else np.asarray(ids, np.int32)
        self.w = rng.random((n, k)).astype(np.float32)
        self.dx = DeviceArray(self.x, dtype, rows_apart=x_apart, shift=shift, fill=0x7fc0 if dtype == "bfloat16" else np.nan)
        self.dg, self.du, self.dd = (DeviceArray(a, dtype, shift=shift, fill=0x7fc0 if dtype == "bfloat16" else np.nan) for a in (self.gate, self.up, self.down))
        self.di, self.dw = DeviceArray(self.ids), DeviceArray(self.w)
        self.y = DeviceArray(np.full((n, dim), 3.0), dtype, rows_apart=y_apart, fill=7)
        self.ws = self.workspace()

    def workspace(self):
        n, k, E, dim, ff = self.sizes
        return DeviceArray(np.full(ops.experts_workspace(n, k, E, dim, ff, self.dtype), 0xff, np.uint8))

    def queue(self, stream=0, y=None, ws=None):
        ops.experts(self.dx, self.di, self.dw, self.dg, self.du, self.dd, y or self.y, ws or self.ws, act=self.act, stream=stream)

    def want(self):
        return ref.experts(self.x, self.ids, self.w, self.gate, self.up, self.down, self.act, HALF[self.dtype])

    def check(self, y=None):
        y = y or self.y
        want, bound = self.want()
        got = y.numpy()
        assert np.all(np.abs(got - want) <= bound), float(np.nanmax(np.abs(got - want) / bound))
        assert y.untouched() and self.ws.untouched()

    def run(self):
        self.queue()
        sync()
        self.check()
        return self.y.bits()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("n, dim, ff, E, k", [(1, 32, 16, 4, 2), (1, 64, 40, 1, 1), (2, 40, 24, 8, 3), (3, 768, 512, 64, 8), (16, 96, 200, 5, 2), (17, 64, 64, 1, 1), (33, 136, 72, 12, 4),
                                              (64, 256, 128, 64, 6), (100, 160, 96, 3, 3), (150, 320, 264, 2, 1), (300, 128, 128, 130, 4), (513, 72, 56, 4, 2)])
def test_experts(n, dim, ff, E, k, dtype):
    Experts(n, dim, ff, E, k, dtype, seed=n).run()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("n, dim, ff", [(5, 33, 17), (20, 1, 1), (1, 7, 3), (40, 101, 50), (9, 36, 20), (200, 65, 130)])
def test_experts_of_odd_widths(n, dim, ff, dtype):
    Experts(n, dim, ff, 6, 2, dtype, seed=n).run()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_experts_rows_apart_and_off_the_boundary(dtype):
    for n in (3, 40, 300):
        Experts(n, 64, 48, 4, 2, dtype, x_apart=72, y_apart=80).run()
        Experts(n, 64, 48, 4, 2, dtype, x_apart=67, y_apart=65).run()
        Experts(n, 64, 48, 4, 2, dtype, shift=1).run()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_experts_ids_that_are_none_and_ids_that_come_twice(dtype):
    ids = np.array([[0, 3], [-1, -1], [2, -1], [-1, 1], [7, 4], [2, 2], [-2 ** 31, 2 ** 31 - 1], [3, 3], [1, 0]], np.int32)      # five experts
    for reps in (1, 30):
        m = Experts(9 * reps, 64, 40, 5, 2, dtype, ids=np.tile(ids, (reps, 1)))
        m.w[np.logical_or(m.ids < 0, m.ids >= 5)] = np.nan          # what is not chosen has any weight
        m.dw.write(m.w)
        clean = np.where(np.isnan(m.w), 0, m.w)
        m.queue()
        sync()
        want, bound = ref.experts(m.x, m.ids, clean, m.gate, m.up, m.down, "silu", HALF[dtype])
        got = m.y.numpy()
        assert np.all(np.abs(got - want) <= bound)
        assert np.all(got[[1, 6]] == 0)
    # no expert at all, and every token at one
    m = Experts(50, 64, 40, 5, 2, dtype, ids=np.full((50, 2), -1))
    m.run()
    assert np.all(m.y.numpy() == 0)
    Experts(50, 64, 40, 5, 1, dtype, ids=np.full((50, 1), 4)).run()
    Experts(333, 64, 40, 5, 1, dtype, ids=np.full((333, 1), 0)).run()


def test_experts_unused_matrices_may_hold_anything():
    for n in (2, 60):
        m = Experts(n, 64, 40, 6, 2, "bfloat16", ids=np.tile([[1, 4]], (n, 1)))
        for a, d in ((m.gate, m.dg), (m.up, m.du), (m.down, m.dd)):
            bad = a.copy()
            bad[[0, 2, 3, 5]] = np.nan
            d.write(bad)
        m.run()


def test_experts_gelu_and_large_arguments():
    for n in (4, 200):
        Experts(n, 64, 40, 4, 2, "float32", act="gelu_tanh").run()
        m = Experts(n, 64, 40, 4, 2, "bfloat16")
        m.gate, m.x = m.gate * 16, m.x * 4                       # sigmoids of up to +- 200
        m.dg.write(m.gate)
        m.dx.write(m.x)
        m.run()


def test_experts_zero_rows_and_more_experts_than_slots():
    m = Experts(2, 64, 40, 1024, 1, "bfloat16")
    m.run()
    before = m.y.bits()
    empty = DeviceArray(np.zeros((0, 64)), "bfloat16")
    ops.experts(empty, DeviceArray(np.zeros((0, 1), np.int32)), DeviceArray(np.zeros((0, 1), np.float32)), m.dg, m.du, m.dd, empty, m.ws)
    sync()
    assert np.array_equal(before, m.y.bits())


def test_experts_the_same_bits_every_time():
    m = Experts(200, 128, 136, 9, 3, "bfloat16")
    first = m.run()
    for _ in range(3):
        assert np.array_equal(first, m.run())


def test_experts_two_streams_and_graphs_with_workspaces_of_their_own():
    s1, s2 = Stream(), Stream()
    a, b = Experts(40, 96, 64, 6, 2, "bfloat16", seed=1), Experts(3, 96, 64, 6, 2, "bfloat16", seed=2)
    for _ in range(4):
        a.queue(s1.number)
        b.queue(s2.number)
    s1.sync()
    s2.sync()
    a.check()
    b.check()
    want_a, want_b = a.y.bits(), b.y.bits()
    play_a, play_b = s1.capture(lambda: a.queue(s1.number)), s2.capture(lambda: b.queue(s2.number))
    zero = np.zeros(a.y.shape)
    for _ in range(4):
        a.y.write(zero)
        b.y.write(zero[:3])
        sync()
        play_a()
        play_b()
        s1.sync()
        s2.sync()
        assert np.array_equal(a.y.bits(), want_a) and np.array_equal(b.y.bits(), want_b)
        b.queue()                                        # eager work between the replays
        sync()
        assert np.array_equal(b.y.bits(), want_b)
    # new inputs in the old places
    rng = np.random.default_rng(9)
    a.x, a.ids = as_type(rng.standard_normal(a.x.shape), "bfloat16"), rng.integers(-1, 6, a.ids.shape).astype(np.int32)
    a.dx.write(a.x)
    a.di.write(a.ids)
    play_a()
    s1.sync()
    a.check()


# ---- residual_norm --------------------------------------------------------------------------------------------------------------

def close_case(n, dim, dtype, post=True, gate="channel", h=True, scale=0.7, in_place=False, apart=0, seed=0, size=1.0, eps=1e-5):
    rng = np.random.default_rng(seed + n + dim)
    x, d = (size * rng.standard_normal((n, dim))).astype(np.float32), as_type(0.5 * size * rng.standard_normal((n, dim)), dtype)
    g = None if gate == "none" else rng.standard_normal(dim if gate == "channel" else (n, dim)).astype(np.float32)
    po = (1 + 0.1 * rng.standard_normal(dim)).astype(np.float32) if post else None
    pr = (1 + 0.1 * rng.standard_normal(dim)).astype(np.float32)
    dev = lambda a, t=None, **kw: None if a is None else DeviceArray(a, t, **kw)  # noqa: E731
    dx = dev(x, rows_apart=apart)
    xo = dx if in_place else dev(np.full((n, dim), 9, np.float32), rows_apart=apart)
    dh = dev(np.full((n, dim), 4.0), dtype, rows_apart=apart) if h else None
    ops.residual_norm(dx, dev(d, dtype, rows_apart=apart), xo, dh, pre=dev(pr) if h else None, post=dev(po),
                      gate=dev(g, rows_apart=apart if gate == "token" else 0), scale=scale, eps=eps)
    sync()
    wx, wh, bx, bh = ref.residual_norm(x, d, pr, po, g, scale, eps, HALF[dtype])
    assert np.all(np.abs(xo.numpy() - wx) <= bx), float(np.max(np.abs(xo.numpy() - wx) / bx))
    assert xo.untouched()
    if h:
        assert np.all(np.abs(dh.numpy() - wh) <= bh), float(np.max(np.abs(dh.numpy() - wh) / bh))
        assert dh.untouched()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("dim", [1, 2, 7, 64, 100, 255, 256, 768, 1023, 1024, 1536, 2047, 2048, 4096, 4100, 8192, 11008, 16384, 20000, 33001])
def test_residual_norm(dim, dtype):
    for n, post, gate in ((1, True, "channel"), (3, False, "token"), (9, True, "none")):
        close_case(n, dim, dtype, post, gate)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_residual_norm_variants(dtype):
    for dim in (96, 770, 1536):
        close_case(5, dim, dtype, h=False)
        close_case(5, dim, dtype, in_place=True)
        close_case(5, dim, dtype, in_place=True, gate="token", apart=dim + 24)
        close_case(5, dim, dtype, gate="token", apart=dim + 3)
        close_case(5, dim, dtype, size=0.0)                      # rows of zeros: norms of eps
        close_case(5, dim, dtype, size=1e-4, eps=0.0)
        close_case(5, dim, dtype, scale=0.0)
        close_case(700, dim, dtype)


# ---- all of a block, as it is used ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("n", [1, 6, 90])
def test_a_block(n, dtype):
    """route, experts and residual_norm behind one another on a stream of their own, eager and as a graph."""
    E, k, dim, ff = 12, 3, 96, 72
    m = Experts(n, dim, ff, E, k, dtype, seed=n)
    rng = np.random.default_rng(n)
    logits, bias = rng.standard_normal((n, E)).astype(np.float32), (0.1 * rng.standard_normal(E)).astype(np.float32)
    res, post, pre = rng.standard_normal((n, dim)).astype(np.float32), np.ones(dim, np.float32), (1 + 0.1 * rng.standard_normal(dim)).astype(np.float32)
    dl, db, dr, dpo, dpr = (DeviceArray(a) for a in (logits, bias, res, post, pre))
    xo, h = DeviceArray(np.zeros((n, dim), np.float32)), DeviceArray(np.zeros((n, dim)), dtype)
    s = Stream()

    def block():
        ops.route(dl, m.di, m.dw, score="sigmoid", bias=db, scale=2.5, stream=s.number)
        m.queue(s.number)
        ops.residual_norm(dr, m.y, xo, h, pre=dpr, post=dpo, scale=0.5, stream=s.number)

    def check():
        m.ids, m.w, _ = ref.route(logits, k, "sigmoid", bias, True, 2.5)
        assert np.array_equal(m.di.numpy(), m.ids)
        m.w = m.dw.numpy()
        m.check()
        wx, wh, bx, bh = ref.residual_norm(res, m.y.numpy(), pre, post, None, 0.5, 1e-5, HALF[dtype])
        assert np.all(np.abs(xo.numpy() - wx) <= bx) and np.all(np.abs(h.numpy() - wh) <= bh)

    block()
    s.sync()
    check()
    play = s.capture(block)
    for i in range(3):
        logits = rng.standard_normal((n, E)).astype(np.float32)
        dl.write(logits)
        play()
        s.sync()
        check()


def test_refusals_on_the_device():
    m = Experts(3, 32, 16, 4, 2, "bfloat16")
    L = _lib.stack_lib()
    d = _lib.NlRouteDesc(4, 2, 0, 1, 1.0)
    for device in (-1, 99):
        assert L.nl_op_route(device, None, d, 3, m.dw.data_ptr(), 4, None, m.di.data_ptr(), m.dw.data_ptr()) == -1
        assert b"device" in L.nl_last_error(None)
