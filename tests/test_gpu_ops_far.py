"""Many tokens, and elements that lie further than 32 bits reach (nanollama_amd.ops)."""
import ctypes as C
from types import SimpleNamespace

import numpy as np
import pytest

import ops_reference as ref
from hip_arrays import DeviceArray, hip, ok, sync
from nanollama_amd import ops
from nanollama_amd.safetensors import to_bf16
from test_gpu_ops import HALF, Experts, as_type, check_route, close_case

pytestmark = pytest.mark.gpu


class Far:
    """Zeroed device memory as an array of this shape and strides; parts of it are written and read."""

    def __init__(self, shape, stride, dtype):
        self.shape, self._stride, self.dtype, self.device = shape, stride, dtype, SimpleNamespace(index=0)
        self._size = 2 if dtype == "bfloat16" else 4
        n = (1 + sum((a - 1) * b for a, b in zip(shape, stride))) * self._size
        self._base = C.c_void_p()
        ok(hip().hipMalloc(C.byref(self._base), n))
        ok(hip().hipMemset(self._base, 0, C.c_size_t(n)))

    def __del__(self):
        hip().hipFree(self._base)

    def data_ptr(self):
        return self._base.value

    def stride(self):
        return self._stride

    def at(self, element):
        return C.c_void_p(self._base.value + element * self._size)

    def write(self, element, values):
        raw = to_bf16(np.asarray(values, np.float32)) if self.dtype == "bfloat16" else np.ascontiguousarray(values, self.dtype)
        ok(hip().hipMemcpy(self.at(element), raw.ctypes.data, raw.nbytes, 1))

    def read(self, element, n):
        out = np.empty(n, np.uint16 if self.dtype == "bfloat16" else self.dtype)
        ok(hip().hipMemcpy(out.ctypes.data, self.at(element), out.nbytes, 2))
        return (out.astype(np.uint32) << 16).view(np.float32) if self.dtype == "bfloat16" else out


def test_many_tokens():
    rng = np.random.default_rng(1)
    n = 70001
    Experts(n, 64, 32, 4, 1, "bfloat16", ids=rng.integers(-1, 4, (n, 1))).run()
    Experts(n, 24, 40, 300, 2, "float32", ids=rng.integers(0, 300, (n, 2))).run()
    check_route(rng.standard_normal((n, 9)).astype(np.float32), 3, renorm=False)
    check_route(rng.standard_normal((n, 70)).astype(np.float32), 2, score="sigmoid", bias=rng.standard_normal(70).astype(np.float32))
    close_case(n, 40, "bfloat16", gate="token")


def test_more_tiles_than_a_grid_is_high():
    n = 1_050_000
    Experts(n, 3, 1, 2, 1, "bfloat16", ids=np.random.default_rng(2).integers(0, 2, (n, 1))).run()


@pytest.mark.parametrize("n", [2, 40])                    # slot by slot, and grouped
def test_experts_behind_32_bits(n):
    E, F, D, e = 1024, 2048, 1032, 1023                   # 2.16e9 elements a matrix
    rng = np.random.default_rng(n)
    t = lambda a: as_type(a, "bfloat16")  # noqa: E731
    x, gate, up, down = t(rng.standard_normal((n, D))), *(t(rng.standard_normal(s) * s[1] ** -0.5) for s in ((F, D), (F, D), (D, F)))
    ids = np.full((n, 1), e, np.int32)
    ids[1::2] = 1022                                      # zeros
    w = rng.random((n, 1)).astype(np.float32)
    mats = [Far((E,) + m.shape, (F * D, m.shape[1], 1), "bfloat16") for m in (gate, up, down)]
    for far, m in zip(mats, (gate, up, down)):
        far.write(e * F * D, m)
    far_x = Far((n, D), (1 << 31 if n == 2 else D, 1), "bfloat16")
    for i in range(n):
        far_x.write(i * far_x.stride()[0], x[i])
    y = DeviceArray(np.full((n, D), 3.0), "bfloat16")
    ops.experts(far_x, DeviceArray(ids), DeviceArray(w), *mats, y, DeviceArray(np.zeros(ops.experts_workspace(n, 1, E, D, F), np.uint8)))
    sync()
    want, bound = ref.experts(x[::2], np.zeros((len(x[::2]), 1), np.int32), w[::2], gate[None], up[None], down[None], "silu", HALF["bfloat16"])
    got = y.numpy()
    assert np.all(np.abs(got[::2] - want) <= bound) and np.all(got[1::2] == 0)


def test_rows_behind_32_bits():
    rng = np.random.default_rng(5)
    ld = (1 << 31) + 4
    logits = rng.standard_normal((2, 50)).astype(np.float32)
    far = Far((2, 50), (ld, 1), "float32")
    for i in range(2):
        far.write(i * ld, logits[i])
    ids, w = DeviceArray(np.zeros((2, 4), np.int32)), DeviceArray(np.zeros((2, 4), np.float32))
    ops.route(far, ids, w)
    sync()
    want, weights, bound = ref.route(logits, 4)
    assert np.array_equal(ids.numpy(), want) and np.all(np.abs(w.numpy() - weights) <= bound)
    # in place, rows and gates as far apart
    dim = 768
    del far
    x, d, g = rng.standard_normal((2, dim)).astype(np.float32), rng.standard_normal((2, dim)).astype(np.float32), rng.standard_normal((2, dim)).astype(np.float32)
    fx, fg, fh = (Far((2, dim), (ld, 1), "float32") for _ in range(3))
    for i in range(2):
        fx.write(i * ld, x[i])
        fg.write(i * ld, g[i])
    ones = np.ones(dim, np.float32)
    ops.residual_norm(fx, DeviceArray(d), fx, fh, pre=DeviceArray(ones), post=DeviceArray(ones), gate=fg, scale=0.5)
    sync()
    wx, wh, bx, bh = ref.residual_norm(x, d, ones, ones, g, 0.5, 1e-5, HALF["float32"])
    for i in range(2):
        assert np.all(np.abs(fx.read(i * ld, dim) - wx[i]) <= bx[i]) and np.all(np.abs(fh.read(i * ld, dim) - wh[i]) <= bh[i])
