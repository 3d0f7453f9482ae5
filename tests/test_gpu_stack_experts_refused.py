"""nl_stack_experts that finds no memory leaves the handle as it was (include/nanollama_ops.h)."""
import ctypes as C

import numpy as np
import pytest

from nanollama_amd import _lib

pytestmark = pytest.mark.gpu
WIDTH, FEW = 256, (8, 2, 32, 1, 1, 1, 1, 1.0)             # 8 experts of 32 with sigmoid scores and a bias
TOO_MANY = (1024, 2, 1 << 20, 1, 1, 1, 1, 1.0)            # 1.1 TB a matrix


def create():
    L = _lib.stack_lib()
    cfg = _lib.NlStackConfig(32, WIDTH, 1, 0, 0, 1, 64, 1, 0, 0, 1, 0, 0, 0, 0, 1e-5, 1.0)
    layers = (_lib.NlLayerDesc * 1)()
    layers[0].lin = _lib.NlLinattnDesc(2, 16, 16, 4, 8.0, 1.0)
    h = C.c_void_p()
    assert L.nl_create_stack(C.byref(cfg), layers, C.byref(h)) == 0
    return L, h


def weights_held(L, h):
    w, kv, st = C.c_uint64(), C.c_uint64(), C.c_uint64()
    assert L.nl_memory_usage(h, C.byref(w), C.byref(kv), C.byref(st)) == 0
    return w.value


def test_a_call_that_finds_no_memory():
    L, h = create()
    before = weights_held(L, h)
    for _ in range(2):
        assert L.nl_stack_experts(h, 0, C.byref(_lib.NlStackExpertsDesc(*TOO_MANY))) < 0 and b"hipMalloc" in L.nl_last_error(h)
        assert weights_held(L, h) == before
    x = np.zeros((8 * WIDTH, WIDTH), np.float32)
    up = lambda name, rows, cols: L.nl_upload_tensor(h, name, 0, x.ctypes.data, rows * cols * 4, rows, cols)  # noqa: E731
    assert up(b"layers.0.norm1", 1, WIDTH) == 0, L.nl_last_error(h)         # the error is not the next call's
    assert up(b"layers.0.ff.router", 8, WIDTH) == -1                        # no experts yet
    assert L.nl_stack_experts(h, 0, C.byref(_lib.NlStackExpertsDesc(*FEW))) == 0
    assert up(b"layers.0.ff.router", 8, WIDTH) == 0 and up(b"layers.0.ff.experts.gate", 8 * 32, WIDTH) == 0 and up(b"layers.0.ff.experts.down", 8 * WIDTH, 32) == 0
    L2, other = create()
    assert L2.nl_stack_experts(other, 0, C.byref(_lib.NlStackExpertsDesc(*FEW))) == 0
    assert weights_held(L, h) == weights_held(L2, other)
    for handle in (h, other):
        L.nl_destroy(handle)
