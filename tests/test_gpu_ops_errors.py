"""What an operator leaves behind: errors of its own launches are told once, by the call that met them (nanollama_amd.ops)."""
import ctypes as C

import numpy as np
import pytest

from hip_arrays import DeviceArray, Stream, hip, ok, sync
from nanollama_amd import _lib, ops

pytestmark = pytest.mark.gpu


def test_an_error_is_not_the_next_calls():
    """A stream whose recording has become invalid refuses launches; nothing of that may reach the program's next look at the runtime's last error."""
    h, s = hip(), Stream()
    l, ids, w = DeviceArray(np.arange(32, dtype=np.float32).reshape(4, 8)), DeviceArray(np.zeros((4, 2), np.int32)), DeviceArray(np.zeros((4, 2), np.float32))
    ok(h.hipStreamBeginCapture(s.handle, 1))
    assert h.hipStreamSynchronize(s.handle) != 0          # not allowed while it records
    h.hipGetLastError()
    with pytest.raises(_lib.NlError, match="route: "):
        ops.route(l, ids, w, stream=s.number)
    left = h.hipPeekAtLastError()
    graph = C.c_void_p()
    assert h.hipStreamEndCapture(s.handle, C.byref(graph)) != 0
    h.hipGetLastError()
    assert left == 0
    ops.route(l, ids, w)
    sync()
    assert np.array_equal(ids.numpy(), np.tile([[7, 6]], (4, 1)))


@pytest.mark.parametrize("stream", [0, 1, 2])             # the default stream, by its other name, and this thread's own
def test_default_streams_have_handles(stream):
    rng = np.random.default_rng(stream)
    logits = rng.standard_normal((5, 8)).astype(np.float32)
    l, ids, w = DeviceArray(logits), DeviceArray(np.zeros((5, 2), np.int32)), DeviceArray(np.zeros((5, 2), np.float32))
    sync()
    ops.route(l, ids, w, stream=stream)
    sync()
    assert np.array_equal(ids.numpy(), np.argsort(-logits, axis=1, kind="stable")[:, :2])
