"""Arrays in device memory for tests of operators that take pointers: numpy in, numpy out, no torch.  The HIP runtime is the one that the
library under test has loaded."""
import ctypes as C
from types import SimpleNamespace

import numpy as np

from nanollama_amd import _lib
from nanollama_amd.safetensors import from_bf16, to_bf16

_hip = None


def hip():
    global _hip
    if _hip is None:
        _lib.stack_lib()
        _hip = C.CDLL("libamdhip64.so.7")
        for name in ("hipMalloc", "hipFree", "hipMemcpy", "hipStreamCreateWithFlags", "hipStreamDestroy", "hipStreamSynchronize", "hipDeviceSynchronize",
                     "hipStreamBeginCapture", "hipStreamEndCapture", "hipGraphInstantiate", "hipGraphLaunch", "hipGraphExecDestroy", "hipGraphDestroy", "hipGetDevice"):
            getattr(_hip, name).restype = C.c_int
        _hip.hipMalloc.argtypes = [C.POINTER(C.c_void_p), C.c_size_t]
        _hip.hipFree.argtypes = [C.c_void_p]
        _hip.hipMemcpy.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int]
    return _hip


def ok(rc):
    assert rc == 0, f"HIP error {rc}"


def sync():
    ok(hip().hipDeviceSynchronize())


class DeviceArray:
    """What nanollama_amd.ops asks of an array.  dtype: float32, int32, uint8 or bfloat16 (held as its bits).  `rows_apart`: elements from a row of
    a matrix to the next, the space between filled with `fill`; `shift`: elements in front of the first one (alignment)."""

    def __init__(self, values, dtype=None, rows_apart=0, shift=0, fill=0):
        values = np.asarray(values)
        self.dtype = dtype or str(values.dtype)
        raw = to_bf16(values.astype(np.float32)).reshape(values.shape) if self.dtype == "bfloat16" else np.ascontiguousarray(values, self.dtype)
        self.shape, self.device = values.shape, SimpleNamespace(index=0)
        self._store, self._size = raw.dtype, raw.dtype.itemsize
        self._ld = rows_apart or (values.shape[-1] if values.ndim else 1)
        assert not rows_apart or (values.ndim == 2 and rows_apart >= values.shape[1])
        self._rows = int(np.prod(values.shape[:-1])) if values.ndim else 1
        self._shift, self._fill = shift, fill
        # (64 elements of fill behind the array too)
        image = np.full(shift + self._rows * self._ld + 64, fill, self._store)
        image[shift:shift + self._rows * self._ld].reshape(self._rows, self._ld)[:, :raw.shape[-1] if raw.ndim else 1] = raw.reshape(self._rows, -1 if self._rows else self._ld)
        self._image = image
        self._base = C.c_void_p()
        ok(hip().hipMalloc(C.byref(self._base), image.nbytes))
        ok(hip().hipMemcpy(self._base, image.ctypes.data, image.nbytes, 1))

    def __del__(self):
        if getattr(self, "_base", None):
            hip().hipFree(self._base)

    def data_ptr(self):
        return self._base.value + self._shift * self._size

    def numel(self):
        return int(np.prod(self.shape))

    def stride(self):
        out, d = [], 1
        for i in range(len(self.shape) - 1, -1, -1):
            out.append(d)
            d *= self._ld if i == len(self.shape) - 1 else self.shape[i]
        return tuple(out[::-1])

    def _read(self):
        image = np.empty_like(self._image)
        ok(hip().hipMemcpy(image.ctypes.data, self._base, image.nbytes, 2))
        return image

    def bits(self):
        """The values as they are stored."""
        body = self._read()[self._shift:self._shift + self._rows * self._ld].reshape(self._rows, self._ld)
        return body[:, :self.shape[-1]].reshape(self.shape).copy()

    def numpy(self):
        b = self.bits()
        return from_bf16(b).reshape(b.shape) if self.dtype == "bfloat16" else b

    def untouched(self):
        """Nothing but the array's own elements has changed."""
        image = self._read()
        image[self._shift:self._shift + self._rows * self._ld].reshape(self._rows, self._ld)[:, :self.shape[-1]] = 0
        was = self._image.copy()
        was[self._shift:self._shift + self._rows * self._ld].reshape(self._rows, self._ld)[:, :self.shape[-1]] = 0
        return np.array_equal(image, was)

    def write(self, values):
        raw = to_bf16(np.asarray(values, np.float32)).reshape(self.shape) if self.dtype == "bfloat16" else np.ascontiguousarray(values, self.dtype)
        self._image[self._shift:self._shift + self._rows * self._ld].reshape(self._rows, self._ld)[:, :self.shape[-1]] = raw.reshape(self._rows, -1 if self._rows else self._ld)
        ok(hip().hipMemcpy(self._base, self._image.ctypes.data, self._image.nbytes, 1))


class Stream:
    def __init__(self):
        self.handle = C.c_void_p()
        ok(hip().hipStreamCreateWithFlags(C.byref(self.handle), 1))      # (does not wait for the default stream)

    @property
    def number(self):
        return self.handle.value

    def sync(self):
        ok(hip().hipStreamSynchronize(self.handle))

    def capture(self, work):
        """The work queued by work() as a graph: a function that replays it on this stream."""
        ok(hip().hipStreamBeginCapture(self.handle, 1))
        work()
        graph, run = C.c_void_p(), C.c_void_p()
        ok(hip().hipStreamEndCapture(self.handle, C.byref(graph)))
        ok(hip().hipGraphInstantiate(C.byref(run), graph, None, None, 0))
        self._graphs = getattr(self, "_graphs", []) + [(graph, run)]
        return lambda: ok(hip().hipGraphLaunch(run, self.handle))

    def __del__(self):
        for graph, run in getattr(self, "_graphs", []):
            hip().hipGraphExecDestroy(run)
            hip().hipGraphDestroy(graph)
        if self.handle:
            hip().hipStreamDestroy(self.handle)
