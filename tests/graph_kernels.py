"""Which kernels a call queues: the call is recorded into a graph (nothing runs), its kernel nodes are named."""
import ctypes as C
import re

from hip_arrays import Stream, hip, ok


class _Dim3(C.Structure):
    _fields_ = [("x", C.c_uint32), ("y", C.c_uint32), ("z", C.c_uint32)]


class _KernelNode(C.Structure):
    _fields_ = [("block", _Dim3), ("extra", C.c_void_p), ("func", C.c_void_p), ("grid", _Dim3), ("params", C.c_void_p), ("lds", C.c_uint32)]


def queued(work):
    """Mangled names of the kernels that work(stream's number) queues, in order."""
    h = hip()
    h.hipKernelNameRefByPtr.restype = C.c_char_p
    h.hipKernelNameRefByPtr.argtypes = [C.c_void_p, C.c_void_p]
    for name in ("hipGraphGetNodes", "hipGraphNodeGetType", "hipGraphKernelNodeGetParams"):
        getattr(h, name).restype = C.c_int
    s = Stream()
    ok(h.hipStreamBeginCapture(s.handle, 1))
    work(s.number)
    graph, count = C.c_void_p(), C.c_size_t()
    ok(h.hipStreamEndCapture(s.handle, C.byref(graph)))
    ok(h.hipGraphGetNodes(graph, None, C.byref(count)))
    nodes = (C.c_void_p * count.value)()
    ok(h.hipGraphGetNodes(graph, nodes, C.byref(count)))
    names = []
    for node in nodes:
        kind, p = C.c_int(-1), _KernelNode()
        ok(h.hipGraphNodeGetType(C.c_void_p(node), C.byref(kind)))
        assert kind.value == 0, "not a kernel"
        ok(h.hipGraphKernelNodeGetParams(C.c_void_p(node), C.byref(p)))
        names.append(h.hipKernelNameRefByPtr(p.func, s.handle).decode())
    ok(h.hipGraphDestroy(graph))
    return names


def product_forms(names):
    """The experts' products among them, first and second: (rows, tokens, stages, bytes a piece, pairs) of a tile, "slots" (slot by slot) or "elements"."""
    forms = {}
    for name in names:
        if "experts_" not in name:
            continue
        template = name.partition("_kernelI")[2]
        if "experts_token_" in name:
            first, form = "experts_token_first" in name, "slots"
        else:
            first, form = bool(int(re.search(r"Lb([01])E", template).group(1))), "elements"
            if "experts_many_kernel" in name:
                rtw, ntw, wr, wt, stages, unit, pair = (int(v) for v in re.findall(r"L[ib](\d+)E", template.partition("Grouped")[2]))
                form = (wr * rtw * 16, wt * ntw * 16, stages, unit, bool(pair))
        assert first not in forms, names
        forms[first] = form
    return forms[True], forms[False]
