"""Operators on device memory (include/nanollama_ops.h): a feed-forward of experts in three calls.

    route(logits, ids, weights, ...)                                     scores of every expert -> each token's experts and weights
    experts(x, ids, weights, gate, up, down, out, workspace, ...)        weighted sum of the chosen experts' gated products
    residual_norm(x, d, x_out, h, ...)                                   x_out = x + scale gate norm(d), h = norm(x_out)

Arrays are anything with data_ptr(), shape, stride(), dtype and device.index as a torch tensor has them (torch itself is not needed, nor
imported): outputs are passed in, rows may be further apart than they are long, everything else lies densely.  Work is queued on `stream`
(a HIP stream's number; 0: the default stream of the arrays' device); nothing waits for it.
"""
from __future__ import annotations

from functools import lru_cache

from . import _lib
from .stack import ACTIVATIONS, DTYPES, SCORES


_names: dict = {}               # an array library's type -> its name


def _type(a) -> str:
    t = _names.get(a.dtype)
    if t is None:
        t = _names[a.dtype] = str(a.dtype).rpartition(".")[2]
    return t


def _shapes(**arrays) -> None:
    """Refuses arrays that do not have so many dimensions: name=(array, dimensions)."""
    for name, (a, dimensions) in arrays.items():
        if len(a.shape) != dimensions:
            raise ValueError(f"{name}: {len(a.shape)} dimensions, expected {dimensions}")


def _device(name: str, a) -> int:
    """Where an operator runs: with its first array."""
    index = a.device.index
    if index is None:
        raise ValueError(f"{name}: in host memory")
    return index


def _array(name: str, a, dtype: str, shape: tuple, device=None, strided=False):
    """Pointer and row distance of an array that has to have this type and shape."""
    if _names.get(a.dtype) != dtype and _type(a) != dtype:
        raise ValueError(f"{name}: type {_type(a)}, expected {dtype}")
    if a.shape != shape:
        raise ValueError(f"{name}: shape {list(a.shape)}, expected {list(shape)}")
    if device is not None and a.device.index != device:
        raise ValueError(f"{name}: on device {a.device.index}, the others on {device}")
    stride = a.stride()
    if stride[-1] == 1 and len(shape) <= 2:              # (nearly always)
        if len(shape) == 1 or stride[0] == shape[1]:
            return a.data_ptr(), shape[-1]
        if strided and shape[0] > 1 and stride[0] > shape[1]:
            return a.data_ptr(), stride[0]
    dense = 1
    for n, s in zip(reversed(shape), reversed(stride)):
        if n > 1 and s != dense:
            raise ValueError(f"{name}: elements are not dense" + (" within a row" if strided else ""))
        dense *= n
    return a.data_ptr(), shape[-1]


def _check(rc: int) -> None:
    if rc != 0:
        raise _lib.NlError(rc, (_lib.stack_lib().nl_last_error(None) or b"").decode())


def _int32(n: int) -> int:
    """A number that the library takes in 32 bits (ctypes would cut it off without a word)."""
    if not -1 << 31 <= n < 1 << 31:
        raise ValueError(f"{n}: more than 32 bits hold")
    return n


@lru_cache(maxsize=256)
def _desc(kind, *fields):
    """A description by its values (plain numbers: anything else would be found again by its identity); the library only reads it."""
    return kind(*(f if isinstance(f, float) else _int32(f) for f in fields))


def _one_of(name: str, value: str, table) -> int:
    if value not in table:
        raise ValueError(f"{name} {value!r}: one of {', '.join(table)}")
    return table[value]


def route(logits, ids, weights, score: str = "softmax", bias=None, renorm: bool = True, scale: float = 1.0, stream: int = 0) -> None:
    """logits [n, experts] float32 -> ids [n, k] int32, weights [n, k] float32; bias [experts] float32 joins sigmoid scores in the choice alone."""
    try:
        (n, count), (_, k) = logits.shape, ids.shape
    except ValueError:
        _shapes(logits=(logits, 2), ids=(ids, 2))
    dev = _device("logits", logits)
    lp, ld = _array("logits", logits, "float32", (n, count), strided=True)
    ip, _ = _array("ids", ids, "int32", (n, k), dev)
    wp, _ = _array("weights", weights, "float32", (n, k), dev)
    bp = None if bias is None else _array("bias", bias, "float32", (count,), dev)[0]
    d = _desc(_lib.NlRouteDesc, count, k, _one_of("score", score, SCORES), int(renorm), float(scale))
    _check(_lib.stack_lib().nl_op_route(dev, stream, d, _int32(n), lp, ld, bp, ip, wp))


def experts_workspace(n: int, per_token: int, count: int, dim: int, ff: int, dtype: str = "bfloat16") -> int:
    """Bytes that experts() needs beside its arrays for up to n tokens."""
    d = _desc(_lib.NlExpertsDesc, count, per_token, dim, ff, 0, _one_of("dtype", dtype, DTYPES))
    size = _lib.stack_lib().nl_op_experts_workspace(d, _int32(n))
    if size == 0:
        _check(-1)
    return size


def experts(x, ids, weights, gate, up, down, out, workspace, act: str = "silu", stream: int = 0) -> None:
    """out [n, dim] = sum over j of weights[:, j] * down[e] (act(gate[e] x) * up[e] x), e = ids[:, j]; an id that is no expert adds nothing.
    x [n, dim], gate and up [experts, ff, dim], down [experts, dim, ff], all of one type; workspace: experts_workspace() bytes of its own."""
    try:
        (n, dim), (count, ff, _), (_, k) = x.shape, gate.shape, ids.shape
    except ValueError:
        _shapes(x=(x, 2), gate=(gate, 3), ids=(ids, 2))
    dev, t = _device("x", x), _type(x)
    xp, ldx = _array("x", x, t, (n, dim), strided=True)
    ip, _ = _array("ids", ids, "int32", (n, k), dev)
    wp, _ = _array("weights", weights, "float32", (n, k), dev)
    gp, _ = _array("gate", gate, t, (count, ff, dim), dev)
    up_, _ = _array("up", up, t, (count, ff, dim), dev)
    dp, _ = _array("down", down, t, (count, dim, ff), dev)
    yp, ldy = _array("out", out, t, (n, dim), dev, strided=True)
    size = workspace.numel()
    sp, _ = _array("workspace", workspace, "uint8", (size,), dev)
    d = _desc(_lib.NlExpertsDesc, count, k, dim, ff, _one_of("act", act, ACTIVATIONS), _one_of("type of x", t, DTYPES))
    _check(_lib.stack_lib().nl_op_experts(dev, stream, d, _int32(n), xp, ldx, ip, wp, gp, up_, dp, yp, ldy, sp, size))


def residual_norm(x, d, x_out, h=None, pre=None, post=None, gate=None, scale: float = 1.0, eps: float = 1e-5, stream: int = 0) -> None:
    """x_out = x + scale * gate * (norm(d) * post), or d itself without post; h = norm(x_out) * pre.  x, x_out [n, dim] float32 (x_out may be x),
    d, h [n, dim] of one type, gate [dim] or [n, dim], post, pre [dim] float32."""
    _shapes(x=(x, 2))
    (n, dim), dev, t = x.shape, _device("x", x), _type(d)
    xp, ldx = _array("x", x, "float32", (n, dim), strided=True)
    dp, ldd = _array("d", d, t, (n, dim), dev, strided=True)
    op, ldo = _array("x_out", x_out, "float32", (n, dim), dev, strided=True)
    hp, ldh = (None, 0) if h is None else _array("h", h, t, (n, dim), dev, strided=True)
    if h is not None and pre is None:
        raise ValueError("h needs the gains pre")
    vec = lambda name, a: None if a is None else _array(name, a, "float32", (dim,), dev)[0]  # noqa: E731
    gp, ldg = None, 0
    if gate is not None:
        gp, ldg = (vec("gate", gate), 0) if len(gate.shape) == 1 else _array("gate", gate, "float32", (n, dim), dev, strided=True)
    desc = _desc(_lib.NlResidualNormDesc, dim, _one_of("type of d", t, DTYPES), float(eps), float(scale))
    _check(_lib.stack_lib().nl_op_residual_norm(dev, stream, desc, _int32(n), xp, ldx, dp, ldd, vec("post", post), gp, ldg, vec("pre", pre), op, ldo, hp, ldh))
