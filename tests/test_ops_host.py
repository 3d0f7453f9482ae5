"""Operators on device memory without a GPU: their surface, and every refusal that comes in front of the device."""
import ctypes as C
import os
import re
from types import SimpleNamespace

import pytest

from nanollama_amd import _lib, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20          # a pointer that nothing follows: every call here is refused in front of the device


def route(n=4, experts=8, per_token=2, score=0, renorm=1, scale=1.0, logits=P, ld=8, bias=None, ids=P, weights=P, desc=True):
    L = _lib.stack_lib()
    d = _lib.NlRouteDesc(experts, per_token, score, renorm, scale)
    return L.nl_op_route(0, None, d if desc else None, n, logits, ld, bias, ids, weights), (L.nl_last_error(None) or b"").decode()


def experts(n=4, count=8, per_token=2, dim=32, ff=16, act=1, dtype=0, ldx=32, ldy=32, size=1 << 30, desc=True, **null):
    L = _lib.stack_lib()
    d = _lib.NlExpertsDesc(count, per_token, dim, ff, act, dtype)
    at = {k: P for k in ("x", "ids", "weights", "gate", "up", "down", "y", "ws")}
    at.update(null)
    return L.nl_op_experts(0, None, d if desc else None, n, at["x"], ldx, at["ids"], at["weights"], at["gate"], at["up"], at["down"], at["y"], ldy, at["ws"], size), \
        (L.nl_last_error(None) or b"").decode()


def close(n=4, dim=32, dtype=0, eps=1e-5, scale=1.0, ldx=32, ldb=32, ldg=0, ldxo=32, ldh=32, desc=True, **null):
    L = _lib.stack_lib()
    d = _lib.NlResidualNormDesc(dim, dtype, eps, scale)
    at = {"x": P, "b": P, "post": P, "gate": None, "pre": P, "xo": 2 * P, "h": P}
    at.update(null)
    return L.nl_op_residual_norm(0, None, d if desc else None, n, at["x"], ldx, at["b"], ldb, at["post"], at["gate"], ldg, at["pre"], at["xo"], ldxo, at["h"], ldh), \
        (L.nl_last_error(None) or b"").decode()


def test_the_header_declares_what_the_library_exports():
    L = C.CDLL(_lib.STACK_LIB_PATH)
    declared = re.findall(r"NL_API\s+[\w\s\*]+?\b(nl_\w+)\s*\(", open(os.path.join(ROOT, "include", "nanollama_ops.h")).read())
    assert {"nl_op_route", "nl_op_experts", "nl_op_experts_workspace", "nl_op_residual_norm"} <= set(declared)
    for name in declared:
        assert hasattr(L, name) and name in _lib.STACK_EXPORTS, name


@pytest.mark.parametrize("call, kw, text", [
    (route, dict(desc=False), "no description"), (route, dict(n=-1), "negative"), (route, dict(experts=0), "0 experts"), (route, dict(experts=1025), "1025 experts"),
    (route, dict(per_token=0), "per token"), (route, dict(per_token=9), "per token"), (route, dict(experts=64, ld=64, per_token=33), "per token"),
    (route, dict(score=2), "score"), (route, dict(bias=P), "bias"), (route, dict(scale=float("nan")), "scale"), (route, dict(scale=float("inf")), "scale"),
    (route, dict(logits=None), "null"), (route, dict(ids=None), "null"), (route, dict(weights=None), "null"), (route, dict(ld=7), "ld 7"),
    (experts, dict(desc=False), "no description"), (experts, dict(n=-1), "n:"), (experts, dict(n=1 << 30), "n:"), (experts, dict(count=0), "experts"), (experts, dict(count=1025), "experts"),
    (experts, dict(per_token=0), "per_token"), (experts, dict(per_token=33), "per_token"), (experts, dict(dim=0), "dim"), (experts, dict(ff=-8), "dim and ff"),
    (experts, dict(act=2), "act"), (experts, dict(dtype=2), "dtype"), (experts, dict(ldx=31), "ldx"), (experts, dict(ldy=31), "ldy"), (experts, dict(size=100), "workspace"),
    (experts, dict(ws=P + 8), "16-byte"), *[(experts, {k: None}, "null") for k in ("x", "ids", "weights", "gate", "up", "down", "y", "ws")],
    (close, dict(desc=False), "no description"), (close, dict(n=-1), "negative"), (close, dict(dim=0), "dim"), (close, dict(dtype=7), "dtype"), (close, dict(eps=-1.0), "eps"),
    (close, dict(eps=float("nan")), "eps"), (close, dict(scale=float("inf")), "scale"), (close, dict(ldx=31), "row distance"), (close, dict(ldb=31), "row distance"),
    (close, dict(gate=P, ldg=31), "row distance"), (close, dict(ldxo=31), "row distance"), (close, dict(ldh=31), "row distance"), (close, dict(pre=None), "null"),
    (close, dict(xo=P, ldxo=40), "other rows"), (close, dict(x=None), "null"), (close, dict(b=None), "null"), (close, dict(xo=None), "null")])
def test_refusals(call, kw, text):
    rc, message = call(**kw)
    assert rc in (-1, -2) and text in message, (rc, message)


def test_no_tokens_is_no_work():
    assert [f(n=0)[0] for f in (route, experts, close)] == [0, 0, 0]


def test_workspace_sizes():
    size = ops.experts_workspace(7, 3, 5, 40, 24)
    assert size >= 7 * 3 * (40 * 4 + 24 * 2) + 6 * 4 + 21 * 4
    # activations of few tokens an expert take as much in either type, those of many half as much in bfloat16
    assert ops.experts_workspace(7, 3, 5, 40, 24, "float32") >= size
    assert ops.experts_workspace(700, 3, 5, 40, 24, "float32") >= ops.experts_workspace(700, 3, 5, 40, 24) + 2000 * 24 * 2
    # a workspace for n tokens serves fewer
    for dtype in ("bfloat16", "float32"):
        sizes = [ops.experts_workspace(n, 3, 50, 40, 24, dtype) for n in range(400)]
        assert sizes == sorted(sizes)
    assert ops.experts_workspace(0, 3, 5, 40, 24) > 0
    with pytest.raises(_lib.NlError, match="per_token"):
        ops.experts_workspace(7, 0, 5, 40, 24)
    with pytest.raises(ValueError, match="dtype"):
        ops.experts_workspace(7, 3, 5, 40, 24, "float16")


class Fake:
    def __init__(self, *shape, dtype="bfloat16", stride=None, device=0):
        self.shape, self.dtype, self.device = shape, dtype, SimpleNamespace(index=device)
        d, s = 1, []
        for n in reversed(shape):
            s.append(d)
            d *= n
        self._stride, self._n = stride or tuple(reversed(s)), d

    def data_ptr(self):
        return P

    def stride(self):
        return self._stride

    def numel(self):
        return self._n


def _experts(**kw):
    a = dict(x=Fake(4, 32), ids=Fake(4, 2, dtype="int32"), weights=Fake(4, 2, dtype="float32"), gate=Fake(8, 16, 32), up=Fake(8, 16, 32), down=Fake(8, 32, 16),
             out=Fake(4, 32), workspace=Fake(100, dtype="uint8"))
    a.update(kw)
    ops.experts(**a)


@pytest.mark.parametrize("kw, text", [
    (dict(ids=Fake(4, 2, dtype="int64")), "ids: type int64"), (dict(weights=Fake(4, 3, dtype="float32")), "weights: shape"), (dict(up=Fake(8, 16, 24)), "up: shape"),
    (dict(down=Fake(8, 16, 32)), "down: shape"), (dict(gate=Fake(8, 16, 32, dtype="float32")), "gate: type"), (dict(x=Fake(4, 32, dtype="float16")), "type"),
    (dict(out=Fake(4, 32, stride=(16, 1))), "not dense"), (dict(x=Fake(4, 32, stride=(1, 4))), "not dense"), (dict(down=Fake(8, 32, 16, stride=(512, 1, 32))), "not dense"),
    (dict(gate=Fake(8, 16, 32, stride=(1024, 32, 1))), "not dense"), (dict(up=Fake(8, 16, 32, device=1)), "device"), (dict(act="relu"), "act")])
def test_arrays_that_do_not_fit(kw, text):
    with pytest.raises(ValueError, match=text):
        _experts(**kw)


def test_arrays_that_fit_reach_the_library():
    with pytest.raises(_lib.NlError, match="workspace of 100 bytes"):
        _experts()
    with pytest.raises(_lib.NlError, match="workspace of 100 bytes"):
        _experts(x=Fake(4, 32, stride=(40, 1)), out=Fake(4, 32, stride=(33, 1)))
    with pytest.raises(ValueError, match="score"):
        ops.route(Fake(4, 8, dtype="float32"), Fake(4, 2, dtype="int32"), Fake(4, 2, dtype="float32"), score="relu")
    with pytest.raises(ValueError, match="gains"):
        ops.residual_norm(Fake(4, 8, dtype="float32"), Fake(4, 8), Fake(4, 8, dtype="float32"), h=Fake(4, 8))
