"""Arguments of nanollama_amd.ops on their way into the library, without a GPU."""
import math

import pytest

from nanollama_amd import _lib, ops
from test_ops_host import Fake


class Library:
    """Takes every call and keeps the descriptions' values."""

    def __init__(self):
        self.seen = []

    def __getattr__(self, name):
        def call(device, stream, d, n, *rest):
            self.seen.append((name, {f: getattr(d, f) for f, _ in d._fields_}, n))
            return 0
        return call


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    monkeypatch.setattr(_lib, "stack_lib", lambda: lib)
    return lib


class Number:
    """A number that changes in its place, as an array of one element does."""

    def __init__(self, value):
        self.value = value

    def __float__(self):
        return self.value


def test_numbers_are_read_at_every_call(library):
    f32 = lambda *shape: Fake(*shape, dtype="float32")  # noqa: E731
    scale, eps = Number(2.0), Number(0.5)
    for s, e in ((2.0, 0.5), (4.0, 0.25), (2.0, 0.125)):
        scale.value, eps.value = s, e
        ops.route(f32(4, 8), Fake(4, 2, dtype="int32"), f32(4, 2), scale=scale)
        ops.residual_norm(f32(4, 8), f32(4, 8), f32(4, 8), scale=scale, eps=eps)
        (_, route, _), (_, close, _) = library.seen[-2:]
        assert route["scale"] == s and close["scale"] == s and close["eps"] == e


def far(*shape, dtype="float32"):
    a = Fake(1, dtype=dtype)
    a.shape = shape
    a._stride = tuple(math.prod(shape[i + 1:]) for i in range(len(shape)))
    return a


@pytest.mark.parametrize("n", [1 << 31, (1 << 32) + 4])
def test_numbers_that_32_bits_do_not_hold_are_refused(library, n):
    ids, w = far(n, 1, dtype="int32"), far(n, 1)
    calls = [lambda: ops.route(far(n, 8), ids, w), lambda: ops.residual_norm(far(n, 8), far(n, 8), far(n, 8)),
             lambda: ops.experts(far(n, 8), ids, w, far(4, 8, 8), far(4, 8, 8), far(4, 8, 8), far(n, 8), Fake(100, dtype="uint8")),
             lambda: ops.experts_workspace(n, 1, 4, 8, 8), lambda: ops.experts_workspace(4, n, 4, 8, 8), lambda: ops.experts_workspace(4, 1, 4, n, 8),
             lambda: ops.residual_norm(far(1, n), far(1, n), far(1, n)), lambda: ops.route(far(1, n), far(1, 2, dtype="int32"), far(1, 2))]
    for call in calls:
        with pytest.raises(ValueError, match=f"{n}: more than 32 bits hold"):
            call()
    assert not library.seen
    ops.residual_norm(far((1 << 31) - 1, 1), far((1 << 31) - 1, 1), far((1 << 31) - 1, 1))
    assert library.seen[0][2] == (1 << 31) - 1


def _calls(**other):
    """The three operators on arrays that fit, but for those named here."""
    f32 = lambda *shape: Fake(*shape, dtype="float32")  # noqa: E731
    i32 = lambda *shape: Fake(*shape, dtype="int32")  # noqa: E731
    a = dict(logits=f32(4, 8), ids=i32(4, 2), weights=f32(4, 2), x=f32(4, 8), gate=f32(8, 16, 8), up=f32(8, 16, 8), down=f32(8, 8, 16), out=f32(4, 8),
             workspace=Fake(100, dtype="uint8"), d=f32(4, 8), x_out=f32(4, 8), h=f32(4, 8), pre=f32(8), post=f32(8), cgate=f32(8))
    a.update(other)
    return dict(route=lambda: ops.route(a["logits"], a["ids"], a["weights"]),
                experts=lambda: ops.experts(a["x"], a["ids"], a["weights"], a["gate"], a["up"], a["down"], a["out"], a["workspace"]),
                residual_norm=lambda: ops.residual_norm(a["x"], a["d"], a["x_out"], a["h"], pre=a["pre"], post=a["post"], gate=a["cgate"]))


def test_arrays_that_fit(library):
    for call in _calls().values():
        call()
    assert [s[0] for s in library.seen] == ["nl_op_route", "nl_op_experts", "nl_op_residual_norm"]


@pytest.mark.parametrize("op, name", [("route", "logits"), ("route", "ids"), ("experts", "x"), ("experts", "ids"), ("experts", "gate"), ("residual_norm", "x")])
@pytest.mark.parametrize("shape", [(), (4,), (4, 2, 2, 2)])
def test_arrays_of_other_dimensions_are_named(library, op, name, shape):
    with pytest.raises(ValueError, match=f"{name}: {len(shape)} dimensions"):
        _calls(**{name: Fake(*shape, dtype="int32" if name == "ids" else "float32")})[op]()
    assert not library.seen


@pytest.mark.parametrize("op, names", [("route", ("logits", "ids", "weights")), ("experts", ("x", "ids", "weights", "gate", "up", "down", "out", "workspace")),
                                       ("residual_norm", ("x", "d", "x_out", "h", "pre", "post", "cgate"))])
def test_arrays_in_host_memory_are_refused(library, op, names):
    """A host array's device has no number: torch's on the CPU."""
    shapes = dict(logits=(4, 8), ids=(4, 2), weights=(4, 2), x=(4, 8), gate=(8, 16, 8), up=(8, 16, 8), down=(8, 8, 16), out=(4, 8), workspace=(100,),
                  d=(4, 8), x_out=(4, 8), h=(4, 8), pre=(8,), post=(8,), cgate=(8,))
    host = {n: Fake(*s, dtype={"ids": "int32", "workspace": "uint8"}.get(n, "float32"), device=None) for n, s in shapes.items()}
    for some in [{n: host[n]} for n in names] + [host]:
        with pytest.raises(ValueError, match="device|host memory"):
            _calls(**some)[op]()
    assert not library.seen
