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
