"""Pointers that no element can lie at are refused in front of the device, by every operator alike."""
import pytest

from test_ops_host import P, close, experts, route


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("call, name, kw", [(route, "logits", {}), (route, "bias", dict(score=1)), (route, "ids", {}), (route, "weights", {}),
                                            (experts, "ids", {}), (experts, "weights", {}),
                                            *[(close, name, {}) for name in ("x", "post", "gate", "pre", "xo")]])
def test_four_byte_arrays_off_their_elements(call, name, kw, off):
    rc, message = call(**{name: P + off}, **kw)
    assert rc == -1 and "boundary of its elements" in message


@pytest.mark.parametrize("dtype, off", [(0, 1), (0, 3), (1, 1), (1, 2), (1, 3)])
@pytest.mark.parametrize("name", ["b", "h"])
def test_rows_of_either_type_off_their_elements(name, dtype, off):
    rc, message = close(dtype=dtype, **{name: P + off})
    assert rc == -1 and "boundary of its elements" in message


def test_arrays_that_are_left_out_are_on_every_boundary():
    for kw in (dict(h=None, pre=None), dict(post=None), dict(gate=None)):
        rc, message = close(dtype=1, b=P + 2, **kw)       # (refused for b alone)
        assert rc == -1 and "boundary of its elements" in message
