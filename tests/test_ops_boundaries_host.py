"""Pointers that no element can lie at are refused in front of the device."""
import pytest

from test_ops_host import P, experts


@pytest.mark.parametrize("dtype, off", [(0, 1), (1, 1), (1, 2), (1, 3)])
@pytest.mark.parametrize("name", ["x", "gate", "up", "down", "y"])
def test_arrays_off_their_elements(dtype, off, name):
    rc, message = experts(dtype=dtype, **{name: P + off})
    assert rc == -1 and "boundary of its elements" in message
