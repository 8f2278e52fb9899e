"""How a call takes the address of an argument: integers as they are, a buffer of the framework by its ptr, a
tensor by its data_ptr(), of an object that has both the ptr, other numbers as integers."""
import numpy as np
import pytest

from tiny_kernel import ops


class Recorded:
    """Counts the names that were looked for in vain."""

    def __init__(self, **names):
        self.missed = []
        self.__dict__.update(names)

    def __getattr__(self, name):
        self.missed.append(name)
        raise AttributeError(name)


def test_addresses():
    assert ops._ptr(None) is None and ops._ptr(77) == 77 and ops._ptr(np.int64(2**40)) == 2**40
    assert ops._ptr(Recorded(ptr=5)) == 5 and ops._ptr(Recorded(ptr=None)) is None
    assert ops._ptr(Recorded(data_ptr=lambda: 6)) == 6
    assert ops._ptr(Recorded(ptr=5, data_ptr=lambda: 6)) == 5
    with pytest.raises((TypeError, ValueError)):
        ops._ptr("buffer")


def test_a_buffer_is_not_asked_for_what_it_has_not():
    """An AttributeError raised and caught costs seven times the address itself."""
    buffer = Recorded(ptr=5)
    ops._ptr(buffer)
    assert buffer.missed == []


def test_errors_of_an_address_are_not_hidden():
    def data_ptr():
        raise AttributeError("no storage")

    with pytest.raises(AttributeError, match="no storage"):
        ops._ptr(Recorded(data_ptr=data_ptr))
