"""How the Python view takes addresses: what it accepts, and that a host array, of
which the layer's forward passes four, gets there without an exception."""
import sys

import numpy as np
import pytest

import qauntrunner_b200 as Q

torch = pytest.importorskip("torch")


def raised(f, *a):
    """(f's result, exceptions raised on the way in Python code, caught ones too)."""
    seen = []

    def trace(frame, event, arg):
        if event == "exception":
            seen.append(arg[0])
        return trace

    before = sys.gettrace()
    sys.settrace(trace)
    try:
        return f(*a), seen
    finally:
        sys.settrace(before)


def test_host_arrays_raise_nothing():
    for a in (np.zeros((3, 4), np.float32), np.zeros(5, np.int32)[1:], np.arange(6, dtype=np.uint8)):
        at, seen = raised(Q._ptr, a)
        assert at == a.__array_interface__["data"][0] and not seen


def test_what_else_has_an_address(tmp_path):
    t = torch.zeros(4)
    assert raised(Q._ptr, t) == (t.data_ptr(), [])
    assert Q._ptr(None) is None and Q._ptr(4096) == 4096
    m = np.memmap(tmp_path / "m", np.uint8, "w+", shape=(16,))   # a subclass of NumPy's array
    assert Q._ptr(m) == m.__array_interface__["data"][0]
    with pytest.raises(AttributeError):
        Q._ptr("no array")
