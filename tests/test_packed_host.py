"""Calls with their arguments in one array refuse what the entries themselves refuse (no GPU)."""
import ctypes
import os

import pytest

from alveare_amd import _lib


@pytest.fixture(scope="module")
def L():
    if not os.path.exists(_lib.LIB_PATH):
        from alveare_amd import build

        build.build()
    return _lib.lib()


@pytest.mark.parametrize("name", sorted(_lib.PACKED))
@pytest.mark.parametrize("value", [1.0, "1", None, [1]])
def test_no_integer(L, name, value):
    types = _lib.SIGNATURES[name][1]
    args = [0.0 if t is ctypes.c_float else 0 for t in types]
    at = types.index(ctypes.c_int)
    args[at] = value
    with pytest.raises(ctypes.ArgumentError):
        getattr(L, name)(*args)
    with pytest.raises(ctypes.ArgumentError):
        _lib.call(L, name, *args)


@pytest.mark.parametrize("name", sorted(_lib.PACKED))
@pytest.mark.parametrize("value", ["1", None, [1]])
def test_no_number(L, name, value):
    types = _lib.SIGNATURES[name][1]
    args = [0.0 if t is ctypes.c_float else 0 for t in types]
    args[types.index(ctypes.c_float)] = value
    with pytest.raises(ctypes.ArgumentError):
        getattr(L, name)(*args)
    with pytest.raises(ctypes.ArgumentError):
        _lib.call(L, name, *args)


@pytest.mark.parametrize("value", [2 ** 31, -2 ** 31 - 1, 2 ** 63, 2 ** 70])
def test_past_the_words(L, value):
    """No integer's upper bits are dropped."""
    for name in _lib.PACKED:
        types = _lib.SIGNATURES[name][1]
        args = [0.0 if t is ctypes.c_float else 0 for t in types]
        args[types.index(ctypes.c_int)] = value
        with pytest.raises((ctypes.ArgumentError, _lib.Q4ValueError)):
            _lib.call(L, name, *args)
