"""vkblas_amd._call hands the functions of vkblas_nn.h the same values as their ctypes prototypes do, at and past
the ends of each type, and declines (None) what it does not convert itself."""
import ctypes

import pytest

import vkblas_amd as vk

vk.load()
NAMES = sorted(vk._NN_ARGS)


def receiver(name):
    got = []
    cb = ctypes.CFUNCTYPE(ctypes.c_int, *vk._NN_ARGS[name])(lambda *a: got.append(a) or -7)
    return cb, ctypes.cast(cb, ctypes.c_void_p).value, got


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("value", [0, 1, 2**31 - 1, 2**31, 2**32 + 5, -1, -2**31, 2**63 - 1, 2**64 - 1])
def test_same_values_as_ctypes(name, value):
    native = vk._nn_calls[name][0]
    cb, addr, got = receiver(name)
    for number in (1.5, -0.0, 1e-60, 3, float("inf")):
        # every argument another value, so that none can take another's place
        args = [number if t is ctypes.c_float else value + 3 * i if t is not ctypes.c_void_p or i % 3 else None
                for i, t in enumerate(vk._NN_ARGS[name])]
        assert native(addr, *args) == -7
        assert cb(*args) == -7
        assert got[-1] == got[-2]


@pytest.mark.parametrize("name", NAMES)
def test_declines_what_ctypes_converts_itself(name):
    native = vk._nn_calls[name][0]
    _, addr, got = receiver(name)
    good = [1.0 if t is ctypes.c_float else 64 for t in vk._NN_ARGS[name]]
    for i, t in enumerate(vk._NN_ARGS[name]):
        for bad in (True, "1", b"x", ctypes.c_void_p(64), 4.0 if t is not ctypes.c_float else 10**400):
            assert native(addr, *good[:i], bad, *good[i + 1:]) is None
    assert got == []
    with pytest.raises(TypeError):
        native(addr, *good[:-1])
    with pytest.raises(ValueError):
        native(0, *good)
