"""The binding refuses what its C types cannot hold, instead of passing what is left of it: sizes and leading
dimensions outside 32 bits, type codes, an ignore_index outside 64.  CPU: empty batches with pointers that no call
follows."""
import ctypes
import inspect
import sys

import pytest
import torch

import test_nn_args as A
import vkblas_amd as vk

LIMITS = {ctypes.c_uint32: (0, 2 ** 32 - 1), ctypes.c_int: (-2 ** 31, 2 ** 31 - 1), ctypes.c_int64: (-2 ** 63, 2 ** 63 - 1)}


def arguments(op):
    """The call's whole-number arguments by name, with their C types, from the prototype's order."""
    fn, good = A.CALLS[op]
    names = [n for n in inspect.signature(fn).parameters if n not in ("check", "stream")]
    return [(n, t) for n, t in zip(names, vk._NN_ARGS[op]) if t in LIMITS]


CASES = [(op, name, value) for op in A.CALLS for name, t in arguments(op)
         for value in ([LIMITS[t][0] - 1, LIMITS[t][1] + 1, 2 * (LIMITS[t][1] + 1)] if name != "M" else [2 ** 32, 2 ** 33, -1])]


@pytest.mark.parametrize("op,name,value", CASES, ids=str)
def test_values_outside_their_type_are_refused(op, name, value):
    fn, good = A.CALLS[op]
    args = {**good, "M": 0, name: value}
    assert fn(**args, check=False) == vk.ERR_PARAM
    with pytest.raises(vk.VkblasError) as e:
        fn(**args)
    assert e.value.status == vk.ERR_PARAM


@pytest.mark.parametrize("op", A.CALLS)
def test_by_ctypes_too(op, monkeypatch):
    """... and where the native conversion is not there for this interpreter."""
    fn, good = A.CALLS[op]
    monkeypatch.setattr(vk, "_nn_calls", {})
    monkeypatch.setattr(vk, "_lib", None)
    monkeypatch.setattr(vk, "_range_check", vk._range_check)      # restored with the rest
    monkeypatch.setitem(sys.modules, "vkblas_amd._call", None)
    monkeypatch.delattr(vk, "_call", raising=False)
    for name, value in [(n, v) for o, n, v in CASES if o == op]:
        assert fn(**{**good, "M": 0, name: value}, check=False) == vk.ERR_PARAM
    assert fn(**{**good, "M": 0, **{k: None for k in ("dx", "dw", "db", "dgu") if k in good}}) == vk.OK


def test_rows_too_far_apart_are_copied():
    """torch_nn: a row stride that the library's leading dimensions cannot hold."""
    from vkblas_amd import torch_nn
    wide = torch.empty(2 ** 33 + 64, device="meta")
    for stride in (2 ** 31, 2 ** 32, 2 ** 32 + 16, 2 ** 33):
        m = torch_nn._rows(wide.as_strided((2, 16), (stride, 1)))
        assert torch_nn._ld(m) == 16
    m = torch_nn._rows(wide.as_strided((2, 16), (2 ** 31 - 1, 1)))
    assert torch_nn._ld(m) == 2 ** 31 - 1
