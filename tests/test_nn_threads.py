"""The operators' first calls from several threads at once: none finds the binding's table half built."""
import ctypes
import threading

import pytest

import test_nn_args as A
import vkblas_amd as vk


@pytest.mark.parametrize("at", range(1, 8))
def test_first_calls_of_two_threads(monkeypatch, at):
    """The first thread's load() is held at its `at`-th address while another makes its first calls."""
    monkeypatch.setattr(vk, "_nn_calls", {})
    monkeypatch.setattr(vk, "_lib", None)
    cast, seen, casts = ctypes.cast, [], []

    def other():
        try:
            for op in reversed(list(A.CALLS)):
                fn, good = A.CALLS[op]
                seen.append(fn(**{**good, "dtype": 99}, check=False))
        except Exception as e:       # noqa: BLE001
            seen.append(e)

    def slow(*args):
        casts.append(args)
        if len(casts) == at:
            t = threading.Thread(target=other)
            t.start()
            t.join(30)
        return cast(*args)
    monkeypatch.setattr(vk.ctypes, "cast", slow)
    fn, good = A.CALLS["layer_norm"]
    assert fn(**{**good, "dtype": 99}, check=False) == vk.ERR_PARAM
    assert seen and set(seen) == {vk.ERR_PARAM}
