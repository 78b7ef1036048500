"""The device of an operator's call (`_lib.on_device`, `_lib.ready`), on a fake of two devices: the
tensors' device is current for PyTorch and for the library within the call, and what was current
before is so again after it."""

from __future__ import annotations

import pytest
import torch

from qweninfer_b200 import _lib


class Machine:
    def __init__(self, monkeypatch, count):
        self.current, self.inits = 0, []
        m = self

        class Guard:
            def __init__(self, idx):
                self.idx = idx

            def __enter__(self):
                self.before, m.current = m.current, self.idx

            def __exit__(self, kind, value, trace):
                m.current = self.before

        class Lib:
            def qi_init(self, idx):
                m.inits.append((idx, m.current))
                return 0

        monkeypatch.setattr(torch.cuda, "current_device", lambda: self.current)
        monkeypatch.setattr(torch.cuda, "device", Guard)
        monkeypatch.setattr(torch.cuda, "device_count", lambda: count)
        monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: self.current, raising=False)
        monkeypatch.setattr(_lib, "lib", Lib)
        monkeypatch.setattr(_lib, "_inited", set())
        monkeypatch.setattr(_lib, "_current", [-1])


def test_one_device(monkeypatch):
    m = Machine(monkeypatch, 1)
    assert not _lib.ready(0)
    with _lib.on_device(torch.device("cuda", 0)):
        assert m.current == 0
    assert m.inits == [(0, 0)] and _lib.ready(0)
    with _lib.on_device(torch.device("cuda")):  # the current one
        pass
    assert m.inits == [(0, 0)]  # set up once


def test_another_device_than_the_current_one(monkeypatch):
    m = Machine(monkeypatch, 2)
    for _ in range(2):
        with _lib.on_device(torch.device("cuda", 1)):
            assert m.current == 1 and _lib._current[0] == 1
        assert m.current == 0 and _lib._current[0] == -1  # the library's is to be set again
    assert m.inits == [(1, 1), (1, 1)]  # set for the thread each time
    with _lib.on_device(torch.device("cuda", 0)):
        assert m.current == 0
    assert m.inits[-1] == (0, 0)
    assert not _lib.ready(0) and not _lib.ready(1)  # with several devices no call skips the context


def test_an_exception_restores_the_device(monkeypatch):
    m = Machine(monkeypatch, 2)
    with pytest.raises(KeyError):
        with _lib.on_device(torch.device("cuda", 1)):
            raise KeyError
    assert m.current == 0


def test_other_devices_are_refused(monkeypatch):
    Machine(monkeypatch, 1)
    with pytest.raises(_lib.QiError):
        _lib.on_device(torch.device("cpu"))


def test_a_failed_set_up_restores_the_device(monkeypatch):
    m = Machine(monkeypatch, 2)

    class Lib:
        def qi_init(self, idx):
            return _lib.QI_ERR_DEVICE

    monkeypatch.setattr(_lib, "lib", Lib)
    with pytest.raises(_lib.QiError):
        with _lib.on_device(torch.device("cuda", 1)):
            pass
    assert m.current == 0 and 1 not in _lib._inited
