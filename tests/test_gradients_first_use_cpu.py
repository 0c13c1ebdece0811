"""The gradients' calls are made once, whichever threads come first: without a GPU, by stand-ins for the extension
and the kernels that take their time."""
import threading
import time
import types

import pytest

from neptune_codegen import gradients as GR


class Calls:
    made = []

    def __init__(self, *sizes):
        self.devices = set()
        Calls.made.append(self)

    def has(self, device):
        return device in self.devices

    def add(self, device, kernels):
        assert len(kernels) == len(GR._KERNELS)
        self.devices.add(device)


class Program:
    def kernel(self, name, args, block, device):
        time.sleep(0.002)                            # (another thread's turn)
        return types.SimpleNamespace(handle=1)


def extension():
    time.sleep(0.02)
    return types.SimpleNamespace(GradientCalls=Calls)


@pytest.mark.parametrize("devices", [(0, 0), (0, 0, 0, 0, None, None), (0, 1, 0, 1)])
def test_threads_that_come_first_share_one_object(monkeypatch, devices):
    monkeypatch.setattr(Calls, "made", [])
    monkeypatch.setattr(GR, "_CALLS", None)
    monkeypatch.setattr(GR, "_program", Program)
    monkeypatch.setattr(GR.dispatch, "extension", extension)
    start, got = threading.Barrier(len(devices)), []

    def first(device):
        start.wait()
        calls = GR._calls(device)
        got.append((calls, device is None or calls.has(device)))

    threads = [threading.Thread(target=first, args=(d,)) for d in devices]
    for t in threads:
        t.start()
    for t in threads:
        t.join(30)
    assert len(got) == len(devices) and len(Calls.made) == 1
    assert all(calls is Calls.made[0] and known for calls, known in got)
