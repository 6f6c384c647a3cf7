"""perf/operators.py: the framework's calls go to the current device and stream
(CPU only, with stand-ins for both)."""
import importlib
import types

import pytest


class Handle:
    def __init__(self, device):
        self.device, self.stream = device, None

    def set_stream(self, stream):
        self.stream = stream


@pytest.fixture
def ops(monkeypatch):
    import torch

    module = importlib.import_module("perf.operators")
    at = types.SimpleNamespace(device=0, stream=0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: at.device)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: types.SimpleNamespace(cuda_stream=at.stream))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: at.stream, raising=False)
    monkeypatch.setattr(module, "_kept", {})
    monkeypatch.setitem(__import__("sys").modules, "b2blas", types.SimpleNamespace(Handle=Handle))
    return module, at


def test_calls_follow_the_current_stream_and_device(ops):
    module, at = ops
    first = module._handle()[1]
    assert (first.device, first.stream) == (0, 0)
    for stream in (77, 0, 77, 78):
        at.stream = stream
        assert module._handle()[1] is first and first.stream == stream
    at.device, at.stream = 1, 5
    second = module._handle()[1]
    assert second is not first and (second.device, second.stream) == (1, 5) and first.stream == 78
    at.device, at.stream = 0, 9
    assert module._handle()[1] is first and first.stream == 9 and second.stream == 5
