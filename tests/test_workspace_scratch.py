"""Which workspace a call gets, on the CPU: torch.cuda is replaced by a machine of two devices, one of whose streams is captured."""
import contextlib
from types import SimpleNamespace

import pytest
import torch

from llm_inference_optimization_b200 import _workspace


@pytest.fixture
def machine(monkeypatch):
    m = SimpleNamespace(current=0, capturing=set())

    @contextlib.contextmanager
    def device(index):
        before, m.current = m.current, index
        yield
        m.current = before

    monkeypatch.setattr(torch.cuda, "current_device", lambda: m.current)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: m.current in m.capturing)
    monkeypatch.setattr(_workspace, "_cache", {})
    real = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **k: real(*a, **k))
    monkeypatch.setattr(_workspace, "get", lambda kind, n, device: _workspace._cache.setdefault((kind, device.index, 7), torch.zeros(n, dtype=torch.uint8)))
    return m


@pytest.mark.parametrize("current", [0, 1])
@pytest.mark.parametrize("index", [0, 1])
def test_a_captured_call_has_its_own(machine, current, index):
    """Whichever device is current, it is the call's own device whose stream decides."""
    machine.current, dev = current, torch.device("cuda", index)
    eager = _workspace.scratch("x", 100, 8, dev, 7)
    assert _workspace.scratch("x", 100, 8, dev, 7) is eager
    machine.capturing = {1 - index}
    assert _workspace.scratch("x", 100, 8, dev, 7) is eager
    machine.capturing = {index}
    a, b = (_workspace.scratch("x", 100, 8, dev, 7) for _ in range(2))
    assert a is not eager and b is not eager and a is not b and not a[:8].any()
    assert machine.current == current and list(_workspace._cache.values()) == [eager]
