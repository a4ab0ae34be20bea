"""How the wrappers of the paged serving step reach the library, without a GPU: a stand-in for torch's devices and streams
records where a call is launched."""

import contextlib
import types

import pytest

from rosylnalive_b200 import native as N
from rosylnalive_b200 import ops as O


class Devices:
    """torch, as far as a launch uses it, with device `current` current."""

    def __init__(self, current):
        self.current, self.entered = current, []
        self._C = types.SimpleNamespace(_cuda_getDevice=lambda: self.current,
                                        _cuda_getCurrentRawStream=lambda dev: 1000 + dev)
        self.cuda = types.SimpleNamespace(device=self.device, current_stream=self.current_stream)

    @contextlib.contextmanager
    def device(self, dev):
        before, self.current = self.current, dev
        self.entered.append(dev)
        try:
            yield
        finally:
            self.current = before

    def current_stream(self, dev):
        return types.SimpleNamespace(cuda_stream=1000 + dev)


@pytest.mark.parametrize("current,dev", [(0, 0), (0, 3), (3, 0)])
@pytest.mark.parametrize("stream", [None, 77])
def test_a_call_runs_on_its_tensors_device_and_leaves_the_current_one(monkeypatch, current, dev, stream):
    torch = Devices(current)
    monkeypatch.setattr(O, "_torch", torch)
    calls = []

    def launch(s, desc):
        calls.append((s, desc, torch.current))
        return N.LRM_OK

    given = None if stream is None else types.SimpleNamespace(cuda_stream=stream)
    O._launch("call", launch, b"descriptor", dev, given)
    assert calls == [(1000 + dev if stream is None else stream, b"descriptor", dev)]
    assert torch.current == current and torch.entered == ([] if dev == current else [dev])


@pytest.mark.parametrize("current,dev", [(0, 0), (0, 3)])
def test_a_refused_call_raises_and_leaves_the_current_device(monkeypatch, current, dev):
    torch = Devices(current)
    monkeypatch.setattr(O, "_torch", torch)
    with pytest.raises(ValueError, match="call"):
        O._launch("call", lambda s, desc: N.LRM_ERR_ARGUMENT, b"", dev, None)
    assert torch.current == current


def test_the_workspace_of_a_machine_without_a_device_is_that_of_a_b200():
    rows, heads = 5, 16  # 148 SMs, two partial results each: 128 + 2 floats a row, and a record of 16 bytes
    assert O.paged_attention_workspace(rows, heads, 8) == 148 * (2 * rows * 2 * 130 * 4 + 16)
