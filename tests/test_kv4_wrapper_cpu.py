"""The wrapper around the q4_0 cache's calls without a GPU: where workspaces come from, which tensors are refused."""
import contextlib
from types import SimpleNamespace

import pytest

import tsrc


class _FakeTorch:
    """As much of torch as a workspace takes, noting the stream that is current at an allocation."""
    uint8 = "uint8"

    def __init__(self):
        self.now, self.made = "current", []
        self.cuda = SimpleNamespace(stream=self._stream, ExternalStream=lambda handle, device=None: ("external", handle, device))

    @contextlib.contextmanager
    def _stream(self, s):
        was, self.now = self.now, s
        yield
        self.now = was

    def empty(self, n, dtype, device):
        self.made.append((n, device, self.now))
        return SimpleNamespace(data_ptr=lambda: 4096, numel=lambda: n, element_size=lambda: 1, record_stream=lambda s: None)


@pytest.mark.parametrize("stream,want", [(None, "current"), ("side", "side"), (77, ("external", 77, "cuda:0")), (0, ("external", 0, "cuda:0"))])
def test_workspace_comes_from_the_calls_own_stream(monkeypatch, stream, want):
    """A block that the current stream still works on may be handed out again to that stream alone."""
    fake = _FakeTorch()
    monkeypatch.setattr(tsrc, "_torch", fake)
    tsrc._workspace(SimpleNamespace(device="cuda:0"), 512, None, stream)
    assert fake.made == [(512, "cuda:0", want)] and fake.now == "current"
