"""Two threads that need a stream's workspace at the same time end up with one, and the shortcut module
knows that one: an address that it kept of the other would be memory that has been freed."""
import contextlib

import torch

import streamk_b200  # noqa: F401
from streamk_b200 import ops

DEVICE = torch.device("cuda", 0)


class Shortcut:
    def __init__(self):
        self.known = {}

    def set_workspace(self, device, stream, ptr, nbytes):
        self.known[device, stream] = ptr


def test_one_workspace_for_both(monkeypatch):
    shortcut, made = Shortcut(), []

    class Workspace:                                  # the second thread runs while the first makes its own
        nbytes = 1

        def __init__(self, device, stream):
            self.ptr = 1000 + len(made)
            made.append(self)
            if len(made) == 1:
                second.append(ops._workspace(DEVICE))
    second = []
    monkeypatch.setattr(ops, "_Workspace", Workspace)
    monkeypatch.setattr(ops, "_workspaces", {})
    monkeypatch.setattr(ops, "_fast", shortcut)
    monkeypatch.setattr(ops, "_stream_ptr", lambda device: 7)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    first = ops._workspace(DEVICE)
    assert len(made) == 2 and first is second[0] is ops._workspaces[0, 7]
    assert shortcut.known == {(0, 7): first.ptr}
