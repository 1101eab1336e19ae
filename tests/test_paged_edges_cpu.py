"""Edges of the paged-cache operators' calls that need no GPU."""
import contextlib

import pytest
import torch


@pytest.mark.parametrize("current", [0, 1])
def test_the_tensors_device_is_current_for_the_workspace_and_the_launch(current, monkeypatch):
    """Both go by the device: the workspace's size by its SMs, the launch by its kernels and stream."""
    from qmtp import paged

    state = {"current": current, "calls": []}

    @contextlib.contextmanager
    def device(index):
        held, state["current"] = state["current"], index
        yield
        state["current"] = held

    monkeypatch.setattr(torch.cuda, "current_device", lambda: state["current"])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)

    class Cache:
        _index = 1

    def workspace(a, c):
        state["calls"].append(("workspace", state["current"], a, c))
        return 64

    def fn(a, c, ws, n, stream):
        state["calls"].append(("launch", state["current"], a, c, n, stream))
        return 0

    paged._launch(Cache, "attention", fn, workspace, "a", "c", torch.empty(1))
    assert state["calls"] == [("workspace", 1, "a", "c"), ("launch", 1, "a", "c", 64, 101)]
    assert state["current"] == current
