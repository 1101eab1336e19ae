"""Edges of the paged-cache operators' calls that need no GPU."""
import contextlib
import ctypes

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


@pytest.mark.parametrize("scale,code", [(2.3e38, 0), (2.4e38, -5), (3.3e38, -5)])
def test_scales_that_the_kernels_base_takes_beyond_fp32_are_refused(scale, code):
    """The kernels work with scale * log2(e) in fp32, which has to be finite.  A taken scale is told by its workspace."""
    from qmtp import _lib

    ptr = 1 << 20
    c = _lib.PagedCacheArgs(k=ptr, v=ptr, table=ptr, lens=ptr, pages=4000, ld_table=1000, n_kv=2, page=16, Dh=128, table_w=1000, B=2)
    a = _lib.PagedArgs(q=ptr, gate=None, out=ptr, q_ld=0, gate_ld=0, gate_hs=0, T=4, n_q=4, scale=scale, window=0, sinks=0)
    L = _lib.lib()
    assert (L.qmtp_paged_attention_workspace(ctypes.byref(a), ctypes.byref(c)) > 0) == (code == 0)
    if code:
        assert L.qmtp_paged_attention(ctypes.byref(a), ctypes.byref(c), ptr, 1 << 40, None) == code
        assert L.qmtp_paged_prompt(ctypes.byref(a), ptr, ctypes.byref(c), ptr, 1 << 40, None) == code
