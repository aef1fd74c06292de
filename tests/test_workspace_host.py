"""CPU: the life of the per-stream workspaces, with torch's device calls replaced by host ones."""

from __future__ import annotations

import gc
import weakref

import pytest
import torch

from mambo_b200 import _runtime

DEV = torch.device("cuda", 0)


@pytest.fixture
def device(monkeypatch):
    """A device of host memory; its ``capturing`` says whether the current stream (handle 7) is being captured."""
    class Device:
        capturing = False

    real_zeros, state = torch.zeros, Device()
    monkeypatch.setattr(torch, "zeros", lambda n, dtype, device: real_zeros(n, dtype=dtype))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state.capturing)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 7, raising=False)
    monkeypatch.setattr(_runtime, "_stream_is_capturing", lambda device, stream: state.capturing, raising=False)
    for name in ("_workspaces", "_captured", "_kept"):
        if hasattr(_runtime, name):
            monkeypatch.setattr(_runtime, name, type(getattr(_runtime, name))())
    return state


def handed_out(stream, nbytes):
    """A weak reference to the buffer a call gets, and its size."""
    ws = _runtime.workspace(DEV, stream, nbytes)
    return weakref.ref(ws), ws.numel()


def alive(ref) -> bool:
    gc.collect()
    return ref() is not None


def test_a_captured_buffer_outlives_its_replacement(device):
    first, size = handed_out(7, 1 << 20)
    device.capturing = True
    same, _ = handed_out(7, 1 << 20)
    device.capturing = False
    assert same() is first()
    second, grown = handed_out(7, 3 << 20)
    assert second() is not first() and grown >= 2 * size
    assert alive(first)
    # Handed out again only after the replacement: not captured, so it may go.
    handed_out(7, grown + 1)
    assert alive(first) and not alive(second)


def test_an_uncaptured_buffer_is_freed(device):
    first, size = handed_out(7, 1 << 20)
    handed_out(7, size + 1)
    assert not alive(first)


def test_another_stream_than_the_current_counts_as_captured(device):
    first, size = handed_out(9, 1 << 20)
    handed_out(9, size + 1)
    assert alive(first)


def test_a_capture_does_not_grow_a_buffer(device):
    device.capturing = True
    with pytest.raises(RuntimeError, match="before capturing"):
        handed_out(7, 1 << 20)
    device.capturing = False
    first, size = handed_out(7, 1 << 20)
    device.capturing = True
    with pytest.raises(RuntimeError, match="before capturing"):
        handed_out(7, size + 1)
    # What the call before it got is still the stream's.
    assert handed_out(7, size)[0]() is first()
