"""CPU: the life of the per-stream workspaces, with torch's device calls replaced by host ones."""

from __future__ import annotations

import gc
import threading
import time
import weakref

import pytest
import torch

from mambo_b200 import _lib, _runtime
from mambo_b200.kernels import fp8_block, moe_fp8

DEV = torch.device("cuda", 0)


@pytest.fixture
def device(monkeypatch):
    """A device of host memory; its ``capturing`` says whether the current stream (handle 7) is being captured."""
    class Device:
        capturing = False

    real_zeros, state = torch.zeros, Device()
    monkeypatch.setattr(torch, "zeros", lambda *shape, dtype=None, device=None: real_zeros(*shape, dtype=dtype))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: state.capturing, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 7, raising=False)
    monkeypatch.setattr(_runtime, "_stream_is_capturing", lambda device, stream: state.capturing, raising=False)
    for name in ("_workspaces", "_kept"):
        monkeypatch.setattr(_runtime, name, type(getattr(_runtime, name))())
    return state


def handed_out(stream, nbytes):
    """A weak reference to the buffer a call gets, and its size."""
    with _runtime.workspace(DEV, stream, nbytes) as ws:
        return weakref.ref(ws.buffer), ws.size


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


class FakeLibrary:
    """Stands for the C library: says which calls are inside it at once, per workspace."""

    def __init__(self):
        self.inside, self.most, self.calls = {}, 0, 0
        self.guard = threading.Lock()

    def __getattr__(self, name):
        if name.endswith("_bytes"):
            return lambda *a: 1 << 20

        def call(*args):
            ws = args[-3]  # the workspace's address, its size, the stream
            with self.guard:
                self.calls += 1
                self.inside[ws] = self.inside.get(ws, 0) + 1
                self.most = max(self.most, self.inside[ws])
            time.sleep(0.01)  # as a C call does, this lets the other threads run
            with self.guard:
                self.inside[ws] -= 1
            return _lib.MAMBO_OK

        return call


@pytest.mark.parametrize("op", ["linear", "grouped", "matmul", "route", "experts"])
def test_calls_of_several_threads_on_a_stream_take_turns(device, monkeypatch, op):
    """A call's launches hand data on through the workspace: another thread's must not come between them."""
    lib = FakeLibrary()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_runtime, "as_cuda_tensor", lambda t: t)
    monkeypatch.setattr(_runtime, "require_device", lambda dev: None)
    for module in (fp8_block, moe_fp8):
        monkeypatch.setattr(module, "_device_guard", lambda dev: fp8_block._NO_GUARD)
    for f in (fp8_block._linear_workspace_bytes, moe_fp8._route_workspace_bytes, moe_fp8._experts_workspace_bytes):
        f.cache_clear()  # the sizes here are not the library's
    packed = torch.zeros(1)

    def weight(n, k, experts, gate_up=False):
        return {"packed": packed, "scales": packed, "n_rows": n, "k": k, "n_experts": experts, "gate_up": gate_up,
                "weight": None}

    x = torch.zeros(4, 8)
    offsets = torch.zeros(3, dtype=torch.int32)
    route = {"ids": torch.zeros(4, 1, dtype=torch.int32), "weights": torch.zeros(4, 1), "offsets": offsets,
             "positions": torch.zeros(4, 1, dtype=torch.int32), "rows": torch.zeros(4, dtype=torch.int32)}
    call = {
        "linear": lambda: fp8_block.fp8_block_linear(x, weight(8, 8, 1)),
        "grouped": lambda: fp8_block.fp8_block_grouped_linear(x, offsets, weight(8, 8, 2)),
        "matmul": lambda: fp8_block.launch_fp8_block_matmul(x.byte(), torch.zeros(4, 1, dtype=torch.uint8), weight(8, 8, 1)),
        "route": lambda: moe_fp8.launch_moe_route(torch.zeros(4, 8), 2),
        "experts": lambda: moe_fp8.fp8_moe_experts(x, route, weight(16, 8, 2, True), weight(8, 8, 2)),
    }[op]
    failures = []

    def many():
        try:
            for _ in range(3):
                call()
        except Exception as e:  # noqa: BLE001
            failures.append(e)

    threads = [threading.Thread(target=many) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=30)
    for f in (fp8_block._linear_workspace_bytes, moe_fp8._route_workspace_bytes, moe_fp8._experts_workspace_bytes):
        f.cache_clear()
    assert not failures and lib.calls == 12
    assert lib.most == 1


def test_a_failed_call_gives_the_workspace_back(device):
    with pytest.raises(ValueError):
        with _runtime.workspace(DEV, 7, 1):
            raise ValueError
    device.capturing = True
    with pytest.raises(RuntimeError):
        _runtime.workspace(DEV, 7, 1 << 30)
    device.capturing = False
    done = []
    t = threading.Thread(target=lambda: done.append(handed_out(7, 1)), daemon=True)
    t.start()
    t.join(timeout=10)
    assert done


def test_a_reset_after_a_failure_zeroes_the_workspaces(device, monkeypatch):
    """Counters that a call left behind when it gave up would keep later calls from summing their parts."""
    class Status:
        code = 0

        def mambo_device_status(self, reset, code, where, block):
            code._obj.value = self.code
            return _lib.MAMBO_OK

    lib = Status()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    first, size = handed_out(7, 1)
    device.capturing = True
    handed_out(7, 1)
    device.capturing = False
    handed_out(7, size + 1)  # the first one stays with the graph
    buffers = [first(), _runtime.workspace(DEV, 9, 1), _runtime.workspace(DEV, 7, 1)]
    for b in buffers[1:]:
        b.lock.release()
    buffers = [buffers[0], buffers[1].buffer, buffers[2].buffer]
    for code, reset, left in ((_lib.MAMBO_ETIMEOUT, True, 0), (_lib.MAMBO_ETIMEOUT, False, 1), (0, True, 1)):
        for b in buffers:
            b.fill_(1)
        lib.code = code
        assert _lib.device_status(reset=reset)[0] == code
        assert all(bool((b == left).all()) for b in buffers)
