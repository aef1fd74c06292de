"""Device plumbing shared by the operators: tensors, streams, device checks, workspaces.

PyTorch provides device memory and streams; the compute is in libmambo_b200.
"""

from __future__ import annotations

import functools
import threading

import torch

from . import _lib

_checked_devices: dict[int, int] = {}
_workspaces: dict[tuple[int, int], "_Workspace"] = {}
_kept: list[torch.Tensor] = []  # buffers that a CUDA graph may use and a larger one has replaced


def as_cuda_tensor(obj) -> torch.Tensor:
    """Zero-copy view of a CUDA array (torch, DLPack or __cuda_array_interface__ object)."""
    if isinstance(obj, torch.Tensor):
        t = obj
    elif hasattr(obj, "__dlpack__"):
        t = torch.from_dlpack(obj)
    elif hasattr(obj, "__cuda_array_interface__"):
        t = torch.as_tensor(obj, device="cuda")
    else:
        raise TypeError(f"expected a CUDA tensor, got {type(obj).__name__}")
    if not t.is_cuda:
        raise ValueError("expected a CUDA tensor (this build has no CPU path)")
    return t


def stream_handle(stream, device: torch.device) -> int:
    """cudaStream_t of `stream` (None = torch's current stream on `device`)."""
    if stream is None:  # without building a torch.cuda.Stream, which takes 2 us
        return torch._C._cuda_getCurrentRawStream(device.index if device.index is not None else torch.cuda.current_device())
    if isinstance(stream, torch.cuda.Stream):
        return stream.cuda_stream
    if isinstance(stream, int):
        return stream
    for attr in ("cuda_stream", "ptr", "handle"):
        if hasattr(stream, attr):
            return int(getattr(stream, attr))
    raise TypeError(f"unsupported stream object {type(stream).__name__}")


def _parts(obj):
    """What a container of tensors holds: a list, tuple, dict or dataclass (prepared weights, routes)."""
    if isinstance(obj, (list, tuple)):
        return obj
    if isinstance(obj, dict):
        return obj.values()
    if hasattr(obj, "__dataclass_fields__"):
        return [getattr(obj, name) for name in obj.__dataclass_fields__]
    return ()


def _device_of(parts) -> torch.device | None:
    for v in parts:
        if isinstance(v, torch.Tensor):
            if v.is_cuda:
                return v.device
        elif (device := _device_of(_parts(v))) is not None:
            return device
    return None


def _record_use(parts, stream: torch.cuda.Stream) -> None:
    """The allocator keeps the tensors' memory until what is queued on ``stream`` now is done."""
    for v in parts:
        if isinstance(v, torch.Tensor):
            if v.is_cuda:
                v.record_stream(stream)
        elif v is not None and not isinstance(v, (int, str)):
            _record_use(_parts(v), stream)


@functools.lru_cache(maxsize=256)
def _external_stream(handle: int, device: torch.device) -> torch.cuda.Stream:
    if handle in (0, 1):  # the legacy default stream by either of its names
        return torch.cuda.default_stream(device)
    return torch.cuda.ExternalStream(handle, device=device)


def with_stream(operator):
    """Runs an operator with its ``stream=`` (a torch stream or any handle) as the current one.

    So what it allocates, copies (rows without unit stride) and fills belongs to
    the stream that its kernels run on. The caller orders that stream with the
    work that made the arguments, and his own with the results. Either may be
    dropped at any time: memory is not used again before both streams are done
    with it.
    """

    @functools.wraps(operator)
    def call(*args, stream=None, **kwargs):
        if stream is None:
            return operator(*args, **kwargs)
        device = _device_of(args) or _device_of(kwargs.values()) or torch.device("cuda", torch.cuda.current_device())
        handle, here = stream_handle(stream, device), torch._C._cuda_getCurrentRawStream(device.index)
        if handle == here or (handle == 1 and here == 0):
            return operator(*args, **kwargs)
        target = stream if isinstance(stream, torch.cuda.Stream) else _external_stream(handle, device)
        current_device, caller = torch.cuda.current_device(), torch.cuda.current_stream(device)
        torch.cuda.set_stream(target)
        try:
            result = operator(*args, **kwargs)
        finally:
            torch.cuda.set_stream(caller)
            if current_device != device.index:
                torch.cuda.set_device(current_device)
        _record_use(args, target)
        _record_use(kwargs.values(), target)
        _record_use((result,), caller)
        return result

    return call


def require_device(device: torch.device) -> None:
    """Raise RuntimeError unless `device` is an sm_100 GPU this library runs on."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    status = _checked_devices.get(index)
    if status is None:
        lib = _lib.load()
        with torch.cuda.device(index):
            status = lib.mambo_device_check()
        _checked_devices[index] = status
    if status != _lib.MAMBO_OK:
        major, minor = torch.cuda.get_device_capability(index)
        raise RuntimeError(f"IQ3_S FP8 kernels have no build for sm{major}{minor} (this library targets sm_100a)")


def _stream_is_capturing(device: torch.device, stream: int) -> bool:
    with torch.cuda.stream(_external_stream(stream, device)):
        return torch.cuda.is_current_stream_capturing()


class _Workspace:
    """The scratch buffer of ``stream``, at ``ptr`` with ``size`` bytes; while it is entered, the calling thread's."""

    __slots__ = ("stream", "lock", "buffer", "ptr", "size", "captured")

    def __init__(self, stream: int):
        self.stream = stream
        self.lock = threading.Lock()
        self.buffer: torch.Tensor | None = None
        self.ptr = self.size = 0
        self.captured = False  # a CUDA graph may use the buffer

    def __enter__(self) -> "_Workspace":
        return self

    def __exit__(self, *exc) -> None:
        self.lock.release()

    def grow(self, device: torch.device, nbytes: int) -> None:
        size = max(nbytes, 1 << 20, 2 * self.size)
        # Drain pending work before swapping buffers: a kernel on the stream
        # may still use the old one, and the zero-fill runs on torch's stream.
        torch.cuda.synchronize(device)
        new = torch.zeros(size, dtype=torch.uint8, device=device)
        torch.cuda.synchronize(device)
        if self.captured:
            _kept.append(self.buffer)
        self.buffer, self.ptr, self.size, self.captured = new, new.data_ptr(), size, False


def workspace(device: torch.device, stream: int | None, nbytes: int) -> _Workspace:
    """Zero-filled scratch for split-K partials and counters, one buffer per (device, stream), to be used as

        with workspace(device, stream, nbytes) as ws:
            ...  # the C call that gets ws.ptr, ws.size and ws.stream

    ``stream`` None: the current stream of ``device``, which is the current device.
    The kernels leave the counter region zeroed again, so the buffer is reused
    across calls on the same stream; calls on different streams get their own.
    A call may be several launches that hand data on through the buffer, so
    another host thread's call on the stream waits here until they are queued.

    A CUDA graph keeps the address of the buffer that its calls were captured
    with. So a buffer that was handed out during a capture is never freed, also
    when a later call on the stream needs a larger one; each is at least twice
    the one before, so what is kept adds up to less than the newest. A capture
    itself cannot make the buffer grow (it could neither be zero-filled at once
    nor outlive the graph): that raises, and the capture goes on undisturbed.
    """
    if stream is None:
        index = device.index
        stream, here = torch._C._cuda_getCurrentRawStream(index), True
    else:
        current = torch.cuda.current_device()
        index = device.index if device.index is not None else current
        here = index == current and stream == torch._C._cuda_getCurrentRawStream(index)
    ws = _workspaces.get((index, stream))
    if ws is None:
        ws = _workspaces.setdefault((index, stream), _Workspace(stream))
    # Only the current stream's capture is a cheap question: any other stream counts as capturing.
    captured = not here or torch._C._cuda_isCurrentStreamCapturing()
    ws.lock.acquire()
    try:
        if ws.size < nbytes:
            dev = torch.device("cuda", index)
            if captured and _stream_is_capturing(dev, stream):
                raise RuntimeError(f"the stream's workspace has {ws.size} bytes and this call needs {nbytes}: run it once on "
                                   "the stream before capturing it")
            ws.grow(dev, nbytes)
        if captured:
            ws.captured = True
    except BaseException:
        ws.lock.release()
        raise
    return ws


def zero_workspaces() -> None:
    """Zero-fill the current device's workspaces, those that only CUDA graphs use among them; nothing may be running there."""
    index = torch.cuda.current_device()
    for (device, _), ws in list(_workspaces.items()):
        if device == index:
            with ws.lock:
                if ws.buffer is not None:
                    ws.buffer.zero_()
    for buffer in _kept:
        if buffer.device.index in (index, None):
            buffer.zero_()
    torch.cuda.synchronize(index)
