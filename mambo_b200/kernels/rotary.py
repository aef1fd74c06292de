"""Rotary positions on sm_100a.

The reference stops at the linears (src/python/mambo/kernels/iq3_s_fp8.py:364-399);
this is what its caller runs on their queries and keys. Pair p of the first
``rotary_dim`` dimensions of a head turns by ``position * frequency[p]``:

    (a, b) -> magnitude * (a cos t - b sin t, a sin t + b cos t)

with (a, b) at dimensions 2p, 2p+1 (interleaved) or p, p + rotary_dim/2
(halves, the default). The other dimensions stay. Frequencies are held as
64-bit fractions of a turn per position, so that the angle is exact modulo a
turn at any position.
"""

from __future__ import annotations

import math
from typing import TypedDict

import torch

from .. import _lib, _runtime
from .fp8_block import _DTYPES, _device_guard

_POSITIONS = {torch.int32: 0, torch.int64: 1}
SCALINGS = (None, "linear", "bands", "yarn")


class RotaryFields(TypedDict):
    turns: torch.Tensor  # int64 [rotary_dim/2]: turns per position, times 2^64, modulo 2^64
    rotary_dim: int
    interleaved: bool
    magnitude: float
    rotary: _lib.MamboRotary  # the C ABI's view of the above


def rotary_frequencies(rotary_dim: int, *, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                       original_length: int = 8192, low: float = 1.0, high: float = 4.0, fast: float = 32.0,
                       slow: float = 1.0) -> tuple[list[float], float]:
    """Radians per position of each pair, base^(-2p/rotary_dim) scaled for a longer context, and the magnitude.

    ``"linear"``: all divided by ``factor``. ``"bands"``: by the turns of a pair
    in the original context: up to ``low`` divided, from ``high`` on kept,
    linear in between. ``"yarn"``: a ramp over the pairs from the one that
    turns ``fast`` times in the original context (kept) to the one that turns
    ``slow`` times (divided), and the magnitude 0.1 ln(factor) + 1.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be an even number of at least 2")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}")
    if not base > 1.0 or not factor > 0.0 or original_length < 1:
        raise ValueError("base must be above 1, factor and original_length positive")
    pairs = rotary_dim // 2
    plain = [base ** (-2.0 * p / rotary_dim) for p in range(pairs)]
    if scaling == "linear":
        return [f / factor for f in plain], 1.0
    if scaling == "bands":
        if not high > low:
            raise ValueError("high must be above low")
        keep = [min(1.0, max(0.0, (original_length * f / (2.0 * math.pi) - low) / (high - low))) for f in plain]
        return [f / factor * (1.0 - k) + f * k for f, k in zip(plain, keep)], 1.0
    if scaling == "yarn":
        def pair_of(turns: float) -> float:
            return rotary_dim * math.log(original_length / (2.0 * math.pi * turns)) / (2.0 * math.log(base))

        first, last = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), rotary_dim - 1)
        divide = [min(1.0, max(0.0, (p - first) / max(last - first, 0.001))) for p in range(pairs)]
        return [f / factor * d + f * (1.0 - d) for f, d in zip(plain, divide)], 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    return plain, 1.0


@_runtime.with_stream
def prepare_rotary_fields(rotary_dim: int, *, base: float = 10000.0, interleaved: bool = False, scaling: str | None = None,
                          factor: float = 1.0, original_length: int = 8192, low: float = 1.0, high: float = 4.0,
                          fast: float = 32.0, slow: float = 1.0, frequencies=None, magnitude: float | None = None,
                          device="cuda", stream=None) -> RotaryFields:
    """The rotation's fields on ``device``, from ``rotary_frequencies``' arguments or the given ``frequencies``.

    ``frequencies``: rotary_dim/2 radians per position (any sequence of
    numbers). ``magnitude``: of the rotated values, in place of the scaling's.
    """
    if frequencies is None:
        radians, scaled = rotary_frequencies(rotary_dim, base=base, scaling=scaling, factor=factor,
                                             original_length=original_length, low=low, high=high, fast=fast, slow=slow)
    else:
        radians, scaled = [float(f) for f in frequencies], 1.0
        if rotary_dim < 2 or rotary_dim % 2 or len(radians) != rotary_dim // 2:
            raise ValueError("frequencies must be rotary_dim / 2 numbers")
        if not all(math.isfinite(f) for f in radians):
            raise ValueError("frequencies must be finite")
    magnitude = scaled if magnitude is None else float(magnitude)
    turns = [round(math.fmod(f / (2.0 * math.pi), 1.0) * 2.0 ** 64) % (1 << 64) for f in radians]
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError("expected a CUDA device (this build has no CPU path)")
    held = torch.tensor([t - (1 << 64) if t >= 1 << 63 else t for t in turns], dtype=torch.int64, device=device)
    _runtime.require_device(held.device)
    return {"turns": held, "rotary_dim": rotary_dim, "interleaved": bool(interleaved), "magnitude": magnitude,
            "rotary": _lib.MamboRotary(held.data_ptr(), rotary_dim, int(bool(interleaved)), magnitude)}


def _check_rope(rope: RotaryFields, dim: int, device: torch.device) -> None:
    if not isinstance(rope, dict) or "rotary" not in rope or "turns" not in rope:
        raise TypeError("rope must come from prepare_rotary_fields")
    if rope["rotary"].turns != rope["turns"].data_ptr():  # a copy of the fields: the kernels would read the first one's table
        raise ValueError("rope's tensors were replaced: call prepare_rotary_fields again")
    if rope["rotary_dim"] > dim:
        raise ValueError("the rotated part is larger than the head")
    if rope["turns"].get_device() != device.index:
        raise ValueError("rope and values must be on one device")


def _head_strides(t: torch.Tensor) -> tuple[int, int]:
    """Strides of a token and of a head of [T,H,D] (one that is alone has no stride that matters)."""
    (tokens, heads, dim), (st, sh, _) = t.shape, t.stride()
    sh = sh if heads > 1 else dim
    return st if tokens > 1 else heads * dim, sh


@_runtime.with_stream
def launch_rotary(x, positions, rope: RotaryFields, *, inverse: bool = False, stream=None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """x [T,H,D] (float32 or bfloat16) with each token's heads turned by ``positions`` [T] (int32 or int64).

    The rotation is computed in float32 and rounded once to x's type. ``out``:
    of x's shape and type; x itself turns in place. ``inverse`` turns back,
    which is also the gradient of the rotation.
    """
    x, positions = _runtime.as_cuda_tensor(x), _runtime.as_cuda_tensor(positions)
    dev = x.device
    if x.ndim != 3 or x.dtype not in _DTYPES or x.shape[1] < 1:
        raise ValueError("x must be float32 or bfloat16 [T,H,D]")
    tokens, heads, dim = x.shape
    if positions.dtype not in _POSITIONS or positions.shape != (tokens,) or positions.get_device() != dev.index:
        raise ValueError("positions must be int32 or int64 [T] on x's device")
    _check_rope(rope, dim, dev)
    _runtime.require_device(dev)
    if x.stride(2) != 1:
        if out is x:
            raise ValueError("x must have unit stride along the head to turn in place")
        x = x.contiguous()
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    elif tuple(out.shape) != (tokens, heads, dim) or out.dtype != x.dtype or out.stride(2) != 1 or out.device != dev:
        raise ValueError("out must have x's shape, type and device and unit stride along the head")
    if tokens:
        if positions.stride(0) != 1 and tokens > 1:
            positions = positions.contiguous()
        with _device_guard(dev):
            st = _runtime.stream_handle(None, dev)
            _lib.check(_lib.load().mambo_rotary(
                x.data_ptr(), _DTYPES[x.dtype], tokens, heads, dim, *_head_strides(x), positions.data_ptr(),
                _POSITIONS[positions.dtype], rope["rotary"], int(inverse), out.data_ptr(), *_head_strides(out), st),
                "launch_rotary")
    return out
