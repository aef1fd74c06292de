"""FP8 block-scaled linear on the sm_100a tcgen05 tensor cores, plain and grouped by expert.

Weights are E4M3 with one float32 scale per 128 x 128 block (checkpoints that
are published in FP8); the reference has no such type, its linears take GGUF
blocks (src/python/mambo/kernels/iq3_s_fp8.py:364-399). The interface is that
of the framework's other linears: weights prepared once on the device,
activations quantized to E4M3 with power-of-two scales, one call.

    out[m, n] = sum_b sw[n // 128, b] * sum_{k in block b} xq[m, k] * 2^e(m, k // group) * wq[n, k]

``group`` is 128 (one activation scale per weight block) or 32 (MXFP8, the
scales launch_quantize_fp8 writes). e is ceil(log2(amax / 448)), clamped to
[-127, 127], 0 for amax == 0, and values round to nearest even. Any N, K and M
of at least 1.
"""

from __future__ import annotations

import functools
from typing import TypedDict

import torch

from .. import _lib, _runtime

BLOCK = 128
GROUPS = (32, 128)


class Fp8BlockFields(TypedDict):
    packed: torch.Tensor  # uint8, mambo_fp8b_packed_bytes(E, N, K) bytes (tile-major records)
    scales: torch.Tensor  # float32, the block scales in the order of the records
    n_rows: int
    k: int
    n_experts: int  # 1 for a weight given as [N,K]
    gate_up: bool
    weight: _lib.MamboFp8BlockWeight  # the C ABI's view of the above


def _device_guard(device: torch.device):
    """torch.cuda.device, or nothing when the device is current already."""
    if device.index == torch._C._cuda_getDevice():
        return _NO_GUARD
    return torch.cuda.device(device)


class _NoGuard:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_NO_GUARD = _NoGuard()


_DTYPES = {torch.float32: _lib.MAMBO_F32, torch.bfloat16: _lib.MAMBO_BF16}


def _out_code(dtype: torch.dtype) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError("out_dtype must be torch.float32 or torch.bfloat16")
    return code


def _check_group(group: int) -> None:
    if group not in GROUPS:
        raise ValueError("activation scales are per 32 or per 128 values")


@_runtime.with_stream
def prepare_fp8_block_fields(values, scales, *, gate_up: bool = False, stream=None) -> Fp8BlockFields:
    """E4M3 weights [N,K] or [E,N,K] and their float32 block scales -> the packed copy the kernels stream.

    ``values``: uint8 or float8_e4m3fn, any strides. ``scales``: float32
    [ceil(N/128), ceil(K/128)] (with the leading E of the values). With
    ``gate_up`` the rows are a gate projection followed by an up projection,
    each with its own row blocks of scales (2 * ceil(N/2/128) scale rows), and
    the result is for ``fp8_moe_experts``.
    """
    values, scales = _runtime.as_cuda_tensor(values), _runtime.as_cuda_tensor(scales)
    if values.dtype == torch.float8_e4m3fn:
        values = values.view(torch.uint8)
    if values.dtype != torch.uint8 or values.ndim not in (2, 3) or min(values.shape) < 1:
        raise ValueError("FP8 weight must be uint8 or float8_e4m3fn [N,K] or [E,N,K]")
    if scales.dtype != torch.float32 or scales.ndim != values.ndim:
        raise ValueError("FP8 block scales must be float32 with as many dimensions as the weight")
    if values.ndim == 2:
        values, scales = values[None], scales[None]
    experts, n, k = values.shape
    if gate_up and n % 2:
        raise ValueError("a gate/up weight has an even number of rows")
    row_blocks = 2 * -(-(n // 2) // BLOCK) if gate_up else -(-n // BLOCK)
    if tuple(scales.shape) != (experts, row_blocks, -(-k // BLOCK)):
        raise ValueError(f"FP8 block scales must be [{experts}, {row_blocks}, {-(-k // BLOCK)}], got {list(scales.shape)}")
    if experts > _lib.MAMBO_MOE_MAX_EXPERTS:
        raise ValueError(f"a weight has at most {_lib.MAMBO_MOE_MAX_EXPERTS} experts")
    if scales.device != values.device:
        raise ValueError("the weight and its scales must be on one device")
    dev = values.device
    _runtime.require_device(dev)
    lib = _lib.load()
    packed = torch.empty(lib.mambo_fp8b_packed_bytes(experts, n, k, int(gate_up)), dtype=torch.uint8, device=dev)
    out_scales = torch.empty(lib.mambo_fp8b_scales_bytes(experts, n, k, int(gate_up)) // 4, dtype=torch.float32,
                             device=dev)
    with _device_guard(dev):
        st = _runtime.stream_handle(None, dev)
        _lib.check(lib.mambo_fp8b_pack(
            values.data_ptr(), experts, n, k, values.stride(0), values.stride(1), values.stride(2), scales.data_ptr(),
            scales.stride(0), scales.stride(1), scales.stride(2), int(gate_up), packed.data_ptr(),
            out_scales.data_ptr(), st), "prepare_fp8_block_fields")
    weight = _lib.MamboFp8BlockWeight(packed.data_ptr(), out_scales.data_ptr(), n, k, experts, int(gate_up))
    return {"packed": packed, "scales": out_scales, "n_rows": n, "k": k, "n_experts": experts,
            "gate_up": bool(gate_up), "weight": weight}


@_runtime.with_stream
def launch_quantize_fp8_block(x, *, group: int = BLOCK, stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Return [M,K] E4M3 bytes and [M,ceil(K/group)] UE8M0 scale bytes of x (float32 or bfloat16 [M,K], any K)."""
    x = _runtime.as_cuda_tensor(x)
    _check_group(group)
    if x.ndim != 2 or x.dtype not in _DTYPES or x.shape[1] < 1:
        raise ValueError("activation must be float32 or bfloat16 [M,K]")
    _runtime.require_device(x.device)
    if x.stride(1) != 1:
        x = x.contiguous()
    m, k = x.shape
    values = torch.empty((m, k), dtype=torch.uint8, device=x.device)
    scales = torch.empty((m, -(-k // group)), dtype=torch.uint8, device=x.device)
    if m:
        with _device_guard(x.device):
            st = _runtime.stream_handle(None, x.device)
            _lib.check(_lib.load().mambo_fp8b_quantize(
                x.data_ptr(), _DTYPES[x.dtype], m, k, _row_stride(x), group, values.data_ptr(), k, scales.data_ptr(),
                scales.shape[1], st), "launch_quantize_fp8_block")
    return values, scales


def _row_stride(t: torch.Tensor) -> int:
    """Row stride of a [M,K] tensor with unit column stride (a single row's is its length)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


@functools.lru_cache(maxsize=1024)
def _linear_workspace_bytes(rows: int, experts: int, n: int, k: int) -> int:
    return _lib.load().mambo_fp8b_linear_workspace_bytes(rows, experts, n, k)


def _output(out, rows: int, n: int, out_dtype: torch.dtype, device: torch.device) -> tuple[torch.Tensor, int]:
    """The output [rows, n], the given one or a new one, and its row stride."""
    if out is None:
        _out_code(out_dtype)
        return torch.empty((rows, n), dtype=out_dtype, device=device), n
    if tuple(out.shape) != (rows, n) or out.dtype not in _DTYPES or (n > 1 and out.stride(1) != 1) \
            or out.device != device:
        raise ValueError("out must be float32 or bfloat16 [M,N] with unit column stride on the activation's device")
    return out, _row_stride(out)


def _check_weight(weight: Fp8BlockFields, device: torch.device, grouped: bool) -> None:
    if not isinstance(weight, dict) or "weight" not in weight:
        raise TypeError("weight must come from prepare_fp8_block_fields")
    if weight["gate_up"]:
        raise ValueError("a gate/up weight is for fp8_moe_experts")
    if not grouped and weight["n_experts"] != 1:
        raise ValueError("a weight of several experts needs fp8_block_grouped_linear")
    if weight["packed"].device != device:
        raise ValueError("weight and activation must be on one device")


@_runtime.with_stream
def launch_fp8_block_matmul(x_values, x_scales, weight: Fp8BlockFields, *, stream=None,
                            out_dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None) -> torch.Tensor:
    """Quantized activations times a prepared weight -> out [M,N].

    ``x_values`` uint8 [M,K]; ``x_scales`` uint8 [M,ceil(K/128)] or
    [M,ceil(K/32)] (launch_quantize_fp8_block, launch_quantize_fp8); for K up
    to 32, where both are one column, it is one scale for the row either way.
    """
    x_values, x_scales = _runtime.as_cuda_tensor(x_values), _runtime.as_cuda_tensor(x_scales)
    dev = x_values.device
    _check_weight(weight, dev, False)
    k = weight["k"]
    if x_values.ndim != 2 or x_values.dtype != torch.uint8 or x_values.shape[1] != k:
        raise ValueError("x_values must be uint8 [M,K]")
    m = x_values.shape[0]
    group = {(m, -(-k // 128)): 128, (m, -(-k // 32)): 32}.get(tuple(x_scales.shape))
    if group is None or x_scales.dtype != torch.uint8 or x_scales.device != dev:
        raise ValueError("x_scales must be uint8 [M,ceil(K/128)] or [M,ceil(K/32)]")
    _runtime.require_device(dev)
    if x_values.stride(1) != 1:
        x_values = x_values.contiguous()
    if x_scales.stride(1) != 1:
        x_scales = x_scales.contiguous()
    out, ldo = _output(out, m, weight["n_rows"], out_dtype, dev)
    if m:
        with _device_guard(dev):
            with _runtime.workspace(dev, None, _linear_workspace_bytes(m, 1, weight["n_rows"], k)) as ws:
                _lib.check(_lib.load().mambo_fp8b_linear(
                    x_values.data_ptr(), _row_stride(x_values), x_scales.data_ptr(), _row_stride(x_scales), group, m,
                    weight["weight"], out.data_ptr(), _DTYPES[out.dtype], ldo, ws.ptr, ws.size, ws.stream),
                    "launch_fp8_block_matmul")
    return out


def _activation(x, weight: Fp8BlockFields, act_group: int, grouped: bool) -> tuple[torch.Tensor, torch.device, int, int]:
    """x [M,K] with unit column stride, its device, M and row stride."""
    x = _runtime.as_cuda_tensor(x)
    dev = x.device
    _check_group(act_group)
    _check_weight(weight, dev, grouped)
    if x.ndim != 2 or x.dtype not in _DTYPES or x.shape[1] != weight["k"]:
        raise ValueError("activation must be float32 or bfloat16 [M,K] with the weight's K")
    _runtime.require_device(dev)
    m, (ldx, unit) = x.shape[0], x.stride()
    if unit != 1:
        x = x.contiguous()
        ldx = weight["k"]
    return x, dev, m, ldx if m > 1 else weight["k"]


@_runtime.with_stream
def fp8_block_linear(x, weight: Fp8BlockFields, *, act_group: int = BLOCK, stream=None,
                     out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """bf16/f32 activations [M,K] -> E4M3 with one scale per ``act_group`` values -> the linear, one C-ABI call."""
    x, dev, m, ldx = _activation(x, weight, act_group, False)
    n = weight["n_rows"]
    out, ldo = _output(out, m, n, out_dtype, dev)
    if m:
        with _device_guard(dev):
            with _runtime.workspace(dev, None, _linear_workspace_bytes(m, 1, n, weight["k"])) as ws:
                _lib.check(_lib.load().mambo_fp8b_linear_fused(
                    x.data_ptr(), _DTYPES[x.dtype], ldx, act_group, m, weight["weight"], out.data_ptr(), _DTYPES[out.dtype],
                    ldo, ws.ptr, ws.size, ws.stream), "fp8_block_linear")
    return out


@_runtime.with_stream
def fp8_block_grouped_linear(x, offsets, weight: Fp8BlockFields, *, act_group: int = BLOCK, stream=None,
                             out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rows offsets[e] .. offsets[e+1]-1 of x [R,K] times expert e's weight, for every expert in one call.

    ``offsets``: int32 [E+1] on the device (launch_moe_route's), 0 first, then
    non-decreasing up to R; it is not read on the host. Segments may be empty;
    output rows that no segment covers are not written.
    """
    x, dev, rows, ldx = _activation(x, weight, act_group, True)
    offsets = _runtime.as_cuda_tensor(offsets)
    n, experts = weight["n_rows"], weight["n_experts"]
    if offsets.dtype != torch.int32 or tuple(offsets.shape) != (experts + 1,) or offsets.device != dev:
        raise ValueError("offsets must be int32 [E+1] on the activation's device")
    if offsets.stride(0) != 1:
        offsets = offsets.contiguous()
    out, ldo = _output(out, rows, n, out_dtype, dev)
    if rows:
        with _device_guard(dev):
            with _runtime.workspace(dev, None, _linear_workspace_bytes(rows, experts, n, weight["k"])) as ws:
                _lib.check(_lib.load().mambo_fp8b_grouped_linear(
                    x.data_ptr(), _DTYPES[x.dtype], ldx, act_group, rows, offsets.data_ptr(), weight["weight"],
                    out.data_ptr(), _DTYPES[out.dtype], ldo, ws.ptr, ws.size, ws.stream),
                    "fp8_block_grouped_linear")
    return out
