"""Routed experts on FP8 block-scaled weights: router, expert products, weighted sum.

The reference has no mixture-of-experts path; this one stands beside its
linears (src/python/mambo/kernels/iq3_s_fp8.py:364-399) and uses the same
activation format between them (MXFP8, quantize_fp8.py:23-52). A layer is

    route = launch_moe_route(logits, top_k)
    out = fp8_moe_experts(x, route, gate_up, down)

with ``gate_up`` and ``down`` from ``prepare_fp8_block_fields``. Nothing is
read back to the host in between. The parts also stand alone: rows sorted by
``route["rows"]`` through ``fp8_block_grouped_linear``, then
``launch_moe_combine``.
"""

from __future__ import annotations

import functools
from typing import TypedDict

import torch

from .. import _lib, _runtime
from .fp8_block import _DTYPES, Fp8BlockFields, _device_guard, _output, _row_stride

_SCORING = {"softmax": _lib.MAMBO_MOE_SOFTMAX, "sigmoid": _lib.MAMBO_MOE_SIGMOID}


class MoeRoute(TypedDict):
    ids: torch.Tensor  # int32 [T,top]: experts of each token, highest score first; -1: none left
    weights: torch.Tensor  # float32 [T,top]
    offsets: torch.Tensor  # int32 [E+1]: first row of each expert in expert order
    positions: torch.Tensor  # int32 [T,top]: row of each choice in expert order, -1: none
    rows: torch.Tensor  # int32 [T*top]: the choice (token * top + j) of each row, -1 past the last
    made: tuple  # the tensors above as launch_moe_route made them: calls that get these very ones skip their checks


@functools.lru_cache(maxsize=1024)
def _route_workspace_bytes(tokens: int, experts: int) -> int:
    return _lib.load().mambo_moe_route_workspace_bytes(tokens, experts)


@functools.lru_cache(maxsize=1024)
def _experts_workspace_bytes(tokens: int, top: int, experts: int, h: int, i: int, out: int) -> int:
    return _lib.load().mambo_moe_experts_workspace_bytes(tokens, top, experts, h, i, out)


@_runtime.with_stream
def launch_moe_route(logits, top_k: int, *, scoring: str = "softmax", bias=None, renormalize: bool = True,
                     scale: float = 1.0, stream=None) -> MoeRoute:
    """The ``top_k`` experts of each token of logits [T,E] (float32 or bfloat16) and the order of their rows.

    ``scoring="softmax"``: weights softmax(logits), selection by logit;
    ``"sigmoid"``: weights sigmoid(logits), selection by them. ``bias``
    (float32 [E]) is added to the selection score only. Highest first, equal
    scores to the lower expert. With ``renormalize`` a token's weights are
    divided by their sum; then all are multiplied by ``scale``. Logits of -inf
    or NaN mask an expert for the token; with fewer than ``top_k`` left the
    rest gets id -1, weight 0 and position -1.
    """
    logits = _runtime.as_cuda_tensor(logits)
    if logits.ndim != 2 or logits.dtype not in _DTYPES or logits.shape[1] < 1:
        raise ValueError("logits must be float32 or bfloat16 [T,E]")
    if scoring not in _SCORING:
        raise ValueError(f"scoring must be one of {sorted(_SCORING)}")
    tokens, experts = logits.shape
    if experts > _lib.MAMBO_MOE_MAX_EXPERTS:
        raise ValueError(f"at most {_lib.MAMBO_MOE_MAX_EXPERTS} experts")
    if not 1 <= top_k <= min(experts, _lib.MAMBO_MOE_MAX_TOP):
        raise ValueError(f"top_k must be in [1, min({_lib.MAMBO_MOE_MAX_TOP}, E)]")
    dev = logits.device
    if bias is not None:
        bias = _runtime.as_cuda_tensor(bias)
        if bias.dtype != torch.float32 or tuple(bias.shape) != (experts,) or bias.device != dev:
            raise ValueError("bias must be float32 [E] on the logits' device")
        bias = bias if bias.stride(0) == 1 else bias.contiguous()
    _runtime.require_device(dev)
    if logits.stride(1) != 1 and experts > 1:
        logits = logits.contiguous()
    # One allocation: the four integer outputs and the float weights between them.
    n = tokens * top_k
    buf = torch.empty(4 * n + experts + 1, dtype=torch.int32, device=dev)
    shape, strides = (tokens, top_k), (top_k, 1)
    ids, positions = buf.as_strided(shape, strides, 0), buf.as_strided(shape, strides, n)
    weights = buf.view(torch.float32).as_strided(shape, strides, 2 * n)
    rows, offsets = buf.as_strided((n,), (1,), 3 * n), buf.as_strided((experts + 1,), (1,), 4 * n)
    if tokens:
        with _device_guard(dev):
            with _runtime.workspace(dev, None, _route_workspace_bytes(tokens, experts)) as ws:
                _lib.check(_lib.load().mambo_moe_route(
                    logits.data_ptr(), _DTYPES[logits.dtype], logits.stride(0) if tokens > 1 else experts,
                    0 if bias is None else bias.data_ptr(),
                    tokens, experts, top_k, _SCORING[scoring], int(renormalize), scale, ids.data_ptr(),
                    weights.data_ptr(), offsets.data_ptr(), positions.data_ptr(), rows.data_ptr(), ws.ptr,
                    ws.size, ws.stream), "launch_moe_route")
    else:
        offsets.zero_()
    return {"ids": ids, "weights": weights, "offsets": offsets, "positions": positions, "rows": rows,
            "made": (ids, weights, positions, rows, offsets)}


def _check_route(route: MoeRoute, tokens: int, device: torch.device) -> int:
    """top_k of a route for `tokens` tokens."""
    ids, weights, positions, rows = route["ids"], route["weights"], route["positions"], route["rows"]
    made = route.get("made")
    if made and made[0] is ids and made[1] is weights and made[2] is positions and made[3] is rows \
            and made[4] is route["offsets"] and ids.shape[0] == tokens and ids.device == device:
        return ids.shape[1]
    if ids.ndim != 2 or ids.shape[0] != tokens or weights.shape != ids.shape or positions.shape != ids.shape:
        raise ValueError("route must have ids, weights and positions [T,top_k] for the activation's T")
    if ids.dtype != torch.int32 or positions.dtype != torch.int32 or weights.dtype != torch.float32 \
            or route["offsets"].dtype != torch.int32 or rows.dtype != torch.int32 or rows.numel() != ids.numel():
        raise ValueError("route must have int32 ids, positions, rows and offsets and float32 weights")
    if not (ids.is_contiguous() and rows.is_contiguous() and weights.is_contiguous() and positions.is_contiguous()
            and route["offsets"].is_contiguous()):
        raise ValueError("route tensors must be contiguous")
    if ids.device != device or rows.device != device or weights.device != device or positions.device != device \
            or route["offsets"].device != device:
        raise ValueError("route and activation must be on one device")
    return ids.shape[1]


@_runtime.with_stream
def launch_moe_combine(y, route: MoeRoute, *, stream=None, out_dtype: torch.dtype = torch.bfloat16,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = sum_j weights[t,j] * y[positions[t,j]] for expert rows y [R,H] in expert order, summed in float32."""
    y = _runtime.as_cuda_tensor(y)
    if y.ndim != 2 or y.dtype not in _DTYPES or y.shape[1] < 1:
        raise ValueError("y must be float32 or bfloat16 [R,H]")
    tokens, dev = route["ids"].shape[0], y.device
    top = _check_route(route, tokens, dev)
    _runtime.require_device(dev)
    if y.stride(1) != 1:
        y = y.contiguous()
    rows, h = y.shape
    out, ldo = _output(out, tokens, h, out_dtype, dev)
    if tokens and not rows:
        out.zero_()
    elif tokens:
        with _device_guard(dev):
            st = _runtime.stream_handle(None, dev)
            _lib.check(_lib.load().mambo_moe_combine(
                y.data_ptr(), _DTYPES[y.dtype], _row_stride(y), rows, route["positions"].data_ptr(),
                route["weights"].data_ptr(), tokens, top, h, out.data_ptr(), _DTYPES[out.dtype], ldo, st),
                "launch_moe_combine")
    return out


@_runtime.with_stream
def fp8_moe_experts(x, route: MoeRoute, gate_up: Fp8BlockFields, down: Fp8BlockFields, *, stream=None,
                    out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """A layer of routed experts, x [T,H] -> out [T,H], in one C-ABI call.

    x is quantized to MXFP8, each chosen expert computes silu(gate) * up
    (quantized again from float32) and its down projection, and a token's rows
    are summed with the route's weights. ``gate_up``: [E, 2I, H] prepared with
    ``gate_up=True``; ``down``: [E, H, I]. Each expert row rounds once to
    ``out_dtype`` before the sum, which is in float32: a bfloat16 result has
    two roundings. For one only, ask for float32 and round the result; that
    keeps the rows in float32 (8 % more time for a prompt).
    """
    x = _runtime.as_cuda_tensor(x)
    for w in (gate_up, down):
        if not isinstance(w, dict) or "weight" not in w:
            raise TypeError("weights must come from prepare_fp8_block_fields")
    if not gate_up["gate_up"] or down["gate_up"]:
        raise ValueError("gate_up must be prepared with gate_up=True and down without")
    h, i, experts, dev = gate_up["k"], gate_up["n_rows"] // 2, gate_up["n_experts"], x.device
    if down["n_experts"] != experts or down["n_rows"] != h or down["k"] != i:
        raise ValueError("down must be [E, H, I] to the gate/up weight's [E, 2I, H]")
    if x.ndim != 2 or x.dtype not in _DTYPES or x.shape[1] != h:
        raise ValueError("activation must be float32 or bfloat16 [T,H]")
    if gate_up["packed"].device != dev or down["packed"].device != dev:
        raise ValueError("weights and activation must be on one device")
    tokens = x.shape[0]
    top = _check_route(route, tokens, dev)
    if tuple(route["offsets"].shape) != (experts + 1,):
        raise ValueError("route and weights must have the same number of experts")
    _runtime.require_device(dev)
    if x.stride(1) != 1:
        x = x.contiguous()
    out, ldo = _output(out, tokens, h, out_dtype, dev)
    if tokens:
        code = _DTYPES[out.dtype]
        with _device_guard(dev):
            with _runtime.workspace(dev, None, _experts_workspace_bytes(tokens, top, experts, h, i, code)) as ws:
                _lib.check(_lib.load().mambo_moe_experts(
                    x.data_ptr(), _DTYPES[x.dtype], x.stride(0) if tokens > 1 else h, tokens, route["ids"].data_ptr(),
                    route["weights"].data_ptr(), route["positions"].data_ptr(), route["offsets"].data_ptr(),
                    route["rows"].data_ptr(), top, gate_up["weight"], down["weight"], out.data_ptr(), code,
                    ldo, ws.ptr, ws.size, ws.stream), "fp8_moe_experts")
    return out
