"""Operators given a ``stream=`` that is not the current one: copies, results and memory let go of early.

The streams are kept busy with a spin of some 30 ms, so that what is queued on one of them has not run when the other
goes on. Only values are wrong where an order is missing.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mambo_b200 import _lib
from mambo_b200.kernels.fp8_block import fp8_block_grouped_linear, fp8_block_linear, launch_fp8_block_matmul, \
    launch_quantize_fp8_block, prepare_fp8_block_fields
from mambo_b200.kernels.moe_fp8 import fp8_moe_experts, launch_moe_combine, launch_moe_route
from test_fp8_block_gpu import make_weight, make_x

pytestmark = pytest.mark.gpu

M, N, K, E = 40, 384, 512, 4


def busy():
    torch.cuda._sleep(60_000_000)


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    torch.cuda.synchronize()
    assert _lib.device_status()[0] == 0


@pytest.fixture(scope="module")
def operators(cuda_device):
    """name -> (call(x, stream), its input's shape): each takes x with any strides."""
    dev = cuda_device

    def weight(n, k, seed, experts=None, **kw):
        codes, scales = make_weight(n, k, seed, experts=experts)
        return prepare_fp8_block_fields(torch.from_numpy(codes).to(dev), torch.from_numpy(scales).to(dev) * 2.0 ** -5, **kw)

    w, grouped = weight(N, K, 1), weight(N, K, 2, E)
    gate_up, down = weight(256, K, 3, E, gate_up=True), weight(K, 128, 4, E)
    offsets = torch.tensor([0, 7, 7, 30, M], dtype=torch.int32, device=dev)
    route = launch_moe_route(torch.randn(M, E, generator=torch.Generator().manual_seed(0)).to(dev), 2)
    ops = {
        "linear": lambda x, s: fp8_block_linear(x, w, stream=s),
        "grouped": lambda x, s: fp8_block_grouped_linear(x, offsets, grouped, stream=s),
        "quantize": lambda x, s: launch_quantize_fp8_block(x, stream=s),
        "route": lambda x, s: [launch_moe_route(x, 3, stream=s)[n] for n in ("ids", "weights", "positions", "offsets", "rows")],
        "combine": lambda x, s: launch_moe_combine(x, route, stream=s),
        "experts": lambda x, s: fp8_moe_experts(x, route, gate_up, down, stream=s),
    }
    torch.cuda.synchronize()
    return ops


NAMES = ["linear", "grouped", "quantize", "route", "combine", "experts"]


def tensors(result):
    return list(result) if isinstance(result, (tuple, list)) else [result]


def equal(a, b):
    return all(torch.equal(s, t) for s, t in zip(tensors(a), tensors(b)))


def strided(seed, rows=M):
    """x [rows, K] without unit column stride, and the same contiguous."""
    x = make_x(rows, K, seed).cuda()
    return x.t().contiguous().t(), x


def fill_freed_memory(nbytes):
    return [torch.full((nbytes,), 0x5A, dtype=torch.uint8, device="cuda") for _ in range(4)]


@pytest.mark.parametrize("handle", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_strided_input_while_the_current_stream_is_busy(operators, name, handle):
    """The copy of a strided input is made on the stream that reads it."""
    x, plain = strided(1, 2 * M if name == "combine" else M)
    ref = operators[name](plain, None)
    side = torch.cuda.Stream()
    operators[name](strided(7, x.shape[0])[0], side)  # workspace, kernels, and other values in what the copy takes up
    torch.cuda.synchronize()
    busy()
    out = operators[name](x, side.cuda_stream if handle else side)
    side.synchronize()
    with torch.cuda.stream(side):
        assert equal(out, ref)


@pytest.mark.parametrize("name", NAMES)
def test_strided_input_while_the_other_stream_is_busy(operators, name):
    """Neither the copy nor the input goes back to the current stream before the other has read it."""
    rows = 2 * M if name == "combine" else M
    x, plain = strided(2, rows)
    ref = operators[name](plain, None)
    side = torch.cuda.Stream()
    operators[name](x, side)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        busy()
    out = operators[name](x, side)
    del x
    junk = fill_freed_memory(rows * K * 4)
    torch.cuda.synchronize()
    assert equal(out, ref) and len(junk) == 4


@pytest.mark.parametrize("name", NAMES)
def test_results_do_not_overwrite_memory_in_use(operators, name):
    """A result does not take memory that the current stream has let go of but still reads."""
    x, plain = strided(3, 2 * M if name == "combine" else M)
    side = torch.cuda.Stream()
    ref = operators[name](plain, None)
    operators[name](x, side)
    torch.cuda.synchronize()
    old = [torch.full_like(t, 3) for t in tensors(ref) for _ in range(2)]
    torch.cuda.synchronize()
    busy()
    copies = [t.clone() for t in old]
    del old
    out = operators[name](x, side)
    torch.cuda.synchronize()
    assert all(bool((c == 3).all()) for c in copies)
    assert equal(out, ref)


@pytest.mark.parametrize("name", NAMES)
def test_results_let_go_of_while_still_read(operators, name):
    """A result's memory is not the other stream's again before the caller's stream has read it."""
    x, plain = strided(4, 2 * M if name == "combine" else M)
    side = torch.cuda.Stream()
    ref = operators[name](plain, None)
    operators[name](x, side)
    torch.cuda.synchronize()
    out = operators[name](x, side)
    torch.cuda.current_stream().wait_stream(side)
    busy()
    copies = [t.clone() for t in tensors(out)]
    del out
    with torch.cuda.stream(side):
        junk = fill_freed_memory(sum(t.numel() * t.element_size() for t in copies)) + [torch.zeros_like(t) for t in copies]
    torch.cuda.synchronize()
    assert equal(copies, tensors(ref)) and junk


def test_strided_codes(cuda_device):
    """launch_fp8_block_matmul's values and scales, both strided."""
    dev = cuda_device
    codes, scales = make_weight(N, K, 1)
    w = prepare_fp8_block_fields(torch.from_numpy(codes).to(dev), torch.from_numpy(scales).to(dev))
    v, s = launch_quantize_fp8_block(make_x(M, K, 6).to(dev), group=32)
    ref = launch_fp8_block_matmul(v, s, w)
    vt, st = v.t().contiguous().t(), s.t().contiguous().t()
    side = torch.cuda.Stream()
    launch_fp8_block_matmul(vt, st, w, stream=side)
    torch.cuda.synchronize()
    busy()
    out = launch_fp8_block_matmul(vt, st, w, stream=side)
    side.synchronize()
    assert np.array_equal(out.cpu().numpy(), ref.cpu().numpy())


def test_empty_results_on_another_stream(cuda_device):
    """Zeros that no kernel writes come from the given stream too."""
    route = launch_moe_route(torch.randn(3, E, device=cuda_device), 2)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    busy()
    empty = launch_moe_route(torch.empty(0, E, device=cuda_device), 2, stream=side)
    out = launch_moe_combine(torch.empty(0, 64, device=cuda_device), route, stream=side, out_dtype=torch.float32)
    side.synchronize()
    with torch.cuda.stream(side):
        assert bool((empty["offsets"] == 0).all()) and bool((out == 0).all())


@pytest.mark.parametrize("handle", [0, 1, 2])
def test_the_default_streams_handles(operators, handle):
    """The legacy default stream as 0 and 1, the per-thread one as 2, from the current stream and from another."""
    x = make_x(M, K, 9).cuda()
    ref = operators["linear"](x, None)
    torch.cuda.synchronize()
    out = operators["linear"](x, handle)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = operators["linear"](x, handle)
        assert torch.cuda.current_stream() == side
    torch.cuda.synchronize()
    assert torch.equal(out, ref) and torch.equal(other, ref)


def test_a_refused_call_leaves_the_current_stream(operators):
    side = torch.cuda.Stream()
    before = torch.cuda.current_stream()
    with pytest.raises(ValueError):
        operators["linear"](torch.zeros(3, K + 1, device="cuda"), side)
    assert torch.cuda.current_stream() == before
