"""The per-stream workspaces on the GPU: graphs captured before a larger one replaces them, and host threads that share one."""

from __future__ import annotations

import threading

import pytest
import torch

from mambo_b200 import _lib, _runtime
from mambo_b200.kernels.fp8_block import fp8_block_linear, prepare_fp8_block_fields
from mambo_b200.kernels.moe_fp8 import fp8_moe_experts, launch_moe_route
from test_fp8_block_gpu import make_weight

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _fresh_workspaces(monkeypatch):
    """Streams come from a pool: without this, an earlier test's large buffer may already be there."""
    monkeypatch.setattr(_runtime, "_workspaces", {})
    yield
    torch.cuda.synchronize()
    assert _lib.device_status()[0] == 0


def workspace_bytes(stream) -> int:
    """The size of the stream's buffer once a call that needs next to nothing has got it."""
    with _runtime.workspace(torch.device("cuda", 0), stream.cuda_stream, 1) as ws:
        return ws.size


def prepared(dev, n, k, seed, experts=None, **kw):
    codes, scales = make_weight(n, k, seed, experts=experts)
    scales *= 2.0 ** -4
    return prepare_fp8_block_fields(torch.from_numpy(codes).to(dev), torch.from_numpy(scales).to(dev), **kw)


def capture(stream, call):
    with torch.cuda.stream(stream):
        call()  # the workspace exists before the capture
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = call()
    return graph, out


@pytest.mark.parametrize("op", ["linear", "experts"])
def test_graphs_of_a_growing_batch(cuda_device, op):
    """Graphs of 1, 8 and 700 tokens captured one after the other on one stream, then replayed among other tensors."""
    dev = cuda_device
    if op == "linear":
        h, w = 1024, prepared(dev, 768, 1024, 3)
        call = lambda x, logits: fp8_block_linear(x, w)  # noqa: E731
    else:
        h, gate_up, down = 512, prepared(dev, 512, 512, 4, experts=8, gate_up=True), prepared(dev, 512, 256, 5, experts=8)
        call = lambda x, logits: fp8_moe_experts(x, launch_moe_route(logits, 3), gate_up, down)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, sizes = [], []
    for m in (1, 8, 700):
        x, logits = torch.zeros(m, h, device=dev, dtype=torch.bfloat16), torch.zeros(m, 8, device=dev)
        graphs.append((x, logits, *capture(side, lambda: call(x, logits))))  # noqa: B023
        with torch.cuda.stream(side):
            sizes.append(workspace_bytes(side))
    torch.cuda.synchronize()
    assert sizes[0] < sizes[2], "the workspace was meant to grow"
    # Whatever memory was given back is somebody else's now.
    others = [torch.full((1 << 20,), i, dtype=torch.int32, device=dev) for i in range(1, 33)]
    for seed in range(2):
        gen = torch.Generator().manual_seed(seed)
        for x, logits, graph, out in graphs:
            x.copy_(torch.randn(x.shape, generator=gen))
            logits.copy_(torch.randn(logits.shape, generator=gen))
            out.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, call(x, logits))
    for i, t in enumerate(others, 1):
        assert bool((t == i).all())


def test_a_capture_that_would_grow_the_workspace_is_refused(cuda_device):
    """The call raises; what else was captured stands and replays."""
    dev = cuda_device
    w = prepared(dev, 768, 1024, 3)
    small, large = (torch.randn(m, 1024, device=dev, dtype=torch.bfloat16) for m in (3, 700))
    ref = fp8_block_linear(small, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fp8_block_linear(small, w)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = fp8_block_linear(small, w)
            with pytest.raises(RuntimeError, match="before capturing"):
                fp8_block_linear(large, w)
            again = fp8_block_linear(small, w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ref) and torch.equal(again, ref)
    with torch.cuda.stream(side):
        assert fp8_block_linear(large, w).shape == (700, 768)


def test_two_threads_on_one_stream(cuda_device):
    """Each thread gets its own results, whatever the other one calls in between."""
    dev = cuda_device
    w = prepared(dev, 768, 1024, 3)
    gate_up, down = prepared(dev, 512, 1024, 4, experts=8, gate_up=True), prepared(dev, 1024, 256, 5, experts=8)

    def layer(x, logits):
        return fp8_block_linear(x, w), fp8_moe_experts(x, launch_moe_route(logits, 3), gate_up, down)

    inputs = [(torch.randn(m, 1024, device=dev, dtype=torch.bfloat16), torch.randn(m, 8, device=dev)) for m in (40, 57, 3, 300)]
    refs = [layer(*i) for i in inputs]
    torch.cuda.synchronize()
    wrong = []

    def many(n):
        for _ in range(60):
            got = layer(*inputs[n])
            torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, refs[n])):
                wrong.append(n)

    threads = [threading.Thread(target=many, args=(n,)) for n in range(len(inputs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
