"""The GGUF operators with a ``stream=`` that is not the current one: strided inputs, and results let go of early."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mambo_b200 import _lib, _runtime
from mambo_b200.kernels.iq3_s_fp8 import fused_linear_into, iq3_s_fp8_linear, iq3_s_fp8_linear_group
from mambo_b200.kernels.q4_k_fp8 import launch_quantize_fp8_sums, prepare_q4_k_fields, q4_k_fp8_linear
from mambo_b200.kernels.quantize_fp8 import launch_quantize_fp8
from mambo_b200.utils.iq3_s_weight import prepare_iq3_s_fields
from oracle import gguf_quants_oracle as G
from oracle import iq3s_oracle as O
from test_streams_gpu import busy, equal, fill_freed_memory, tensors

pytestmark = pytest.mark.gpu

M, N, K = 12, 256, 512
NAMES = ["iq3", "group", "quantize", "sums", "q4k", "prepare_q4k"]


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    torch.cuda.synchronize()
    assert _lib.device_status()[0] == 0


@pytest.fixture(scope="module")
def operators(cuda_device):
    dev = cuda_device
    w3 = prepare_iq3_s_fields(torch.from_numpy(O.make_synthetic_iq3s(N, K, seed=3)).to(dev))
    w4 = prepare_q4_k_fields(torch.from_numpy(G.make_synthetic_q4_k(N, K, seed=4)).to(dev))
    torch.cuda.synchronize()
    return {
        "iq3": lambda x, s: iq3_s_fp8_linear(x, w3, stream=s),
        "group": lambda x, s: iq3_s_fp8_linear_group([x, x], [w3, w3], stream=s),
        "quantize": lambda x, s: launch_quantize_fp8(x, stream=s),
        "sums": lambda x, s: launch_quantize_fp8_sums(x, stream=s),
        "q4k": lambda x, s: q4_k_fp8_linear(x, w4, stream=s),
        "prepare_q4k": lambda x, s: prepare_q4_k_fields(x, stream=s)["packed"],
    }


def strided(name, seed):
    """An input without unit column stride, and the same contiguous."""
    if name == "prepare_q4k":
        raw = torch.from_numpy(np.ascontiguousarray(G.make_synthetic_q4_k(N, K, seed=seed)).reshape(N, -1)).cuda()
    else:
        raw = torch.randn(M, K, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()
    return raw.t().contiguous().t(), raw


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("which", ["current", "other"])
def test_strided_input_while_a_stream_is_busy(operators, name, which):
    x, plain = strided(name, 1)
    ref = operators[name](plain, None)
    side = torch.cuda.Stream()
    operators[name](strided(name, 7)[0], side)  # workspace, kernels, and other values in what the copy takes up
    torch.cuda.synchronize()
    with torch.cuda.stream(side if which == "other" else torch.cuda.current_stream()):
        busy()
    out = operators[name](x, side)
    nbytes = x.numel() * x.element_size()
    del x
    if which == "other":
        junk = fill_freed_memory(nbytes)
        torch.cuda.synchronize()
    else:
        junk = None
        side.synchronize()
    with torch.cuda.stream(side):
        assert equal(out, ref)
    del junk


@pytest.mark.parametrize("name", NAMES)
def test_results_do_not_overwrite_memory_in_use(operators, name):
    x, plain = strided(name, 3)
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


@pytest.mark.parametrize("handle", [0, 1, 2])
def test_into_calls_with_the_default_streams_handles(cuda_device, handle, monkeypatch):
    """The calls into given outputs take raw handles too, whose workspaces then come and grow."""
    monkeypatch.setattr(_runtime, "_workspaces", {})
    w = prepare_iq3_s_fields(torch.from_numpy(O.make_synthetic_iq3s(N, K, seed=3)).to(cuda_device))
    for m in (2, 12, 600):
        x = torch.randn(m, K, generator=torch.Generator().manual_seed(m)).bfloat16().to(cuda_device)
        ref, out = iq3_s_fp8_linear(x, w), torch.zeros(m, N, dtype=torch.bfloat16, device=cuda_device)
        torch.cuda.synchronize()
        fused_linear_into(x, w, out, stream=handle)
        torch.cuda.synchronize()
        assert torch.equal(out, ref)
