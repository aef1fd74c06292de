"""Tiles split along K in every form that the rule reaches: each tile width, after a whole wave, CTA pairs, hidden epilogue."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mambo_b200 import _lib
from mambo_b200.kernels.fp8_block import fp8_block_linear, prepare_fp8_block_fields
from mambo_b200.kernels.moe_fp8 import fp8_moe_experts, launch_moe_route
from test_fp8_block_gpu import check, frob, make_weight, make_x, quantize64, weight64
from test_moe_fp8_gpu import EXPERTS_F32_TOL, experts_ref, make_experts, route_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert _lib.device_status()[0] == 0


@pytest.mark.parametrize("m,n,k", [(1, 300, 14336), (16, 2000, 8192), (2, 19000, 4200), (32, 1024, 8192), (20, 19000, 4200),
                                   (64, 2048, 14336), (50, 4100, 20480), (384, 2000, 14336), (100, 4096, 20000)])
def test_split_linear(cuda_device, m, n, k):
    codes, scales = make_weight(n, k, n + m)
    w = prepare_fp8_block_fields(torch.from_numpy(codes).to(cuda_device), torch.from_numpy(scales).to(cuda_device))
    x = make_x(m, k, 5).bfloat16()
    out = fp8_block_linear(x.to(cuda_device), w, out_dtype=torch.float32)
    check(out, quantize64(x.double().numpy(), 128)[0] @ weight64(codes, scales).T)
    for _ in range(3):  # the same sums in the same order, whichever CTA arrives last
        assert torch.equal(out, fp8_block_linear(x.to(cuda_device), w, out_dtype=torch.float32))
    assert torch.equal(out.bfloat16(), fp8_block_linear(x.to(cuda_device), w))


@pytest.mark.parametrize("t,e,k,h,i", [(1, 4, 3, 6000, 100), (32, 1, 1, 8192, 64), (40, 2, 1, 20480, 500), (64, 1, 1, 24576, 512),
                                       (16, 2, 2, 300, 8192), (60, 1, 1, 520, 16384)])
def test_split_experts(cuda_device, t, e, k, h, i):
    """Split gate/up products (their parts meet before the hidden activations are formed) and split down products."""
    gu, gus, down, downs = make_experts(e, h, i, t + e)
    gus *= np.float32((4096 / max(h, 4096)) ** 0.5)
    dev = cuda_device
    wg = prepare_fp8_block_fields(torch.from_numpy(gu).to(dev), torch.from_numpy(gus).to(dev), gate_up=True)
    wd = prepare_fp8_block_fields(torch.from_numpy(down).to(dev), torch.from_numpy(downs).to(dev))
    logits = np.random.default_rng(t).standard_normal((t, e)).astype(np.float32)
    x = make_x(t, h, 3) * 0.25
    route = launch_moe_route(torch.from_numpy(logits).to(dev), k)
    ref = experts_ref(x.numpy(), route_ref(logits, k), gu, gus, down, downs)
    out = fp8_moe_experts(x.to(dev), route, wg, wd, out_dtype=torch.float32)
    assert frob(out.cpu(), ref) < EXPERTS_F32_TOL
    for _ in range(3):
        assert torch.equal(out, fp8_moe_experts(x.to(dev), route, wg, wd, out_dtype=torch.float32))
