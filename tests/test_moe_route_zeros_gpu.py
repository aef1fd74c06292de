"""Router: zeros of either sign are equal scores, so the lower expert comes first."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mambo_b200 import _lib
from mambo_b200.kernels.moe_fp8 import launch_moe_route

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bias", [None, 0.0, -0.0])
@pytest.mark.parametrize("e", [8, 70, 256])
def test_zeros_of_either_sign_tie(cuda_device, e, bias, dtype):
    signs = np.random.default_rng(e).integers(0, 2, size=(20, e))
    logits = torch.from_numpy(np.where(signs, -0.0, 0.0).astype(np.float32)).to(cuda_device, dtype)
    b = None if bias is None else torch.full((e,), bias, device=cuda_device)
    route = launch_moe_route(logits, 6, bias=b)
    assert np.array_equal(route["ids"].cpu().numpy(), np.tile(np.arange(6), (20, 1)))
    # 1/e each, divided by the sum of six: 8 roundings of 2^-24 at most.
    assert np.allclose(route["weights"].cpu().numpy(), 1 / 6, rtol=8 * 2.0 ** -24, atol=0)
    assert _lib.device_status()[0] == 0
