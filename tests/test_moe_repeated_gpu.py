"""Routes that name an expert more than once for a token, which launch_moe_route never makes but a caller may."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mambo_b200 import _lib
from mambo_b200.kernels.fp8_block import prepare_fp8_block_fields
from mambo_b200.kernels.moe_fp8 import fp8_moe_experts
from test_fp8_block_gpu import frob, make_x
from test_moe_fp8_gpu import EXPERTS_F32_TOL, experts_ref, make_experts

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert _lib.device_status()[0] == 0


def route_of(ids: np.ndarray, weights: np.ndarray, experts: int, dev) -> dict:
    """The route of given choices [T,top] (-1: none): rows in expert order, stable by token."""
    flat = np.where(ids < 0, experts, ids).reshape(-1)
    order = np.argsort(flat, kind="stable")
    positions = np.empty(flat.size, dtype=np.int32)
    positions[order] = np.arange(flat.size)
    positions[flat == experts] = -1
    offsets = np.searchsorted(flat[order], np.arange(experts + 1))
    rows = np.where(flat[order] == experts, -1, order)
    ints = lambda a: torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).to(dev)  # noqa: E731
    return {"ids": ints(ids), "weights": torch.from_numpy(weights.astype(np.float32)).to(dev), "offsets": ints(offsets),
            "positions": ints(positions.reshape(ids.shape)), "rows": ints(rows)}


def choices(kind: str, t: int, top: int, e: int) -> tuple[np.ndarray, np.ndarray]:
    rng = np.random.default_rng(top + t)
    weights = rng.uniform(0.1, 1.0, size=(t, top))
    if kind == "same":
        ids = np.full((t, top), e - 1)
    elif kind == "pairs":  # each expert twice
        ids = np.arange(top)[None] // 2 % e + np.zeros((t, 1), dtype=int)
    else:  # all but the first choice masked, as expert 0 with weight 0
        ids = np.zeros((t, top), dtype=int)
        ids[:, 0] = e - 1
        weights[:, 1:] = 0
    return ids, weights


@pytest.mark.parametrize("t", [1, 2, 3])
@pytest.mark.parametrize("kind,top,e,h,i", [("same", 3, 4, 256, 128), ("pairs", 6, 5, 200, 100), ("masked", 8, 8, 1003, 64),
                                            ("same", 9, 1, 384, 64), ("same", 32, 2, 256, 33), ("same", 17, 3, 4096, 64)])
def test_repeated_experts(cuda_device, t, kind, top, e, h, i):
    gu, gus, down, downs = make_experts(e, h, i, t + top)
    dev = cuda_device
    wg = prepare_fp8_block_fields(torch.from_numpy(gu).to(dev), torch.from_numpy(gus).to(dev), gate_up=True)
    wd = prepare_fp8_block_fields(torch.from_numpy(down).to(dev), torch.from_numpy(downs).to(dev))
    ids, weights = choices(kind, t, top, e)
    route = route_of(ids, weights, e, dev)
    for dtype in (torch.bfloat16, torch.float32):
        x = make_x(t, h, 3).to(dtype)
        ref = experts_ref(x.double().numpy(), (ids, weights.astype(np.float32).astype(np.float64)), gu, gus, down, downs)
        out = fp8_moe_experts(x.to(dev), route, wg, wd, out_dtype=torch.float32)
        assert frob(out.cpu(), ref) < EXPERTS_F32_TOL
        assert torch.equal(out, fp8_moe_experts(x.to(dev), route, wg, wd, out_dtype=torch.float32))
