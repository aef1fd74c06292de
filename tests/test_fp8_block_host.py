"""CPU: the FP8 block and expert entry points check their arguments and sizes before any device work."""

from __future__ import annotations

import pytest
import torch

from mambo_b200 import _lib
from mambo_b200.kernels import fp8_block, moe_fp8


def test_sizes():
    lib = _lib.load()
    # One 16 KB record per (128-row tile, 128-wide K block) and expert, two scales each; gate and up in whole blocks of
    # 128 features.
    assert lib.mambo_fp8b_packed_bytes(1, 128, 128, 0) == 16384
    assert lib.mambo_fp8b_packed_bytes(3, 129, 257, 0) == 3 * 2 * 3 * 16384
    assert lib.mambo_fp8b_packed_bytes(1, 200, 128, 1) == 2 * 16384
    assert lib.mambo_fp8b_packed_bytes(1, 258, 128, 1) == 4 * 16384
    assert lib.mambo_fp8b_scales_bytes(3, 129, 257, 0) == 3 * 2 * 3 * 8
    assert lib.mambo_fp8b_packed_bytes(0, 128, 128, 0) == 0 and lib.mambo_fp8b_packed_bytes(2000, 128, 128, 0) == 0
    sizes = [lib.mambo_fp8b_linear_workspace_bytes(m, 1, 4096, 4096) for m in (1, 16, 64, 4096)]
    assert all(0 < a <= b for a, b in zip(sizes, sizes[1:]))
    assert lib.mambo_fp8b_linear_workspace_bytes(0, 1, 4096, 4096) == 0
    assert lib.mambo_moe_route_workspace_bytes(16384, 256) > lib.mambo_moe_route_workspace_bytes(1, 8) > 0
    assert lib.mambo_moe_experts_workspace_bytes(4, 2, 8, 256, 128, _lib.MAMBO_F32) \
        > lib.mambo_moe_experts_workspace_bytes(4, 2, 8, 256, 128, _lib.MAMBO_BF16) > 0


def test_arguments_are_refused_without_a_device():
    lib, e = _lib.load(), _lib.MAMBO_EINVAL
    w = _lib.MamboFp8BlockWeight(4096, 4096, 256, 256, 1, 0)
    experts = _lib.MamboFp8BlockWeight(4096, 4096, 256, 256, 4, 0)
    gate_up = _lib.MamboFp8BlockWeight(4096, 4096, 256, 256, 4, 1)
    empty = _lib.MamboFp8BlockWeight()

    def linear(x=4096, dt=_lib.MAMBO_BF16, ldx=256, group=128, m=4, weight=w, out=4096, odt=_lib.MAMBO_BF16, ldo=256):
        return lib.mambo_fp8b_linear_fused(x, dt, ldx, group, m, weight, out, odt, ldo, None, 0, None)

    for bad in (dict(x=None), dict(out=None), dict(dt=7), dict(ldx=255), dict(group=64), dict(m=0), dict(m=1 << 29),
                dict(weight=None), dict(weight=empty), dict(weight=experts), dict(weight=gate_up), dict(odt=3), dict(ldo=255)):
        assert linear(**bad) == e, bad
        assert _lib.last_error()
    assert lib.mambo_fp8b_linear(4096, 256, None, 2, 128, 4, w, 4096, 0, 256, None, 0, None) == e
    assert lib.mambo_fp8b_linear(4096, 256, 4096, 1, 128, 4, w, 4096, 0, 256, None, 0, None) == e
    assert lib.mambo_fp8b_grouped_linear(4096, 0, 256, 128, 4, None, experts, 4096, 0, 256, None, 0, None) == e
    assert lib.mambo_fp8b_pack(4096, 1, 255, 128, 0, 1, 1, 4096, 0, 1, 1, 1, 4096, 4096, None) == e
    assert lib.mambo_fp8b_pack(4096, 1, 256, 128, 0, 1, 1, 4096, 0, 1, 1, 0, 4097, 4096, None) == e
    assert lib.mambo_fp8b_quantize(4096, 0, 4, 100, 100, 128, 4096, 100, 4096, 0, None) == e
    assert lib.mambo_moe_route(4096, 0, 8, None, 4, 8, 9, 0, 1, 1.0, 1, 1, 1, 1, None, 4096, 1 << 30, None) == e
    assert lib.mambo_moe_route(4096, 0, 8, None, 4, 8, 2, 5, 1, 1.0, 1, 1, 1, 1, None, 4096, 1 << 30, None) == e
    assert lib.mambo_moe_route(4096, 0, 8, None, 4, 8, 2, 0, 1, 1.0, 1, 1, 1, 1, None, 4096, 16, None) == _lib.MAMBO_EWORKSPACE
    assert lib.mambo_moe_combine(4096, 0, 7, 4, 4096, 4096, 2, 2, 8, 4096, 0, 8, None) == e
    assert lib.mambo_moe_experts(1, 1, 256, 4, 1, 1, 1, 1, 1, 2, w, w, 1, 1, 256, None, 0, None) == e
    assert lib.mambo_moe_experts(1, 1, 256, 4, 1, 1, 1, 1, 1, 2, gate_up, experts, 1, 1, 256, None, 0, None) == e


def test_cpu_tensors_are_refused():
    c, s = torch.zeros(256, 256, dtype=torch.uint8), torch.ones(2, 2)
    with pytest.raises(ValueError, match="CUDA"):
        fp8_block.prepare_fp8_block_fields(c, s)
    with pytest.raises(ValueError, match="CUDA"):
        fp8_block.launch_quantize_fp8_block(torch.zeros(2, 256))
    with pytest.raises(ValueError, match="CUDA"):
        moe_fp8.launch_moe_route(torch.zeros(2, 8), 2)
