"""The dimensions behind the rotated part are copied bit for bit, whatever they and their neighbours hold."""

from __future__ import annotations

import math

import pytest
import torch

from mambo_b200 import _lib
from mambo_b200.kernels.rotary import launch_rotary, prepare_rotary_fields

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [3, 700])  # one head a thread, and several
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(96, 72), (128, 2), (128, 126), (64, 32), (48, 46), (80, 48)])
@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, torch.int16), (torch.float32, torch.int32)])
def test_what_does_not_turn_is_copied(cuda_device, dtype, bits, dim, rotary, interleaved, aligned, tokens):
    gen = torch.Generator().manual_seed(dim + rotary)
    heads, off = 24, 0 if aligned else 1
    base = torch.randn(tokens * heads * dim + 1, generator=gen).to(dtype).cuda()
    x = base[off:off + tokens * heads * dim].view(tokens, heads, dim)
    rest = x[..., rotary:]
    for i, special in enumerate((math.inf, -math.inf, math.nan, -0.0)):
        rest[i % 3, i::4, i % rest.shape[2]] = special
    rest[1, 5] = -0.0
    # NaN with other bits than the usual ones
    rest[2, 3].view(bits).fill_(0x7FC1 if dtype is torch.bfloat16 else 0x7FC00123)
    positions = torch.arange(tokens, dtype=torch.int32, device="cuda") + 17
    for inverse in (False, True):
        out = launch_rotary(x, positions, prepare_rotary_fields(rotary, interleaved=interleaved), inverse=inverse)
        assert torch.equal(out[..., rotary:].contiguous().view(bits), rest.contiguous().view(bits))
        assert out[..., :rotary].isfinite().all()
    assert _lib.device_status()[0] == 0
