"""Rotation, append and attention called one behind the other see what the call before has written."""

from __future__ import annotations

import pytest
import torch

from mambo_b200 import _lib
from mambo_b200.kernels.attention_fp8 import fp8_paged_attention, launch_fp8_kv_append, prepare_fp8_kv_cache
from mambo_b200.kernels.rotary import launch_rotary, prepare_rotary_fields

pytestmark = pytest.mark.gpu


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def test_steps_without_a_pause(cuda_device):
    """Ragged steps whose calls follow one another on the GPU, in which single tokens and chunks come together: the same
    bits as with the GPU waited for between the calls. Values grow from step to step, so that the scales of begun pages,
    and with them the older codes, are written anew each time."""
    gen = torch.Generator().manual_seed(5)
    heads, kv, dim, page, batch, columns = 8, 2, 64, 32, 6, 24
    counts = [[1, 60, 1, 7, 100, 1], [5, 1, 70, 1, 1, 90], [1, 1, 1, 1, 1, 40], [33, 2, 1, 90, 1, 1]]
    rope = prepare_rotary_fields(dim)
    table = torch.randperm(batch * columns, generator=gen).int().view(batch, columns).cuda()
    lengths, steps = [i32([200, 3, 90, 31, 64, 0])], []
    for i, n in enumerate(counts):
        total = sum(n)
        q, k, v = ((torch.randn(total, h, dim, generator=gen) * 2.0 ** i).bfloat16().cuda() for h in (heads, kv, kv))
        at = torch.cat([int(b) + torch.arange(c, dtype=torch.int32) for b, c in zip(lengths[-1].tolist(), n)]).cuda()
        steps.append((q, k, v, at, i32([sum(n[:b]) for b in range(batch + 1)])))
        lengths.append(lengths[-1] + i32(n))

    def go(pause):
        cache, outs = prepare_fp8_kv_cache(batch * columns, kv, page, dim), []
        torch.cuda.synchronize()
        for i, (q, k, v, at, offsets) in enumerate(steps):
            turned = launch_rotary(q, at, rope)
            pause()
            launch_fp8_kv_append(cache, k, v, table, lengths[i], offsets=offsets, rope=rope)
            pause()
            outs.append(fp8_paged_attention(turned, cache, table, lengths[i + 1], offsets=offsets, out=turned))
            pause()
        torch.cuda.synchronize()
        return [*outs, *cache.values()]

    want = go(torch.cuda.synchronize)
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(go(lambda: None), want))
    assert _lib.device_status()[0] == 0
