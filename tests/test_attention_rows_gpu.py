"""A row of the form for few rows has the same bits whatever the other rows of its unit are."""

from __future__ import annotations

import pytest
import torch

from mambo_b200 import _lib
from mambo_b200.kernels.attention_fp8 import fp8_paged_attention, launch_fp8_kv_append, prepare_fp8_kv_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rise", [2.0, 3.0, 6.0, 10.0])
@pytest.mark.parametrize("group", [2, 7, 16, 20, 32])
def test_a_row_beside_others(cuda_device, group, rise):
    """The first head's scores rise by less than the weights' headroom from tile to tile, or by more; those of the others
    stay, or rise by far more, or are not finite."""
    gen = torch.Generator().manual_seed(group)
    n, page, dim, batch = 1000, 32, 64, 170
    k, v = (torch.randn(n, 1, dim, generator=gen) for _ in range(2))
    k[:, 0, 0] = torch.arange(n) // 128 * rise * 0.6931 / 6  # of 8 there: 8 / sqrt(64) = 1
    k[:, 0, 1] = torch.arange(n) // 128 * 6.0
    cache, table = prepare_fp8_kv_cache(32, 1, page, dim), torch.randperm(32, generator=gen).int()[None].cuda()
    launch_fp8_kv_append(cache, k.cuda(), v.cuda(), table, torch.zeros(1, dtype=torch.int32, device="cuda"),
                         offsets=torch.tensor([0, n], dtype=torch.int32, device="cuda"))
    q = torch.randn(batch, group, dim, generator=gen).bfloat16().cuda()
    q[..., :2] = 0
    q[:, 0, 0] = 8
    lengths = (n - torch.arange(batch, dtype=torch.int32) * 3).cuda()
    calls = []
    for other in (0.0, 8.0, -8.0, float("nan"), float("inf")):
        q[:, 1:, 1] = other
        calls.append(fp8_paged_attention(q, cache, table.expand(batch, -1), lengths, return_lse=True))
    calls.append(fp8_paged_attention(q[:, :1], cache, table.expand(batch, -1), lengths, return_lse=True))
    for out, lse in calls[1:] if group <= 16 else calls[1:-1]:  # one head alone has the form for 16 rows
        assert torch.equal(out[:, 0].view(torch.int16), calls[0][0][:, 0].view(torch.int16))
        assert torch.equal(lse[:, 0], calls[0][1][:, 0])
    assert _lib.device_status()[0] == 0
