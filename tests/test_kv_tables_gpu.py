"""Page tables whose rows share memory: sequences over the same pages."""

from __future__ import annotations

import pytest
import torch

from kv_reference import make_cache
from mambo_b200 import _lib
from mambo_b200.kernels.attention_fp8 import fp8_paged_attention, launch_fp8_kv_append, prepare_fp8_kv_cache

pytestmark = pytest.mark.gpu


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("tokens", [1, 40])
def test_rows_that_share_memory(cuda_device, tokens):
    """One row expanded to all sequences, and rows that begin a page apart in the same memory."""
    batch, page, columns = 5, 32, 6
    cache = make_cache(torch.Generator().manual_seed(1), 12, 2, page, 64, "cuda")
    q = torch.randn(batch * tokens, 8, 64, device="cuda").bfloat16()
    lengths, offsets = i32([190, 70, 33, 128, 150]), None if tokens == 1 else i32([tokens * b for b in range(batch + 1)])
    pages = torch.randperm(12, generator=torch.Generator().manual_seed(2)).int().cuda()
    for table in (pages[:columns].expand(batch, columns), pages.as_strided((batch, columns), (1, 1))):
        want = fp8_paged_attention(q, cache, table.clone(memory_format=torch.contiguous_format), lengths, offsets=offsets)
        assert torch.equal(fp8_paged_attention(q, cache, table, lengths, offsets=offsets), want)
    assert _lib.device_status()[0] == 0


def test_append_to_one_of_the_sequences(cuda_device):
    """An expanded row in an append that has tokens of one sequence alone."""
    k, v = (torch.randn(50, 2, 64, device="cuda") for _ in range(2))
    row, caches = i32([3, 1, 0, 2]), [prepare_fp8_kv_cache(4, 2, 16, 64) for _ in range(2)]
    for cache, table in zip(caches, (row.expand(3, 4), row.expand(3, 4).contiguous())):
        launch_fp8_kv_append(cache, k, v, table, i32([0, 5, 0]), offsets=i32([0, 0, 50, 50]))
    assert all(torch.equal(caches[0][n], caches[1][n]) for n in caches[0]) and caches[0]["keys"].any()
