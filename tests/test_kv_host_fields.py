"""CPU: rotary fields whose tensor was replaced, and cache sizes past 64 bits, are refused before anything is launched."""

from __future__ import annotations

import types

import pytest
import torch

from mambo_b200 import _lib
from mambo_b200.kernels import rotary

P = 4096  # a pointer that no refused call follows
CPU = types.SimpleNamespace(index=-1)  # the device of tensors that have none


def test_replaced_tables_are_refused():
    """A copy of the fields with another table (moved, cloned): its C view still points to the first one's memory."""
    turns = torch.zeros(4, dtype=torch.int64)
    rope = {"turns": turns, "rotary_dim": 8, "interleaved": False, "magnitude": 1.0,
            "rotary": _lib.MamboRotary(turns.data_ptr(), 8, 0, 1.0)}
    rotary._check_rope(rope, 8, CPU)
    rotary._check_rope({**rope}, 16, CPU)
    for other in (turns.clone(), turns[1:], torch.zeros(8, dtype=torch.int64)):
        with pytest.raises(ValueError, match="replaced"):
            rotary._check_rope({**rope, "turns": other}, 8, CPU)
    for missing in ("turns", "rotary"):
        with pytest.raises(TypeError):
            rotary._check_rope({k: v for k, v in rope.items() if k != missing}, 8, CPU)


@pytest.mark.parametrize("pages,heads", [(1 << 54, 1024), (1 << 62, 4), (1 << 63 - 1, 2), ((1 << 62) + 1, 4), (1 << 31, 2)])
def test_cache_sizes_past_64_bits(pages, heads):
    """Pages times heads that wrap to something small."""
    lib = _lib.load()
    cache = _lib.MamboKvCache(P, P, P, P, pages, heads, 16, 64)
    seq = _lib.MamboKvSequences(P, 4, 4, P, None, 3)
    assert lib.mambo_kv_append(cache, P, 128, 64, P, 128, 64, _lib.MAMBO_BF16, 3, seq, None, None) == _lib.MAMBO_EINVAL
    assert "pages" in _lib.last_error()
    need = lib.mambo_kv_attention_workspace_bytes(heads, heads, 0)
    assert lib.mambo_kv_attention(P, 64 * heads, 64, 3, heads, cache, seq, 0, 1.0, P, 64 * heads, 64, None, heads, 1, P, need,
                                  None) == _lib.MAMBO_EINVAL
    assert "pages" in _lib.last_error()
