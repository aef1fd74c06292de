"""CPU: rotary fields whose tensor was replaced are refused before anything is launched."""

from __future__ import annotations

import types

import pytest
import torch

from mambo_b200 import _lib
from mambo_b200.kernels import rotary

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
