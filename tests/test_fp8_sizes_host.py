"""CPU: size functions and argument checks of the FP8 block and expert entry points at the ends of 64 bits."""

from __future__ import annotations

import subprocess
import sys

from conftest import ROOT
from mambo_b200 import _lib

HUGE = [1 << 29, 1 << 31, 1 << 32, (1 << 32) + 1, 1 << 40, (1 << 60) + 1, 1 << 62, (1 << 63) - 1]


def isolated(code: str) -> str:
    """The output of a process of its own, which a crash ends with another status than 0."""
    run = subprocess.run([sys.executable, "-c", "from mambo_b200 import _lib\nlib = _lib.load()\n" + code], cwd=ROOT,
                         capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, (run.returncode, run.stderr[-500:])
    return run.stdout


def test_sizes_of_huge_calls_are_zero():
    """No size function divides by zero, and none wraps around to a small size."""
    out = isolated(f"""
for v in {HUGE}:
    for args in ((v, 8), (v, 1024)):
        assert lib.mambo_moe_route_workspace_bytes(*args) == 0, args
    assert lib.mambo_moe_route_workspace_bytes(16, v) == 0
    for i in range(4):
        a = [16, 2, 256, 256]
        a[i] = v
        assert lib.mambo_fp8b_linear_workspace_bytes(*a) == 0, a
    for i in (0, 2, 3, 4):
        a = [16, 2, 8, 256, 128, 1]
        a[i] = v
        assert lib.mambo_moe_experts_workspace_bytes(*a) == 0, a
    for i in range(3):
        a = [2, 256, 256, 0]
        a[i] = v
        assert lib.mambo_fp8b_packed_bytes(*a) == 0 and lib.mambo_fp8b_scales_bytes(*a) == 0, a
for top in (33, 1 << 20, (1 << 31) - 1):
    assert lib.mambo_moe_experts_workspace_bytes(16, top, 64, 256, 128, 1) == 0
print("done")
""")
    assert out.strip() == "done"


def test_token_counts_do_not_wrap_around():
    """tokens * top past 64 bits is refused like any other size past the limit."""
    out = isolated(f"""
e, big = _lib.MAMBO_EINVAL, (1 << 63) - 1
gate_up = _lib.MamboFp8BlockWeight(4096, 4096, 256, 256, 64, 1)
down = _lib.MamboFp8BlockWeight(4096, 4096, 256, 128, 64, 0)
for tokens in {HUGE}:
    for top in (2, 4, 16, 32):
        assert lib.mambo_moe_route(4096, 0, 64, None, tokens, 64, top, 0, 1, 1.0, 4096, 4096, 4096, 4096, None, 4096, big,
                                   None) == e and "tokens" in _lib.last_error(), (tokens, top)
        assert lib.mambo_moe_combine(4096, 0, 8, 4, 4096, 4096, tokens, top, 8, 4096, 0, 8, None) == e, (tokens, top)
        assert lib.mambo_moe_experts(4096, 1, 256, tokens, 4096, 4096, 4096, 4096, 4096, top, gate_up, down, 4096, 1, 256,
                                     4096, big, None) == e and "tokens" in _lib.last_error(), (tokens, top)
assert lib.mambo_moe_combine(4096, 0, 8, 4, 4096, 4096, 1 << 40, 1 << 24, 8, 4096, 0, 8, None) == e
assert lib.mambo_moe_combine(4096, 0, 8, 4, 4096, 4096, 4, (1 << 31) - 1, 8, 4096, 0, 8, None) == e
print("done")
""")
    assert out.strip() == "done"
