"""CPU: size functions and argument checks of the FP8 block and expert entry points: huge sizes, unaligned pointers."""

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


def test_unaligned_pointers_are_refused():
    """A pointer off its elements' alignment is an error of the call, never a fault of the GPU (no device is needed)."""
    lib, e, f32, bf16 = _lib.load(), _lib.MAMBO_EINVAL, _lib.MAMBO_F32, _lib.MAMBO_BF16
    big = (1 << 63) - 1
    w = _lib.MamboFp8BlockWeight(4096, 4096, 256, 256, 1, 0)
    grouped = _lib.MamboFp8BlockWeight(4096, 4096, 256, 256, 4, 0)
    gate_up = _lib.MamboFp8BlockWeight(4096, 4096, 256, 256, 4, 1)
    down = _lib.MamboFp8BlockWeight(4096, 4096, 256, 128, 4, 0)

    def refused(call, good, pointers):
        for name, off in pointers:
            assert call(**{**good, name: 4096 + off}) == e, (name, off)
            assert "aligned" in _lib.last_error()

    refused(lambda s, ps: lib.mambo_fp8b_pack(4096, 1, 256, 256, 0, 256, 1, s, 0, 2, 1, 0, 4096, ps, None),
            dict(s=4096, ps=4096), [("s", 2), ("ps", 2)])
    refused(lambda x, t: lib.mambo_fp8b_quantize(x, t, 4, 256, 256, 128, 4096, 256, 4096, 2, None), dict(x=4096, t=f32),
            [("x", 1), ("x", 2)])
    refused(lambda x, t: lib.mambo_fp8b_quantize(x, t, 4, 256, 256, 128, 4096, 256, 4096, 2, None), dict(x=4096, t=bf16),
            [("x", 1)])
    for t, off in ((f32, 2), (bf16, 1)):
        refused(lambda x, out: lib.mambo_fp8b_linear_fused(x, t, 256, 128, 4, w, out, t, 256, 4096, big, None),  # noqa: B023
                dict(x=4096, out=4096), [("x", off), ("out", off)])
        refused(lambda out: lib.mambo_fp8b_linear(4097, 256, 4097, 2, 128, 4, w, out, t, 256, 4096, big, None),  # noqa: B023
                dict(out=4096), [("out", off)])
        refused(lambda x, o, out: lib.mambo_fp8b_grouped_linear(x, t, 256, 128, 4, o, grouped, out, t, 256, 4096,  # noqa: B023
                                                                big, None),
                dict(x=4096, o=4096, out=4096), [("x", off), ("o", 2), ("out", off)])
        refused(lambda l, b, i, wt, o, p, r: lib.mambo_moe_route(l, t, 8, b, 4, 8, 2, 0, 1, 1.0, i, wt, o, p, r, 4096,  # noqa: B023
                                                                 big, None),
                dict(l=4096, b=4096, i=4096, wt=4096, o=4096, p=4096, r=4096),
                [("l", off), ("b", 2), ("i", 2), ("wt", 2), ("o", 2), ("p", 2), ("r", 2)])
        refused(lambda y, p, wt, out: lib.mambo_moe_combine(y, t, 8, 8, p, wt, 4, 2, 8, out, t, 8, None),  # noqa: B023
                dict(y=4096, p=4096, wt=4096, out=4096), [("y", off), ("p", 2), ("wt", 2), ("out", off)])
        refused(lambda x, i, wt, p, o, r, out: lib.mambo_moe_experts(x, t, 256, 4, i, wt, p, o, r, 2, gate_up, down,  # noqa: B023
                                                                     out, t, 256, 4096, big, None),
                dict(x=4096, i=4096, wt=4096, p=4096, o=4096, r=4096, out=4096),
                [("x", off), ("i", 2), ("wt", 2), ("p", 2), ("o", 2), ("r", 2), ("out", off)])
