"""Rotary positions against float64, at the sizes, layouts and strides where they can go wrong."""

from __future__ import annotations

import math

import pytest
import torch

from kv_reference import turned64, turned_bound
from mambo_b200 import _lib
from mambo_b200.kernels.rotary import launch_rotary, prepare_rotary_fields, rotary_frequencies

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert _lib.device_status()[0] == 0


def check(out, x, positions, rotary, *, interleaved=False, inverse=False, radians=None, magnitude=1.0):
    radians = rotary_frequencies(rotary)[0] if radians is None else radians
    ref = turned64(x, positions, radians, interleaved=interleaved, magnitude=magnitude, inverse=inverse)
    off, bound = (out.double() - ref).abs(), turned_bound(x, rotary, magnitude, interleaved)
    bound = bound.repeat_interleave(2, dim=-1) if interleaved else torch.cat([bound, bound], dim=-1)
    if out.dtype == BF16:
        bound = bound * (1 + 2.0 ** -8) + 2.0 ** -8 * ref[..., :rotary].abs()
    assert (off[..., :rotary] <= bound).all(), float((off[..., :rotary] - bound).max())
    assert torch.equal(out[..., rotary:], x[..., rotary:])


def inputs(tokens, heads, dim, dtype, far=5000, seed=0, int64=False):
    gen = torch.Generator().manual_seed(seed + 1000 * tokens + dim)
    x = torch.randn(tokens, heads, dim, generator=gen).to(dtype).cuda()
    return x, torch.randint(0, far, (tokens,), generator=gen, dtype=torch.int64 if int64 else torch.int32).cuda()


SIZES = [(1, 1, 2, 2), (1, 1, 128, 128), (3, 5, 128, 128), (7, 3, 96, 72), (130, 2, 64, 16), (5, 40, 80, 80), (2, 1, 10, 6),
         (33, 7, 144, 144), (2, 3, 576, 64), (257, 8, 128, 64), (2, 1, 7, 4), (1000, 33, 16, 16), (3, 1024, 16, 8)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rotary", SIZES)
def test_sizes_and_layouts(cuda_device, tokens, heads, dim, rotary, interleaved, dtype):
    x, positions = inputs(tokens, heads, dim, dtype)
    rope = prepare_rotary_fields(rotary, interleaved=interleaved)
    out = launch_rotary(x, positions, rope)
    assert out.shape == x.shape and out.dtype == x.dtype
    check(out, x, positions, rotary, interleaved=interleaved)
    assert torch.equal(launch_rotary(x, positions, rope), out)


@pytest.mark.parametrize("kwargs", [dict(scaling="linear", factor=4.0), dict(scaling="bands", factor=8.0),
                                    dict(scaling="yarn", factor=16.0, original_length=4096), dict(base=500000.0),
                                    dict(scaling="yarn", factor=0.5), dict(magnitude=-0.25)])
def test_scalings(cuda_device, kwargs):
    x, positions = inputs(20, 6, 128, F32, far=1 << 20)
    radians, magnitude = rotary_frequencies(128, **{k: v for k, v in kwargs.items() if k != "magnitude"})
    out = launch_rotary(x, positions, prepare_rotary_fields(128, **kwargs))
    check(out, x, positions, 128, radians=radians, magnitude=kwargs.get("magnitude", magnitude))


def test_given_frequencies(cuda_device):
    """Frequencies above a turn and below zero; the angle is one in 64 bits."""
    x, positions = inputs(50, 3, 12, F32, far=100)
    radians = [7.5, -0.3, 0.0, 100.25, math.pi, -2 * math.pi]
    check(launch_rotary(x, positions, prepare_rotary_fields(12, frequencies=radians)), x, positions, 12, radians=radians)


def test_far_and_negative_positions(cuda_device):
    x = inputs(9, 4, 64, F32)[0]
    positions = torch.tensor([0, 1, -1, -5000, 1 << 20, (1 << 31) - 1, -(1 << 31), 1 << 33, -(1 << 33)], device="cuda")
    rope = prepare_rotary_fields(64)
    # A frequency's rounding in 64 bits moves the angle at 2^33 by 2^33 * 2^-53: 2^-20, which is added to the bound.
    ref = turned64(x, positions, rotary_frequencies(64)[0])
    bound = turned_bound(x, 64, 1.0, False) + 2 * 2.0 ** -20 * (x.double().abs()[..., :32] + x.double().abs()[..., 32:])
    assert ((launch_rotary(x, positions, rope).double() - ref).abs() <= torch.cat([bound, bound], -1)).all()
    near = positions[:7].int()
    assert torch.equal(launch_rotary(x[:7], near, rope), launch_rotary(x[:7], positions[:7], rope))


@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_is_the_gradient(cuda_device, interleaved):
    """Of sum(w * rotary(x)): by the formula, and by differences, which of a linear function are exact but for roundings."""
    x, positions = inputs(6, 5, 48, F32)
    w = torch.randn_like(x)
    rope = prepare_rotary_fields(32, interleaved=interleaved, scaling="yarn", factor=4.0)
    radians, magnitude = rotary_frequencies(32, scaling="yarn", factor=4.0)
    grad = launch_rotary(w, positions, rope, inverse=True)
    check(grad, w, positions, 32, interleaved=interleaved, inverse=True, radians=radians, magnitude=magnitude)
    step = torch.randn_like(x)
    up, down = (launch_rotary(x + s * step, positions, rope).double() for s in (1.0, -1.0))
    difference = (w.double() * (up - down)).sum() / 2
    # 1440 terms, each off by some 2^-21 of |w| * (|x| + |step|) on either side: 1440 * 2 * 16 * 2^-21 at most.
    assert abs(float(difference - (grad.double() * step.double()).sum())) < 1440 * 32 * 2.0 ** -21
    back = launch_rotary(launch_rotary(x, positions, rope), positions, rope, inverse=True)
    assert torch.allclose(back[..., :32], x[..., :32] * magnitude ** 2, rtol=0, atol=2.0 ** -18 * float(x.abs().max()))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("offset", [0, 1, 4, 8])
def test_strides_and_alignment(cuda_device, offset, interleaved, dtype):
    """Views of a projection's output (first element anywhere), a transposed and an expanded one, positions with a stride."""
    tokens, heads, dim, rotary = 11, 6, 64, 48
    base = torch.randn(tokens, offset + 10 * dim + 3, device="cuda").to(dtype)
    x = base[:, offset:offset + heads * dim].view(tokens, heads, dim) if offset == 0 else \
        base.as_strided((tokens, heads, dim), (base.shape[1], dim, 1), offset)
    positions = torch.randint(0, 999, (tokens, 2), device="cuda")[:, 1]
    rope = prepare_rotary_fields(rotary, interleaved=interleaved)
    check(launch_rotary(x, positions, rope), x, positions, rotary, interleaved=interleaved)
    for view in (x.transpose(0, 1).contiguous().transpose(0, 1), x[:, ::2], x[:1].expand(tokens, heads, dim),
                 x.transpose(1, 2).contiguous().transpose(1, 2)):
        check(launch_rotary(view, positions, rope), view, positions, rotary, interleaved=interleaved)
    held = base.clone()
    out = held.as_strided((tokens, heads, dim), (base.shape[1], dim, 1), offset)
    assert launch_rotary(x, positions, rope, out=out) is out
    check(out, x, positions, rotary, interleaved=interleaved)
    out.copy_(x)
    assert torch.equal(held, base)  # nothing else was written
    want = launch_rotary(x, positions, rope)
    assert torch.equal(launch_rotary(out, positions, rope, out=out), want)  # in place


def test_offsets_past_32_bits(cuda_device):
    """Tokens 2^31 elements apart, and the second at an offset of more than 2^32 bytes."""
    rope, stride = prepare_rotary_fields(64), (1 << 31) + 64
    big = torch.empty(2 * stride, dtype=BF16, device="cuda")
    x = big.as_strided((2, 3, 64), (stride, 64, 1))
    x.copy_(torch.randn(2, 3, 64))
    positions = torch.tensor([3, 70], dtype=torch.int32, device="cuda")
    check(launch_rotary(x, positions, rope), x, positions, 64)
    want = launch_rotary(x, positions, rope)
    assert torch.equal(launch_rotary(x, positions, rope, out=x), want)


def test_not_finite(cuda_device):
    """A NaN or an infinity stays in its pair."""
    x, positions = inputs(4, 2, 32, F32)
    rope = prepare_rotary_fields(32)
    clean = launch_rotary(x, positions, rope)
    x[1, 0, 3], x[2, 1, 20] = math.nan, math.inf
    out = launch_rotary(x, positions, rope)
    touched = torch.zeros_like(x, dtype=torch.bool)
    touched[1, 0, [3, 19]] = touched[2, 1, [4, 20]] = True
    assert torch.equal(out[~touched], clean[~touched]) and not out[touched].isfinite().any()


def test_no_tokens_streams_and_graphs(cuda_device):
    rope = prepare_rotary_fields(64)
    x, positions = inputs(40, 8, 64, BF16)
    assert launch_rotary(x[:0], positions[:0], rope).shape == (0, 8, 64)
    want = launch_rotary(x, positions, rope)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = launch_rotary(x, positions, rope, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = launch_rotary(x, positions, rope)
    positions += 5
    x.mul_(0.5)
    graph.replay()
    check(held, x, positions, 64)


def test_refusals(cuda_device):
    rope = prepare_rotary_fields(64)
    x, positions = inputs(4, 2, 64, BF16)
    for bad in (x.half(), x[0], x[:, :0]):
        with pytest.raises(ValueError):
            launch_rotary(bad, positions, rope)
    for bad in (positions[:3], positions.float(), positions.short(), positions[:, None]):
        with pytest.raises(ValueError):
            launch_rotary(x, bad, rope)
    with pytest.raises(ValueError, match="CUDA"):
        launch_rotary(x, positions.cpu(), rope)
    with pytest.raises(ValueError, match="larger than the head"):
        launch_rotary(x[..., :32], positions, rope)
    with pytest.raises(TypeError):
        launch_rotary(x, positions, {"turns": rope["turns"]})
    for out in (x.float(), x[:3], torch.empty(4, 64, 2, dtype=BF16, device="cuda").transpose(1, 2)):
        with pytest.raises(ValueError):
            launch_rotary(x, positions, rope, out=out)
    turned = x.transpose(1, 2).contiguous().transpose(1, 2)
    with pytest.raises(ValueError, match="in place"):
        launch_rotary(turned, positions, rope, out=turned)
