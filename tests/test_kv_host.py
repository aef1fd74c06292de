"""CPU: rotation frequencies against their formulas, and the cache's entry points refuse bad arguments without a device."""

from __future__ import annotations

import math

import pytest
import torch

from mambo_b200 import _lib
from mambo_b200.kernels import attention_fp8, rotary

P = 4096  # a pointer that no refused call follows


def test_plain_frequencies():
    radians, magnitude = rotary.rotary_frequencies(8, base=10000.0)
    assert magnitude == 1.0
    assert radians == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-15)
    assert rotary.rotary_frequencies(8, scaling="linear", factor=4.0)[0] == pytest.approx([0.25, 0.025, 0.0025, 0.00025])


def test_bands():
    """Pairs that turn at least four times in the original context stay, those with one turn at most are divided."""
    plain = rotary.rotary_frequencies(128, base=500000.0)[0]
    scaled, magnitude = rotary.rotary_frequencies(128, base=500000.0, scaling="bands", factor=8.0, original_length=8192)
    assert magnitude == 1.0
    for f, s in zip(plain, scaled):
        turns = 8192 * f / (2 * math.pi)
        if turns >= 4:
            assert s == f
        elif turns <= 1:
            assert s == f / 8
        else:  # the wavelength's share of the band between the two
            keep = (turns - 1) / 3
            assert s == pytest.approx((1 - keep) * f / 8 + keep * f, rel=1e-12) and f / 8 < s < f


def test_yarn():
    plain = rotary.rotary_frequencies(64)[0]
    scaled, magnitude = rotary.rotary_frequencies(64, scaling="yarn", factor=16.0, original_length=4096)
    assert magnitude == pytest.approx(0.1 * math.log(16.0) + 1)
    ratio = [s / f for s, f in zip(scaled, plain)]
    assert ratio[0] == 1.0 and ratio[-1] == pytest.approx(1 / 16)
    assert all(a >= b - 1e-15 for a, b in zip(ratio, ratio[1:]))
    # Pairs that turn 32 times and once: rotary_dim * ln(length / (2 pi turns)) / (2 ln base).
    first, last = (64 * math.log(4096 / (2 * math.pi * n)) / (2 * math.log(10000.0)) for n in (32, 1))
    for p, r in enumerate(ratio):
        ramp = min(1, max(0, (p - math.floor(first)) / (math.ceil(last) - math.floor(first))))
        assert r == pytest.approx(ramp / 16 + 1 - ramp, rel=1e-12)


@pytest.mark.parametrize("kwargs", [dict(rotary_dim=0), dict(rotary_dim=7), dict(scaling="other"), dict(base=1.0),
                                    dict(factor=0.0), dict(original_length=0), dict(scaling="bands", low=4.0, high=4.0),
                                    dict(base=math.nan), dict(factor=-1.0)])
def test_frequency_refusals(kwargs):
    with pytest.raises(ValueError):
        rotary.rotary_frequencies(**{"rotary_dim": 64, **kwargs})


def test_prepare_refusals():
    for frequencies in ([1.0], [1.0, math.inf], [math.nan, 1.0]):
        with pytest.raises(ValueError):
            rotary.prepare_rotary_fields(4, frequencies=frequencies)
    with pytest.raises(ValueError):
        rotary.prepare_rotary_fields(3, frequencies=[1.0])
    with pytest.raises(ValueError, match="CUDA"):
        rotary.prepare_rotary_fields(4, device="cpu")
    for bad in ((1, 1, 8, 64), (1, 1, 256, 64), (1, 1, 16, 24), (1, 1, 16, 144), (1, 1, 16, 0), (0, 1, 16, 64), (1, 0, 16, 64)):
        with pytest.raises(ValueError):
            attention_fp8.prepare_fp8_kv_cache(*bad)
    with pytest.raises(ValueError, match="CUDA"):
        attention_fp8.prepare_fp8_kv_cache(1, 1, 16, 64, device="cpu")


def test_cpu_tensors_are_refused():
    x, at = torch.zeros(1, 1, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    codes, scales = torch.zeros(1, 1, 16, 64, dtype=torch.uint8), torch.zeros(1, 1, dtype=torch.uint8)
    cache = {"keys": codes, "values": codes, "key_scales": scales, "value_scales": scales}
    with pytest.raises(ValueError, match="CUDA"):
        rotary.launch_rotary(x, at, {})
    with pytest.raises(ValueError, match="CUDA"):
        attention_fp8.launch_fp8_kv_append(cache, x, x, at[:, None], at)
    with pytest.raises(ValueError, match="CUDA"):
        attention_fp8.fp8_paged_attention(x, cache, at[:, None], at)
    for other in ({}, {"keys": codes}, [codes], None):
        with pytest.raises(TypeError):
            attention_fp8.fp8_paged_attention(x, other, at[:, None], at)


def views(**changes):
    cache = dict(keys=P, values=P, key_scales=P, value_scales=P, pages=8, kv_heads=2, page_tokens=16, head_dim=64)
    seq = dict(page_table=P, table_stride=4, table_pages=4, lengths=P, offsets=None, batch=3)
    cache.update({k: v for k, v in changes.items() if k in cache})
    seq.update({k: v for k, v in changes.items() if k in seq})
    return _lib.MamboKvCache(*cache.values()), _lib.MamboKvSequences(*seq.values())


BAD_VIEWS = [dict(keys=None), dict(values=None), dict(key_scales=None), dict(value_scales=None), dict(pages=0),
             dict(pages=1 << 31, kv_heads=2), dict(kv_heads=0), dict(kv_heads=1025), dict(page_tokens=8), dict(page_tokens=24),
             dict(head_dim=0), dict(head_dim=72), dict(head_dim=144), dict(keys=P + 8), dict(values=P + 1),
             dict(page_table=None), dict(table_stride=3), dict(table_pages=0), dict(lengths=None), dict(batch=0),
             dict(batch=4097), dict(batch=4), dict(page_table=P + 2), dict(lengths=P + 1), dict(offsets=P + 1)]


def test_append_refusals():
    lib, e = _lib.load(), _lib.MAMBO_EINVAL
    rope = _lib.MamboRotary(P, 64, 0, 1.0)

    def append(k=P, v=P, dtype=_lib.MAMBO_BF16, tokens=3, rotary=rope, **changes):
        cache, seq = views(**changes)
        return lib.mambo_kv_append(cache, k, 128, 64, v, 128, 64, dtype, tokens, seq, rotary, None)

    for bad in (*BAD_VIEWS, dict(k=None), dict(v=None), dict(dtype=5), dict(tokens=0), dict(tokens=(1 << 24) + 1),
                dict(k=P + 1), dict(v=P + 2, dtype=_lib.MAMBO_F32), dict(rotary=_lib.MamboRotary(None, 64, 0, 1.0)),
                dict(rotary=_lib.MamboRotary(P, 66, 0, 1.0)), dict(rotary=_lib.MamboRotary(P, 7, 0, 1.0)),
                dict(rotary=_lib.MamboRotary(P + 4, 64, 0, 1.0))):
        assert append(**bad) == e, bad
        assert _lib.last_error()
    assert lib.mambo_kv_append(None, P, 128, 64, P, 128, 64, 1, 3, views()[1], None, None) == e
    assert lib.mambo_kv_append(views()[0], P, 128, 64, P, 128, 64, 1, 3, None, None, None) == e


def test_rotary_refusals():
    lib, e = _lib.load(), _lib.MAMBO_EINVAL

    def turn(x=P, dtype=_lib.MAMBO_F32, tokens=4, heads=2, dim=64, positions=P, wide=0, turns=P, part=64, out=P):
        return lib.mambo_rotary(x, dtype, tokens, heads, dim, heads * dim, dim, positions, wide,
                                _lib.MamboRotary(turns, part, 0, 1.0), 0, out, heads * dim, dim, None)

    for bad in (dict(x=None), dict(out=None), dict(positions=None), dict(turns=None), dict(dtype=9), dict(tokens=0),
                dict(tokens=(1 << 24) + 1), dict(heads=0), dict(heads=1025), dict(dim=1, part=2), dict(dim=65537), dict(part=0),
                dict(part=66), dict(part=3), dict(x=P + 2), dict(out=P + 1), dict(positions=P + 2),
                dict(positions=P + 4, wide=1), dict(turns=P + 4), dict(tokens=1 << 24, heads=1024, dim=65536)):
        assert turn(**bad) == e, bad
        assert _lib.last_error()
    assert lib.mambo_rotary(P, 0, 4, 2, 64, 128, 64, P, 0, None, 0, P, 128, 64, None) == e


def test_attention_refusals():
    lib, e = _lib.load(), _lib.MAMBO_EINVAL
    need = lib.mambo_kv_attention_workspace_bytes(8, 2, 0)
    assert need > 0

    def attend(q=P, q_strides=(512, 64), tokens=3, heads=8, window=0, scale=0.125, out=P, out_strides=(512, 64), lse=None,
               workspace=P, size=need, **changes):
        cache, seq = views(**changes)
        return lib.mambo_kv_attention(q, *q_strides, tokens, heads, cache, seq, window, scale, out, *out_strides, lse, 8, 1,
                                      workspace, size, None)

    for bad in (*BAD_VIEWS, dict(q=None), dict(out=None), dict(heads=0), dict(heads=7), dict(heads=1026), dict(window=-1),
                dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(q=P + 8), dict(out=P + 2),
                dict(q_strides=(508, 64)), dict(q_strides=(512, 60)), dict(out_strides=(516, 64)), dict(out_strides=(512, 4)),
                dict(lse=P + 2), dict(workspace=P + 128), dict(table_pages=(1 << 24) + 1, table_stride=1 << 25),
                dict(tokens=1 << 24, heads=512, offsets=P, size=1 << 40),
                dict(table_pages=1 << 24, table_stride=1 << 24, page_tokens=128, batch=4000, tokens=4000)):
        assert attend(**bad) == e, bad
        assert _lib.last_error()
    assert attend(workspace=None) == _lib.MAMBO_EWORKSPACE and attend(size=need - 1) == _lib.MAMBO_EWORKSPACE
    assert attend(offsets=P) == _lib.MAMBO_EWORKSPACE  # queries of any number need room for the prompt form too


def test_workspace_sizes():
    lib = _lib.load()

    def size(*a):
        return lib.mambo_kv_attention_workspace_bytes(*a)

    assert size(0, 1, 0) == size(8, 0, 0) == size(7, 2, 0) == size(2048, 8, 0) == 0
    # More rows of a key head than the form for few takes: it always runs the other, and has no room for the first.
    assert size(64, 1, 0) == size(64, 1, 1)
    assert size(16, 1, 0) <= size(32, 1, 0) < size(32, 1, 1)  # two CTAs of 16 rows or one of 32
    assert size(8, 2, 0) == size(32, 8, 0)
