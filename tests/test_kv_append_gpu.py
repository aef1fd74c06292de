"""The append of keys and values to the paged FP8 cache against float64.

Values are rounded once, so codes and scales of values have to be equal; so have older codes that a growing scale rounds
anew. Keys are turned in float32 first: a key may be off by half a step of E4M3 and the rotation's bound, and its page's
scale is compared through the unrounded values that it was derived from.
"""

from __future__ import annotations

import math

import pytest
import torch

from kv_reference import append64, make_cache, make_table, starts, turned64, turned_bound
from mambo_b200 import _lib
from mambo_b200.kernels.attention_fp8 import launch_fp8_kv_append, prepare_fp8_kv_cache
from mambo_b200.kernels.rotary import prepare_rotary_fields, rotary_frequencies

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert _lib.device_status()[0] == 0


def numbers(codes):
    return codes.view(torch.float8_e4m3fn).double().cpu()


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def positions_of(lengths, counts):
    return torch.tensor([p + i for p, n in zip(lengths, counts) for i in range(n)])


def check_append(cache, before, k, v, table, lengths, counts, *, rotary=0, interleaved=False, magnitude=1.0):
    """The cache after an append, against what it was ``before`` and the call's arguments."""
    offsets, rows = starts(counts), table.tolist()
    old = {n: (numbers(before[n]), before[n[:-1] + "_scales"].int().cpu() - 127) for n in ("keys", "values")}
    values, exps, _ = append64(*old["values"], v.double().cpu(), rows, lengths, offsets)
    assert torch.equal(cache["value_scales"].int().cpu() - 127, exps)
    assert torch.equal(numbers(cache["values"]), values)
    x, bound = k.double().cpu(), torch.zeros(k.shape, dtype=torch.float64)
    if rotary:
        half = turned_bound(x, rotary, magnitude, interleaved)
        bound[..., :rotary] = half.repeat_interleave(2, dim=-1) if interleaved else torch.cat([half, half], dim=-1)
        x = turned64(x, positions_of(lengths, counts), rotary_frequencies(rotary)[0], interleaved=interleaved, magnitude=magnitude)
    keys, exps, unrounded = append64(*old["keys"], x, rows, lengths, offsets)
    assert torch.equal(cache["key_scales"].int().cpu() - 127, exps)
    got, new = numbers(cache["keys"]), ~unrounded.isnan()
    assert torch.equal(got[~new], keys[~new])
    if not rotary:
        assert torch.equal(got, keys)
        return
    # Half a step (2^-4 of the value, 2^-10 where it is small) and the rotation's error in units of the scale: both of a
    # pair's values are at most its |a| + |b|, whose largest over the call stands for all.
    near = float(bound.max()) * torch.exp2(-exps.double())[:, :, None, None]
    off = (got - unrounded.clamp(-448, 448)).abs()
    half_step = torch.exp2(torch.floor(torch.log2(unrounded.abs().clamp_min(2.0 ** -6))) - 4)
    assert (off <= half_step + 2 * near)[new].all()
    assert (got != keys)[new].double().mean() < 1e-3


CASES = [  # page, heads, dim, lengths before, new tokens, rotary, interleaved
    (16, 1, 16, [0], [1], 0, False),
    (16, 2, 64, [0, 5, 16, 31], [1, 1, 1, 1], 64, False),
    (32, 3, 128, [0, 1, 31, 32, 33, 500], [1, 32, 1, 33, 64, 7], 128, False),
    (64, 8, 128, [100, 0, 63], [64, 200, 1], 128, True),
    (128, 5, 80, [0, 127, 128, 300], [129, 2, 128, 0], 40, True),
    (128, 1, 112, [7], [1000], 112, False),
    (16, 40, 48, [3, 0], [14, 15], 16, False),
    (64, 2, 96, [10, 20, 30], [0, 0, 5], 6, False),
    (32, 4, 32, [0, 0, 0], [3, 0, 70], 32, True),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page,heads,dim,lengths,counts,rotary,interleaved", CASES)
def test_against_float64(cuda_device, page, heads, dim, lengths, counts, rotary, interleaved, dtype):
    gen = torch.Generator().manual_seed(page + dim)
    totals = [p + n for p, n in zip(lengths, counts)]
    pages = sum(-(-n // page) for n in totals) + 5
    cache = make_cache(gen, pages, heads, page, dim, "cuda")
    table = make_table(gen, totals, page, pages)
    k, v = ((torch.randn(sum(counts), heads, dim, generator=gen) * torch.exp2(torch.randint(-9, 10, (heads, 1), generator=gen)))
            .to(dtype) for _ in range(2))
    before = {n: t.clone() for n, t in cache.items()}
    rope = prepare_rotary_fields(rotary, interleaved=interleaved, magnitude=1.25) if rotary else None
    offsets = None if counts == [1] * len(counts) else i32(starts(counts))
    assert launch_fp8_kv_append(cache, k.cuda(), v.cuda(), table.cuda(), i32(lengths), offsets=offsets, rope=rope) is None
    check_append(cache, before, k, v, table, lengths, counts, rotary=rotary, interleaved=interleaved, magnitude=1.25)


def test_token_by_token(cuda_device):
    """A page filled by single tokens that grow and shrink: its scale grows with them and older codes are rounded anew."""
    gen = torch.Generator().manual_seed(3)
    cache, table = prepare_fp8_kv_cache(6, 2, 16, 32), torch.tensor([[4, 1], [0, 5]], dtype=torch.int32)
    for step in range(20):
        size = 2.0 ** torch.randint(-12, 13, (2, 2, 1), generator=gen)
        k, v = (torch.randn(2, 2, 32, generator=gen) * size for _ in range(2))
        before = {n: t.clone() for n, t in cache.items()}
        lengths = [step, step + 3]
        launch_fp8_kv_append(cache, k.cuda(), v.cuda(), table.cuda(), i32(lengths))
        check_append(cache, before, k, v, table, lengths, [1, 1])


def test_one_call_equals_single_tokens_where_the_scale_stays(cuda_device):
    """With the largest value first, a chunk and its tokens one by one leave the same cache."""
    gen = torch.Generator().manual_seed(5)
    k, v = (torch.randn(100, 3, 64, generator=gen).clamp(-3, 3).bfloat16().cuda() for _ in range(2))
    k[::32, :, 0] = v[::32, :, 0] = 7.0
    table = torch.tensor([[2, 0, 3, 1]], dtype=torch.int32, device="cuda")
    one, many = prepare_fp8_kv_cache(4, 3, 32, 64), prepare_fp8_kv_cache(4, 3, 32, 64)
    launch_fp8_kv_append(one, k, v, table, i32([0]), offsets=i32([0, 100]))
    for t in range(100):
        launch_fp8_kv_append(many, k[t:t + 1], v[t:t + 1], table, i32([t]))
    assert all(torch.equal(one[n], many[n]) for n in one)


def test_extreme_values(cuda_device):
    """Zeros, the smallest and largest numbers, and values just below and above a scale's largest."""
    cache, table = prepare_fp8_kv_cache(9, 1, 16, 16), torch.arange(9, dtype=torch.int32)[:, None]
    x = torch.zeros(9, 1, 16)
    tiny, huge = 2.0 ** -149, 3.4028234663852886e38
    for i, value in enumerate([0.0, tiny, huge, 448.0, 448.0000305, 2.0 ** -64, 449 * 2.0 ** -64, -1.17e-38, -huge]):
        x[i, 0, 3] = value
        x[i, 0, 4] = -value / 3
    before = {n: t.clone() for n, t in cache.items()}
    launch_fp8_kv_append(cache, x.cuda(), x.cuda(), table.cuda(), i32([0] * 9))
    check_append(cache, before, x, x, table, [0] * 9, [1] * 9)


def test_not_finite(cuda_device):
    """A page of a head that gets NaN or infinity has scale 255 until it is begun again; others are as without it."""
    gen = torch.Generator().manual_seed(7)
    k, v = (torch.randn(40, 2, 32, generator=gen).cuda() for _ in range(2))
    table, offsets = torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda"), i32([0, 40])
    clean, cache = prepare_fp8_kv_cache(3, 2, 16, 32), prepare_fp8_kv_cache(3, 2, 16, 32)
    launch_fp8_kv_append(clean, k, v, table, i32([0]), offsets=offsets)
    k2, v2 = k.clone(), v.clone()
    k2[3, 1, 5], v2[20, 0, 0] = math.inf, math.nan
    launch_fp8_kv_append(cache, k2, v2, table, i32([0]), offsets=offsets)
    assert cache["key_scales"][0, 1] == 255 and cache["value_scales"][1, 0] == 255
    for name, at in (("key", (0, 1)), ("value", (1, 0))):
        same = torch.ones(3, 2, dtype=torch.bool, device="cuda")
        same[at] = False
        assert torch.equal(cache[name + "_scales"][same], clean[name + "_scales"][same])
        assert torch.equal(cache[name + "s"][same], clean[name + "s"][same])
    launch_fp8_kv_append(cache, k[:1], v[:1], table, i32([40]))  # another page: stays
    assert cache["key_scales"][0, 1] == 255
    launch_fp8_kv_append(cache, k[:1], v[:1], table, i32([15]))  # the same page: stays NaN
    assert cache["key_scales"][0, 1] == 255
    launch_fp8_kv_append(cache, k, v, table, i32([0]), offsets=offsets)
    assert all(torch.equal(cache[n][:2], clean[n][:2]) for n in clean)


def test_tokens_without_a_page(cuda_device):
    """Entries outside the cache and columns behind the table drop their tokens; lengths and offsets that lie are clamped."""
    gen = torch.Generator().manual_seed(9)
    cache = make_cache(gen, 8, 2, 16, 32, "cuda")
    before = {n: t.clone() for n, t in cache.items()}
    table = torch.tensor([[0, -1, 1], [2, 8, 3], [(1 << 31) - 1, -(1 << 31), 4]], dtype=torch.int32)
    lengths, counts = [0, 10, 20], [60, 38, 40]  # 48 tokens fit
    k, v = (torch.randn(138, 2, 32, generator=gen) for _ in range(2))
    launch_fp8_kv_append(cache, k.cuda(), v.cuda(), table.cuda(), i32(lengths), offsets=i32(starts(counts)))
    check_append(cache, before, k, v, table, lengths, counts)
    before = {n: t.clone() for n, t in cache.items()}
    launch_fp8_kv_append(cache, k[:3].cuda(), v[:3].cuda(), table.cuda(), i32([48, 1000, (1 << 31) - 1]))
    launch_fp8_kv_append(cache, k[:3].cuda(), v[:3].cuda(), table.cuda(), i32([5, 5, 5]), offsets=i32([3, 3, 3, 3]))
    launch_fp8_kv_append(cache, k[:3].cuda(), v[:3].cuda(), table.cuda(), i32([5, 5, 5]), offsets=i32([9, 7, 5, 1 << 30]))
    launch_fp8_kv_append(cache, k[:0].cuda(), v[:0].cuda(), table.cuda(), i32([5, 5, 5]), offsets=i32([0, 0, 0, 0]))
    assert all(torch.equal(cache[n], before[n]) for n in cache)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_strides_and_alignment(cuda_device, offset, dtype):
    """Keys and values as views of a projection's output, anywhere in it, tables with strides, and tokens behind the last."""
    gen = torch.Generator().manual_seed(11)
    heads, dim, lengths, counts = 3, 64, [5, 30, 0], [20, 1, 40]
    base = torch.randn(70, offset + 8 * heads * dim, generator=gen).to(dtype).cuda()
    k = base.as_strided((70, heads, dim), (base.shape[1], dim, 1), offset + dim)
    v = base.as_strided((70, heads, dim), (base.shape[1], dim, 1), offset + 4 * dim)
    cache = make_cache(gen, 12, heads, 16, dim, "cuda")
    table = make_table(gen, [p + n for p, n in zip(lengths, counts)], 16, 12)
    rope = prepare_rotary_fields(dim)
    wide = torch.stack([table, table + 1], dim=2).cuda()
    for tables in (table.cuda(), wide[:, :, 0], torch.cat([table, table], dim=1).cuda()[:, :table.shape[1]]):
        for kk, vv in ((k, v), (k.transpose(0, 1).contiguous().transpose(0, 1), v.transpose(1, 2).contiguous().transpose(1, 2))):
            mine = {n: t.clone() for n, t in cache.items()}
            launch_fp8_kv_append(mine, kk, vv, tables, torch.stack([i32(lengths)] * 2, 1)[:, 0], offsets=i32(starts(counts)),
                                 rope=rope)
            check_append(mine, cache, k[:61].cpu(), v[:61].cpu(), table, lengths, counts, rotary=dim)


def test_many_sequences(cuda_device):
    gen = torch.Generator().manual_seed(13)
    batch = 4096
    lengths = torch.randint(0, 16, (batch,), generator=gen).tolist()
    table = torch.randperm(batch, generator=gen).int()[:, None]
    cache = make_cache(gen, batch, 1, 16, 16, "cuda")
    before = {n: t.clone() for n, t in cache.items()}
    k, v = (torch.randn(batch, 1, 16, generator=gen) for _ in range(2))
    launch_fp8_kv_append(cache, k.cuda(), v.cuda(), table.cuda(), i32(lengths))
    check_append(cache, before, k, v, table, lengths, [1] * batch)


def test_refusals(cuda_device):
    cache = prepare_fp8_kv_cache(4, 2, 16, 64)
    assert cache["keys"].shape == (4, 2, 16, 64) and int(cache["keys"].sum()) == 0 and (cache["key_scales"] == 63).all()
    k, table, lengths = torch.zeros(2, 2, 64, dtype=BF16, device="cuda"), i32([[0], [1]]), i32([0, 0])
    rope = prepare_rotary_fields(64)

    def refused(error=ValueError, cache=cache, k=k, v=k, table=table, lengths=lengths, **kwargs):
        with pytest.raises(error):
            launch_fp8_kv_append(cache, k, v, table, lengths, **kwargs)

    refused(k=k.half(), v=k.half())
    refused(k=k[:, :1], v=k[:, :1])
    refused(k=k[..., :32], v=k[..., :32])
    refused(k=k[0], v=k[0])
    refused(v=k.float())
    refused(v=k[:1])
    refused(k=k[:1], v=k[:1])  # without offsets a token for each sequence
    refused(table=table.long())
    refused(table=table[:, 0])
    refused(table=table[:, :0])
    refused(table=table.cpu())
    refused(lengths=lengths.long())
    refused(lengths=lengths[:1])
    refused(offsets=i32([0, 2]))
    refused(offsets=i32([0, 1, 2]).long())
    refused(rope=prepare_rotary_fields(128))
    refused(TypeError, rope={"turns": rope["turns"]})
    refused(TypeError, cache={n: t for n, t in cache.items() if n != "values"})
    for name, other in (("keys", cache["keys"][:2]), ("values", cache["values"].view(torch.int8)), ("key_scales", cache["key_scales"].T),
                        ("value_scales", cache["value_scales"].cpu()), ("keys", cache["keys"].transpose(0, 1))):
        refused(cache={**cache, name: other})
    many = k.new_zeros(4097, 2, 64)
    refused(k=many, v=many, table=table[:1].expand(4097, 1), lengths=i32([0] * 4097))
