"""Attention over the paged FP8 cache against float64: single tokens, a few, prompts, chunks and mixtures of them.

The bounds of single values are kv_reference's. A result also has two independent roundings of at most 2^-8 (weights of
8 bits, bf16), each of 2^-8 / sqrt(3) of the norm at most, which add up in squares: 2^-8 * 0.82 over many values.
"""

from __future__ import annotations

import math

import pytest
import torch

from kv_reference import attention64, make_cache, make_table, starts, turned64
from mambo_b200 import _lib
from mambo_b200.kernels.attention_fp8 import fp8_paged_attention, launch_fp8_kv_append, prepare_fp8_kv_cache
from mambo_b200.kernels.rotary import launch_rotary, prepare_rotary_fields, rotary_frequencies

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert _lib.device_status()[0] == 0


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def check(got, lse, q, cache, table, lengths, offsets, window=0, scale=None):
    out, ref_lse, bound, lse_bound = attention64(q, cache, table, lengths, offsets, window, scale)
    nan = out.isnan()
    assert torch.equal(got.isnan(), nan)
    off = (got.double() - out).abs()
    assert (off <= bound)[~nan].all(), float((off / bound.clamp_min(1e-300))[~nan].max())
    if int((out != 0).sum()) >= 4096 and not nan.any():
        assert float(off.norm() / out.norm()) < 2.0 ** -8
    if lse is not None:
        empty = ref_lse == -math.inf
        assert torch.equal(lse == -math.inf, empty)
        ok = ~empty & ~ref_lse.isnan() & ~nan.any(dim=-1)
        assert ((lse.double() - ref_lse).abs() <= lse_bound)[ok].all(), float((lse.double() - ref_lse).abs()[ok].max())


def problem(page, kv, group, dim, lengths, counts, *, seed=0, spread=3, size=1.0):
    gen = torch.Generator().manual_seed(seed + page + dim + group)
    pages = sum(-(-n // page) for n in lengths) + 3
    cache = make_cache(gen, pages, kv, page, dim, "cuda", spread)
    table = make_table(gen, lengths, page, pages).cuda()
    q = (torch.randn(sum(counts), kv * group, dim, generator=gen) * size).to(BF16).cuda()
    return q, cache, table


def run(page, kv, group, dim, lengths, counts, window=0, scale=None, **kwargs):
    q, cache, table = problem(page, kv, group, dim, lengths, counts, **kwargs)
    offsets = None if counts == [1] * len(counts) else starts(counts)
    got, lse = fp8_paged_attention(q, cache, table, i32(lengths), offsets=None if offsets is None else i32(offsets),
                                   window=window, scale=scale, return_lse=True)
    check(got, lse, q, cache, table, lengths, offsets, window, scale)
    alone = fp8_paged_attention(q, cache, table, i32(lengths), offsets=None if offsets is None else i32(offsets),
                                window=window, scale=scale)
    assert torch.equal(alone.view(torch.int16), got.view(torch.int16))  # the same bits on every run


SINGLE = [  # page, key heads, group, dim, lengths, window
    (16, 1, 1, 16, [1], 0),
    (16, 1, 1, 128, [0], 0),
    (16, 2, 4, 64, [1, 0, 17, 16, 15, 128, 129], 0),
    (32, 8, 4, 128, [1000, 31, 32, 33, 0, 2500], 0),
    (64, 3, 7, 96, [500, 64, 65, 1], 0),
    (128, 2, 16, 112, [127, 128, 129, 4000], 0),
    (128, 1, 17, 80, [300, 1], 0),
    (64, 2, 32, 128, [777, 0, 12], 0),
    (16, 1, 33, 48, [200, 40, 0], 0),
    (32, 1, 64, 128, [3000], 0),
    (16, 4, 2, 32, [5000, 100, 1], 1),
    (64, 4, 8, 128, [5000, 100, 64, 0], 128),
    (128, 2, 40, 64, [900, 4], 129),
    (64, 1, 1, 144 - 16, [20000], 0),
    (16, 5, 3, 16, [333] * 40, 50),
]


@pytest.mark.parametrize("page,kv,group,dim,lengths,window", SINGLE)
def test_single_tokens(cuda_device, page, kv, group, dim, lengths, window):
    run(page, kv, group, dim, lengths, [1] * len(lengths), window)


RAGGED = [  # page, key heads, group, dim, lengths, tokens, window
    (16, 1, 1, 16, [1, 2], [0, 2], 0),
    (16, 2, 4, 64, [40, 9, 130], [4, 3, 0], 0),           # a few tokens each: the form for few rows
    (32, 2, 5, 128, [100, 6, 300], [6, 6, 1], 0),
    (64, 2, 4, 128, [500], [500], 0),                     # a prompt
    (64, 1, 1, 128, [513, 255, 256, 257], [513, 255, 256, 257], 0),
    (128, 2, 3, 80, [1000, 130, 700], [300, 130, 1], 0),  # a chunk, a prompt and a token
    (16, 3, 2, 48, [700, 33, 1, 0, 64], [129, 1, 1, 0, 64], 0),
    (32, 1, 40, 112, [300, 77], [20, 77], 0),
    (64, 2, 16, 64, [200, 1500, 31], [100, 1, 31], 17),
    (128, 1, 6, 96, [2000, 400], [700, 400], 300),
    (16, 1, 8, 128, [5000], [200], 1),
    (32, 1, 2, 32, [50, 60], [64, 90], 0),                # more queries than cached tokens: the first see nothing
    (64, 1, 4, 128, [3, 0], [300, 4], 0),
    (64, 8, 1, 128, [300] * 20, [30] * 20, 0),
]


@pytest.mark.parametrize("page,kv,group,dim,lengths,counts,window", RAGGED)
def test_ragged(cuda_device, page, kv, group, dim, lengths, counts, window):
    run(page, kv, group, dim, lengths, counts, window)


@pytest.mark.parametrize("counts", [[1, 1, 1], [60, 1, 200]])
@pytest.mark.parametrize("kwargs", [dict(scale=1.0, size=0.25), dict(scale=1e-9), dict(scale=0.3, size=3.0), dict(spread=40),
                                    dict(size=1e-20), dict(size=1e4, scale=1e-4)])
def test_scores_of_every_size(cuda_device, counts, kwargs):
    """From equal weights to one that takes all, pages whose scales are 2^80 apart, queries of any size."""
    run(32, 2, 4, 64, [300, 700, 200], counts, **kwargs)


@pytest.mark.parametrize("counts", [[1], [150]])
def test_scores_that_rise(cuda_device, counts):
    """Keys whose scores grow along the context by far more than the weights' range, up, down and at once."""
    gen = torch.Generator().manual_seed(1)
    n, page, dim = 1500, 32, 64
    for slope in (0.1, -0.1, 1.0):
        cache = prepare_fp8_kv_cache(48, 1, page, dim)
        k = torch.zeros(n, 1, dim)
        k[:, 0, 0] = torch.arange(n) * slope
        v = torch.randn(n, 1, dim, generator=gen)
        table = torch.randperm(48, generator=gen).int()[None].cuda()
        launch_fp8_kv_append(cache, k.cuda(), v.cuda(), table, i32([0]), offsets=i32([0, n]))
        q = torch.zeros(counts[0], 4, dim, dtype=BF16, device="cuda")
        q[..., 0] = 8.0
        offsets = starts(counts)
        got, lse = fp8_paged_attention(q, cache, table, i32([n]), offsets=i32(offsets), return_lse=True)
        check(got, lse, q, cache, table, [n], offsets)


@pytest.mark.parametrize("counts", [[1], [150]])
@pytest.mark.parametrize("jump", [9.0, 60.0, 100.0, 140.0, 190.0, 400.0, 1e5])
def test_one_score_far_above(cuda_device, jump, counts):
    """One key whose score is far above all before it, at each of the places that a thread takes together."""
    gen = torch.Generator().manual_seed(2)
    n, page, dim = 600, 64, 32
    k, v = (torch.randn(n, 1, dim, generator=gen) for _ in range(2))
    table = torch.randperm(10, generator=gen).int()[None].cuda()
    q = torch.randn(counts[0], 2, dim, generator=gen).to(BF16).cuda()
    q[..., 0] = 1.0
    for place in range(296, 312):
        k[:, 0, 0] = 0.0
        k[place, 0, 0] = jump * dim ** 0.5
        cache = prepare_fp8_kv_cache(10, 1, page, dim)
        launch_fp8_kv_append(cache, k.cuda(), v.cuda(), table, i32([0]), offsets=i32([0, n]))
        got, lse = fp8_paged_attention(q, cache, table, i32([n]), offsets=i32([0, counts[0]]), return_lse=True)
        check(got, lse, q, cache, table, [n], [0, counts[0]])


@pytest.mark.parametrize("counts", [[1], [150]])
def test_scores_near_the_ends_of_float32(cuda_device, counts):
    """All scores far below zero, one of them above the others; values of one, so that the weights' sum shows."""
    n, page, dim = 200, 16, 16
    k = torch.zeros(n, 1, dim)
    k[:, 0, 0] = -1e18
    k[130, 0, 0] = -0.5e18
    cache, table = prepare_fp8_kv_cache(13, 1, page, dim), torch.arange(13, dtype=torch.int32, device="cuda")[None]
    launch_fp8_kv_append(cache, k.cuda(), torch.ones(n, 1, dim, device="cuda"), table, i32([0]), offsets=i32([0, n]))
    q = torch.zeros(counts[0], 2, dim, dtype=BF16, device="cuda")
    q[..., 0] = 1e18
    got = fp8_paged_attention(q, cache, table, i32([n]), offsets=i32([0, counts[0]]), scale=1.0)
    assert (got == 1).all()


@pytest.mark.parametrize("counts", [[1, 1, 1], [40, 1, 200]])
@pytest.mark.parametrize("window", [0, 90])
def test_anything_in_masked_places(cuda_device, counts, window):
    """What no query sees may hold NaN codes and NaN scales: behind the lengths, before the window, in other pages."""
    lengths, page = [300, 70, 255], 32
    q, cache, table = problem(page, 2, 4, 64, lengths, counts)
    offsets = starts(counts)
    args = dict(offsets=i32(offsets) if counts[0] > 1 else None, window=window, return_lse=True)
    want, want_lse = fp8_paged_attention(q, cache, table, i32(lengths), **args)
    check(want, want_lse, q, cache, table, lengths, offsets, window)
    dirty = {n: torch.full_like(t, 0xFF if n.endswith("scales") else 0x7F) for n, t in cache.items()}
    for b, length in enumerate(lengths):
        low = max(0, length - counts[b] - window + 1) if window else 0
        for j in range(length):
            at = int(table[b, j // page])
            if j >= low:
                for n in ("keys", "values"):
                    dirty[n][at, :, j % page] = cache[n][at, :, j % page]
                for n in ("key_scales", "value_scales"):
                    dirty[n][at] = cache[n][at]
    got, lse = fp8_paged_attention(q, dirty, table, i32(lengths), **args)
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    # Columns behind the sequences' pages are not looked at.
    wide = torch.cat([table, torch.full_like(table, 1 << 30)], dim=1)
    assert torch.equal(fp8_paged_attention(q, dirty, wide, i32(lengths), **args)[0], want)


@pytest.mark.parametrize("counts", [[1, 1], [100, 70]])
def test_not_finite(cuda_device, counts):
    """A NaN or infinite query has NaN results, as has a query that sees a NaN page; all others are as without them."""
    lengths, page = [200, 90], 16
    q, cache, table = problem(page, 2, 4, 64, lengths, counts)
    offsets = starts(counts)
    off = i32(offsets) if counts[0] > 1 else None
    clean = fp8_paged_attention(q, cache, table, i32(lengths), offsets=off)
    q[0, 3, 7], q[1, 6, 0] = math.nan, math.inf
    got = fp8_paged_attention(q, cache, table, i32(lengths), offsets=off)
    assert got[0, 3].isnan().all() and got[1, 6].isnan().all()
    got[0, 3], got[1, 6] = clean[0, 3], clean[1, 6]
    assert torch.equal(got, clean)
    q[0, 3, 7], q[1, 6, 0] = 0.5, 0.5
    cache["key_scales"][int(table[0, 160 // page]), 1] = 255    # seen by the first sequence's queries from 160 on
    cache["value_scales"][int(table[1, 80 // page]), 0] = 255
    got, lse = fp8_paged_attention(q, cache, table, i32(lengths), offsets=off, return_lse=True)
    check(got, lse, q, cache, table, lengths, offsets)
    assert got.isnan().any() and not got.isnan().all()


@pytest.mark.parametrize("counts", [[1, 1, 1], [50, 40, 90]])
def test_pages_outside_the_cache(cuda_device, counts):
    """Positions of a page outside the cache do not exist; lengths are clamped to the table."""
    lengths, page = [200, 90, 100], 16
    q, cache, table = problem(page, 2, 2, 32, lengths, counts)
    table[0, 3], table[0, 12], table[1, :], table[2, 0] = -1, cache["keys"].shape[0], (1 << 31) - 1, -(1 << 31)
    offsets = starts(counts)
    off = i32(offsets) if counts[0] > 1 else None
    got, lse = fp8_paged_attention(q, cache, table, i32(lengths), offsets=off, return_lse=True)
    check(got, lse, q, cache, table, lengths, offsets)
    assert not got[offsets[1]:offsets[2]].any() and (lse[offsets[1]:offsets[2]] == -math.inf).all()
    lies = [1000, -5, 1 << 30]
    got, lse = fp8_paged_attention(q, cache, table, i32(lies), offsets=off, return_lse=True)
    check(got, lse, q, cache, table, lies, offsets)


def test_rows_behind_the_last_sequence(cuda_device):
    """Tokens that no sequence has keep what out holds, offsets that lie stay within the call."""
    q, cache, table = problem(16, 2, 4, 64, [100, 50], [30, 3])
    padded = torch.cat([q, torch.full_like(q[:20], math.nan)])
    out = torch.full_like(padded, 7.0)
    got = fp8_paged_attention(padded, cache, table, i32([100, 50]), offsets=i32([0, 30, 33]), out=out)
    assert got is out and (out[33:] == 7).all()
    check(out[:33], None, q, cache, table, [100, 50], [0, 30, 33])
    out.fill_(7.0)
    fp8_paged_attention(padded, cache, table, i32([100, 50]), offsets=i32([33, 33, 33]), out=out)
    fp8_paged_attention(padded, cache, table, i32([100, 50]), offsets=i32([40, 20, -3]), out=out)
    assert (out == 7).all()
    fp8_paged_attention(q, cache, table, i32([100, 50]), offsets=i32([-9, 30, 1 << 30]), out=out[:33])
    check(out[:33], None, q, cache, table, [100, 50], [0, 30, 33])


@pytest.mark.parametrize("counts", [[1, 1], [90, 1]])
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_strides_and_alignment(cuda_device, offset, counts):
    """Queries and results as views of larger rows, aligned or not, transposed ones, and results in the queries' place."""
    kv, group, dim, lengths = 2, 4, 80, [300, 33]
    q, cache, table = problem(64, kv, group, dim, lengths, counts)
    offsets, tokens, heads = starts(counts), sum(counts), kv * group
    off = i32(offsets) if counts[0] > 1 else None
    want = fp8_paged_attention(q, cache, table, i32(lengths), offsets=off)
    check(want, None, q, cache, table, lengths, offsets)
    base = torch.randn(tokens, offset + (heads + 3) * dim, dtype=BF16, device="cuda")
    view = base.as_strided((tokens, heads, dim), (base.shape[1], dim, 1), offset)
    view.copy_(q)
    held = base.clone()
    out = held.as_strided((tokens, heads, dim), (base.shape[1], dim, 1), offset)
    assert fp8_paged_attention(view, cache, table, i32(lengths), offsets=off, out=out) is out
    assert torch.equal(out, want)
    out.copy_(view)
    assert torch.equal(held, base)
    for other in (view.transpose(0, 1).contiguous().transpose(0, 1), view.transpose(1, 2).contiguous().transpose(1, 2)):
        assert torch.equal(fp8_paged_attention(other, cache, table, i32(lengths), offsets=off), want)
        out = torch.empty_like(other)
        assert torch.equal(fp8_paged_attention(q, cache, table, i32(lengths), offsets=off, out=out), want)
    fp8_paged_attention(view, cache, table, i32(lengths), offsets=off, out=view)
    assert torch.equal(view, want)
    strided = torch.stack([table, table], dim=2)[:, :, 0]
    assert torch.equal(fp8_paged_attention(q, cache, strided, torch.stack([i32(lengths)] * 2, 1)[:, 0], offsets=off), want)


def test_offsets_past_32_bits(cuda_device):
    """A cache of 2^32 bytes and more each for keys and values: its last pages are as good as its first."""
    pages, kv, page, dim = (1 << 18) + 40, 2, 64, 128
    cache = prepare_fp8_kv_cache(pages, kv, page, dim)
    assert cache["keys"].numel() > 1 << 32
    order = [pages - 1, 0, pages - 2, 1 << 17, (1 << 17) - 1]
    table, n = i32([order]), 300
    k, v = (torch.randn(n, kv, dim, dtype=BF16, device="cuda") for _ in range(2))
    launch_fp8_kv_append(cache, k, v, table, i32([0]), offsets=i32([0, n]))
    small = {name: t[order].contiguous() for name, t in cache.items()}
    want = prepare_fp8_kv_cache(5, kv, page, dim)
    launch_fp8_kv_append(want, k, v, i32([[0, 1, 2, 3, 4]]), i32([0]), offsets=i32([0, n]))
    assert all(torch.equal(small[name], want[name]) for name in want)
    for tokens in (1, 300):
        q = torch.randn(tokens, 8, dim, dtype=BF16, device="cuda")
        got = fp8_paged_attention(q, cache, table, i32([n]), offsets=i32([0, tokens]))
        assert torch.equal(got, fp8_paged_attention(q, small, i32([[0, 1, 2, 3, 4]]), i32([n]), offsets=i32([0, tokens])))
        check(got, None, q, small, i32([[0, 1, 2, 3, 4]]), [n], [0, tokens])


def test_most_sequences(cuda_device):
    """4096 sequences, most of them empty or short, of one token and of several."""
    lengths = [(i * 37) % 90 if i % 3 else 0 for i in range(4096)]
    q, cache, table = problem(16, 1, 2, 16, lengths, [1] * 4096)
    got, lse = fp8_paged_attention(q, cache, table, i32(lengths), return_lse=True)
    check(got, lse, q, cache, table, lengths, None)
    counts = [0 if i % 5 else 40 if i % 2 else 2 for i in range(4096)]
    q = torch.randn(sum(counts), 2, 16, device="cuda").to(BF16)
    got, lse = fp8_paged_attention(q, cache, table, i32(lengths), offsets=i32(starts(counts)), return_lse=True)
    check(got, lse, q, cache, table, lengths, starts(counts))


def test_joined_parts_of_a_context(cuda_device):
    """Results over two parts of a context and their logarithms give the whole's."""
    n, cut = 1000, 512
    q, cache, table = problem(64, 2, 4, 128, [n], [1])
    whole, lse = fp8_paged_attention(q, cache, table, i32([n]), return_lse=True)
    parts = [fp8_paged_attention(q, cache, t.contiguous(), i32([m]), return_lse=True)
             for t, m in ((table[:, :cut // 64], cut), (table[:, cut // 64:], n - cut))]
    joined = torch.logaddexp(parts[0][1], parts[1][1])
    # each logarithm is off by its bound; results by 2^-8 (bf16) and 2^-8 (weights) of what they sum, and so is the whole
    assert (joined - lse).abs().max() < 2.0 ** -14
    out = sum(o.float() * (l - joined).exp()[..., None] for o, l in parts)
    bound = attention64(q, cache, table, [n])[2]
    assert ((out - whole).double().abs() <= 3 * bound + 2.0 ** -8 * sum(o.abs() for o, _ in parts).double()).all()


def test_several_streams(cuda_device):
    """Calls on several streams at once, each with its own workspace."""
    problems = [problem(32, 2, 4, 64, [1500 + 100 * i, 20], [1, 1] if i % 2 else [200, 1], seed=i) for i in range(4)]
    calls = [dict(offsets=None if i % 2 else i32([0, 200, 201])) for i in range(4)]
    want = [fp8_paged_attention(q, c, t, i32([1500 + 100 * i, 20]), **a) for i, ((q, c, t), a) in enumerate(zip(problems, calls))]
    lengths = [i32([1500 + 100 * i, 20]) for i in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(5):
        got = [fp8_paged_attention(q, c, t, n, stream=s, **a)
               for (q, c, t), n, s, a in zip(problems, lengths, streams, calls)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("captured", [False, True])
def test_steps_together(cuda_device, captured):
    """Prompts, then decode steps: queries turned, keys and values appended, attention, all from the projection's output.

    The decode step is also captured once and replayed with other data, lengths and tables.
    """
    gen = torch.Generator().manual_seed(21)
    heads, kv, dim, page, pages, batch = 8, 2, 64, 16, 64, 3
    rope, radians = prepare_rotary_fields(dim, base=500000.0), rotary_frequencies(dim, base=500000.0)[0]
    cache, lengths = prepare_fp8_kv_cache(pages, kv, page, dim), [0, 0, 0]
    table = torch.randperm(pages, generator=gen).int()[:batch * 20].view(batch, 20).cuda()
    held = i32(lengths)

    def step(qkv, counts, offsets):
        q, k, v = qkv.split([heads * dim, kv * dim, kv * dim], dim=1)
        positions = torch.cat([held[b] + torch.arange(n, device="cuda", dtype=torch.int32) for b, n in enumerate(counts)])
        q = launch_rotary(q.view(-1, heads, dim), positions, rope)
        launch_fp8_kv_append(cache, k.view(-1, kv, dim), v.view(-1, kv, dim), table, held, offsets=offsets, rope=rope)
        held.add_(new)
        return q, fp8_paged_attention(q, cache, table, held, offsets=offsets)

    def verify(q, out, qkv, counts):
        """The queries against float64; the result against attention over the cache as it is, which the append's tests check."""
        at = torch.tensor([p + i for p, n in zip(lengths, counts) for i in range(n)])
        ref = turned64(qkv[:, :heads * dim].view(-1, heads, dim), at, radians)
        assert ((q.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -18 * float(qkv.abs().max())).all()
        for b, n in enumerate(counts):
            lengths[b] += n
        check(out, None, q, cache, table, lengths, starts(counts))
        # and the cached values against the projection's: half a step of E4M3 of the page's largest at most
        v = qkv[:, (heads + kv) * dim:].view(-1, kv, dim).double()
        cached = cache["values"].view(torch.float8_e4m3fn).double() * torch.exp2(cache["value_scales"].double() - 127)[..., None, None]
        at = at.cuda()
        seq = torch.repeat_interleave(torch.arange(batch), torch.tensor(counts)).cuda()
        rows = cached[table[seq, at // page].long(), :, at % page]
        assert ((rows - v).abs() <= 2.0 ** -4 * v.abs() + 2.0 ** -10 * 2.0 ** -6 * float(v.abs().max())).all()

    counts = [70, 3, 20]
    new = i32(counts)
    qkv = torch.randn(sum(counts), (heads + 2 * kv) * dim, generator=gen).to(BF16).cuda()
    q, out = step(qkv, counts, i32(starts(counts)))
    verify(q, out, qkv, counts)
    counts, new = [1] * batch, i32([1] * batch)
    qkv = torch.randn(batch, (heads + 2 * kv) * dim, generator=gen).to(BF16).cuda()
    if captured:
        before, side = {n: t.clone() for n, t in cache.items()}, torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(qkv, counts, None)  # the stream's workspace
            held.sub_(new)
            for n, t in before.items():
                cache[n].copy_(t)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            q, out = step(qkv, counts, None)
    for i in range(6):
        qkv.copy_(torch.randn(qkv.shape, generator=gen))
        if captured:
            graph.replay()
        else:
            q, out = step(qkv, counts, None)
        verify(q, out, qkv, counts)
        if i == 2:  # another page table: the sequences' pages move
            moved = torch.randperm(pages, generator=gen).cuda()
            for t in cache.values():
                t.copy_(t.clone()[torch.argsort(moved)])
            table.copy_(moved[table.long()].int())


def test_graphs_that_share_a_workspace(cuda_device):
    """Two captured calls and an eager one of the same stream, replayed in any order."""
    problems = [problem(32, 2, 4, 64, [3000, 200], c, seed=s) for s, c in ((1, [1, 1]), (2, [300, 1]))]
    args = [(q, c, t, i32([3000, 200])) for q, c, t in problems]
    off, side = [None, i32([0, 300, 301])], torch.cuda.Stream()
    want = [fp8_paged_attention(*a, offsets=o) for a, o in zip(args, off)]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for a, o in zip(args, off):
            fp8_paged_attention(*a, offsets=o)
        graphs, got = [], []
        for a, o in zip(args, off):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=side):
                got.append(fp8_paged_attention(*a, offsets=o))
        for order in ((0, 1), (1, 1), (1, 0), (0, 0)):
            for i in order:
                got[i].zero_()
                graphs[i].replay()
                assert torch.equal(fp8_paged_attention(*args[1 - i], offsets=off[1 - i]), want[1 - i])
                assert torch.equal(got[i], want[i])


def test_example_layer(cuda_device):
    """A chunk at a time or all at once, a layer's last token sees the same context."""
    import sys
    from pathlib import Path

    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    from fp8_attention_layer import AttentionLayer

    x = torch.randn(2 * 40, 256, dtype=BF16, device="cuda")
    outs = []
    for cuts in ([40], [17, 22, 1]):
        layer, at = AttentionLayer(256, 4, 2, 64, batch=2, most=64, page=16), 0
        for n in cuts:
            rows = torch.cat([x[at:at + n], x[40 + at:40 + at + n]])
            positions = torch.arange(at, at + n, device="cuda").repeat(2)
            out = layer(rows, positions, i32([0, n, 2 * n]) if n > 1 else None)
            at += n
        assert layer.lengths.tolist() == [40, 40] and out.isfinite().all()
        outs.append(out)
    assert outs[0].shape == (80, 256) and outs[1].shape == (2, 256)


def test_refusals(cuda_device):
    cache = prepare_fp8_kv_cache(4, 2, 16, 64)
    q, table, lengths = torch.zeros(2, 4, 64, dtype=BF16, device="cuda"), i32([[0], [1]]), i32([1, 1])

    def refused(error=ValueError, q=q, cache=cache, table=table, lengths=lengths, **kwargs):
        with pytest.raises(error):
            fp8_paged_attention(q, cache, table, lengths, **kwargs)

    refused(q=q.float())
    refused(q=q[..., :32])
    refused(q=q[0])
    refused(q=q[:, :3])
    refused(q=q[:, :0])
    refused(q=q[:1])
    refused(window=-1)
    refused(table=table.long())
    refused(lengths=lengths[:1])
    refused(lengths=lengths.cpu())
    refused(offsets=i32([0, 2]))
    refused(offsets=i32([0, 1, 2]).long())
    refused(out=q[:1])
    refused(out=q.float())
    for scale in (0.0, -1.0, math.nan, math.inf):
        refused(scale=scale)
    refused(cache={**cache, "keys": cache["keys"][:2]})
    refused(TypeError, cache={"keys": cache["keys"]})
    out, lse = fp8_paged_attention(q[:0], cache, table, lengths, offsets=i32([0, 0, 0]), return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
