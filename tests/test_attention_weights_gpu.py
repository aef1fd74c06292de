"""Attention in which many small weights add up: beside one position that has much of the mass, and in pages of small values.

The bound is on the sum of what the weights are off by, against the weights' sum, not on each of them against the largest.
With w a weight times its position's value scale and W the row's largest, a kernel may be off by

    2^-10 w + 2^-24 W      for each position:

a weight's rounding to f16 (2^-11 w, or 2^-25 W for the smallest), its terms of 8 bits (2^-12 w, or 2^-24 W), the float32
argument and exponential (2^-14 w). Sums in float32, on the tensor core and of the weights: 2^-12 of the products' sum, a
step of 2^-23 for each of up to 2048 products of 32 positions. Scores: the queries' values below 2^-18 of their largest
and a float32 sum, as the other tests have it. The result's rounding to bf16: 2^-8.
"""

from __future__ import annotations

import math

import pytest
import torch

from mambo_b200 import _lib
from mambo_b200.kernels.attention_fp8 import fp8_paged_attention

pytestmark = pytest.mark.gpu

PAGE, FORMS = 64, [  # key heads, group, head size, queries of a sequence
    pytest.param(8, 4, 128, 1, id="16 rows, group 4"),
    pytest.param(8, 16, 64, 1, id="16 rows, group 16"),
    pytest.param(8, 20, 128, 1, id="32 rows, group 20"),
    pytest.param(8, 2, 64, 5, id="16 rows, 5 tokens"),
    pytest.param(4, 8, 128, 40, id="many rows"),
    pytest.param(2, 40, 64, 1, id="many rows, group 40"),
]


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert _lib.device_status()[0] == 0


def quantized(x, page):
    """x [H,N,D] as cache pages [N/page,H,page,D] of codes and scale codes [N/page,H]."""
    h, n, d = x.shape
    x = x.view(h, n // page, page, d).transpose(0, 1)
    top = x.abs().amax(dim=(2, 3)).clamp_min(2.0 ** -60)
    e = torch.ceil(torch.log2(top / 448.0)).clamp(-64, 127)
    codes = (x * torch.exp2(-e)[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8).contiguous()
    return codes, (e + 127).to(torch.uint8).contiguous()


def dequantized(codes, scales):
    x = codes.view(torch.float8_e4m3fn).double() * torch.exp2(scales.double() - 127)[..., None, None]
    return x.transpose(0, 1).reshape(codes.shape[1], -1, codes.shape[3])


def exact(q, k, v, scales):
    """q [n,H*g,D] at the last n positions of k and v [H,N,D]: results, and how far a kernel may be off."""
    (n, heads, dim), (kv, length, _) = q.shape, k.shape
    qs = q.double().view(n, kv, heads // kv, dim)
    s = torch.einsum("nhgd,hjd->nhgj", qs, k) * dim ** -0.5
    seen = torch.arange(length, device=q.device)[None] <= length - n + torch.arange(n, device=q.device)[:, None]
    s = torch.where(seen[:, None, None], s, torch.full_like(s, -math.inf))
    p = torch.softmax(s, dim=-1)
    o = torch.einsum("nhgj,hjd->nhgd", p, v)
    factor = torch.exp2(scales.double() - 127).T.repeat_interleave(PAGE, dim=1)  # [H, N]
    codes, w = v.abs() / factor[..., None], p * factor[None, :, None]
    off = torch.where(seen[:, None, None], 2.0 ** -10 * w + 2.0 ** -24 * w.amax(dim=-1, keepdim=True), torch.zeros_like(w))
    mass = torch.einsum("nhgj,hjd->nhgd", p, v.abs())
    bound = torch.einsum("nhgj,hjd->nhgd", off, codes) + 2.0 ** -12 * mass
    es = 2.0 ** -18 * qs.abs().amax(dim=-1) * k.abs().sum(dim=-1).amax(dim=-1)[None, :, None] + \
        2.0 ** -20 * torch.einsum("nhgd,hjd->nhgj", qs.abs(), k.abs()).amax(dim=-1)
    bound = bound + 2 * dim ** -0.5 * es[..., None] * mass
    bound = bound * (1 + 2.0 ** -7) + 2.0 ** -8 * o.abs()
    return o.reshape(n, heads, dim), bound.reshape(n, heads, dim)


def verify(q, k, v, tokens, batch):
    """A batch of sequences over the same pages, `tokens` queries each, of which some are checked. -> their results, exact ones."""
    kc, ks = quantized(k, PAGE)
    vc, vs = quantized(v, PAGE)
    n, pages = k.shape[1], kc.shape[0]
    cache = {"keys": kc, "values": vc, "key_scales": ks, "value_scales": vs}
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].repeat(batch, 1)
    lengths = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    offsets = None if tokens == 1 else torch.arange(0, batch * tokens + 1, tokens, dtype=torch.int32, device="cuda")
    got = fp8_paged_attention(q, cache, table, lengths, offsets=offsets)
    kd, vd = dequantized(kc, ks), dequantized(vc, vs)
    outs = []
    for b in sorted({0, 1, batch // 2, batch - 1}):
        rows = slice(b * tokens, (b + 1) * tokens)
        want, bound = exact(q[rows], kd, vd, vs)
        off = (got[rows].double() - want).abs()
        assert (off <= bound).all(), (float((off / bound).max()), float(off.norm() / want.norm()))
        outs.append((got[rows], want))
    return outs


def first_key(tail, share, dim):
    """Two dimensions of a key whose score takes `share` of the mass beside the sum `tail` of the others' exponentials,
    for queries of 16 and 1 there: the second makes up for the first's rounding to E4M3."""
    score = math.log(tail * share / (1 - share)) * dim ** 0.5
    coarse = float(torch.tensor(score / 16).to(torch.float8_e4m3fn).float())
    return coarse, score - 16 * coarse


@pytest.mark.parametrize("batch", [1, 64])
@pytest.mark.parametrize("share", [0.5, 0.8, 0.99])
@pytest.mark.parametrize("n", [1024, 8192, 32768])
@pytest.mark.parametrize("kv,group,dim,tokens", FORMS)
def test_first_position_has_much_of_the_mass(cuda_device, kv, group, dim, tokens, n, share, batch):
    """Scores of the others are N(0, 1), their values N(0.25, 1); the first one's values are small."""
    gen = torch.Generator(device="cuda").manual_seed(n + dim + group)
    k, v = (torch.randn(kv, n, dim, generator=gen, device="cuda", dtype=torch.float32) for _ in range(2))
    v = v + 0.25
    k[..., :2] = 0
    k[:, 0] = 0
    v[:, 0] *= 0.01
    k[:, 0, 0], k[:, 0, 1] = first_key(n * math.exp(0.5), share, dim)
    q = torch.randn(batch * tokens, kv * group, dim, generator=gen, device="cuda").bfloat16()
    q[..., 0], q[..., 1] = 16, 1
    verify(q, k, v, tokens, batch)


@pytest.mark.parametrize("n", [512, 4096, 16384, 16384 + 11 * 1024])
@pytest.mark.parametrize("kv,group,dim,tokens", FORMS)
def test_equal_small_weights(cuda_device, kv, group, dim, tokens, n):
    """Half of the mass at the first position, whose values are zero; all others have the same weight and values of one."""
    k, v = torch.zeros(kv, n, dim, device="cuda"), torch.ones(kv, n, dim, device="cuda")
    v[:, 0] = 0
    k[:, 0, 0], k[:, 0, 1] = first_key(n - 1, 0.5, dim)
    batch = 64 if tokens == 1 else 8
    q = torch.zeros(batch * tokens, kv * group, dim, device="cuda", dtype=torch.bfloat16)
    q[..., 0], q[..., 1] = 16, 1
    for got, want in verify(q, k, v, tokens, batch):
        assert abs(float(want.mean()) - 0.5) < 0.05 and abs(float(got.float().mean() / want.mean()) - 1) < 2.0 ** -7


@pytest.mark.parametrize("apart", [8, 12, 16])
@pytest.mark.parametrize("kv,group,dim,tokens", FORMS)
def test_pages_of_small_values(cuda_device, kv, group, dim, tokens, apart):
    """One page has a value 2^apart times as large as all others' in one dimension, and zeros in the other dimensions,
    where the results are what the other pages hold."""
    gen = torch.Generator(device="cuda").manual_seed(apart)
    n = 2048
    k = torch.randn(kv, n, dim, generator=gen, device="cuda")
    v = torch.rand(kv, n, dim, generator=gen, device="cuda") + 0.5
    v[:, 5 * PAGE:6 * PAGE] = 0
    v[:, 5 * PAGE + 7, 3] = 2.0 ** apart
    q = torch.randn(64 * tokens, kv * group, dim, generator=gen, device="cuda").bfloat16()
    for got, want in verify(q, k, v, tokens, 64):
        small = torch.arange(dim, device="cuda") != 3
        assert float((got.double() - want)[..., small].norm() / want[..., small].norm()) < 2.0 ** -7


@pytest.mark.parametrize("apart", [18, 20])
@pytest.mark.parametrize("kv,group,dim,tokens", FORMS)
def test_pages_of_far_smaller_values(cuda_device, kv, group, dim, tokens, apart):
    """The same with values of which few bits are left: the bound is an eighth and half of the others' values."""
    gen = torch.Generator(device="cuda").manual_seed(apart)
    n = 2048
    k = torch.randn(kv, n, dim, generator=gen, device="cuda")
    v = torch.rand(kv, n, dim, generator=gen, device="cuda") + 0.5
    v[:, 5 * PAGE:6 * PAGE] = 0
    v[:, 5 * PAGE + 7, 3] = 2.0 ** apart
    q = torch.randn(64 * tokens, kv * group, dim, generator=gen, device="cuda").bfloat16()
    verify(q, k, v, tokens, 64)


@pytest.mark.parametrize("share", [0.5, 0.9])
@pytest.mark.parametrize("group", [4, 20])
def test_a_token_alone_and_in_a_prompt(cuda_device, group, share):
    """The same query as a single token and as the last of a chunk: both kernels within their roundings of one another."""
    gen = torch.Generator(device="cuda").manual_seed(group)
    kv, dim, n, tokens, batch = 2, 128, 16384, 40, 64
    k, v = (torch.randn(kv, n, dim, generator=gen, device="cuda") for _ in range(2))
    v = v + 0.5
    k[..., :2] = 0
    k[:, 0] = 0
    v[:, 0] *= 0.01
    k[:, 0, 0], k[:, 0, 1] = first_key(n * math.exp(0.5), share, dim)
    q = torch.randn(tokens, kv * group, dim, generator=gen, device="cuda").bfloat16()
    q[..., 0], q[..., 1] = 16, 1
    chunk = verify(q, k, v, tokens, 1)[0]
    for alone in verify(q[-1:].repeat(batch, 1, 1), k, v, 1, batch):
        assert float((alone[0][0].double() - chunk[0][-1].double()).norm() / chunk[1][-1].norm()) < 2.0 ** -8


@pytest.mark.parametrize("qe,ke", [(122, -64), (100, -64), (-100, 60), (-120, 100)])
@pytest.mark.parametrize("kv,group,dim,tokens", FORMS)
def test_large_queries_over_small_keys(cuda_device, kv, group, dim, tokens, qe, ke):
    """Queries and keys near either end of float32 whose products are not: one position has all of the weight."""
    n, at = 512, 333
    k = torch.zeros(kv, n, dim, device="cuda")
    k[:, at] = 1
    codes, _ = quantized(k, PAGE)
    values = torch.arange(n, device="cuda").float().remainder(16)[None, :, None].expand(kv, n, dim)
    vc, vs = quantized(values, PAGE)
    cache = {"keys": codes, "values": vc, "key_scales": torch.full_like(vs, 127 + ke), "value_scales": vs}
    q = torch.full((8 * tokens, kv * group, dim), 2.0 ** qe, device="cuda", dtype=torch.bfloat16)
    # codes of 2^8: scores of 2^(8 + qe + ke) times the head size at that position, zero at the others
    scale = max(1.0, 2.0 ** -(qe + ke))
    assert float(codes.view(torch.float8_e4m3fn).float().max()) == 256
    table = torch.arange(n // PAGE, dtype=torch.int32, device="cuda")[None].repeat(8, 1)
    lengths = torch.full((8,), n, dtype=torch.int32, device="cuda")
    offsets = None if tokens == 1 else torch.arange(0, 8 * tokens + 1, tokens, dtype=torch.int32, device="cuda")
    got, lse = fp8_paged_attention(q, cache, table, lengths, offsets=offsets, scale=scale, return_lse=True)
    assert (got == at % 16).all()
    want = scale * 2.0 ** (8 + qe + ke) * dim
    assert (lse.double() / want - 1).abs().max() < 2.0 ** -20


@pytest.mark.parametrize("kv,group,dim,tokens", FORMS)
def test_not_finite_and_nothing_to_see(cuda_device, kv, group, dim, tokens):
    """A query that is not finite and sees nothing has zeros like any other: all of its pages are outside the cache, or
    those in its window. One that sees anything is NaN."""
    n, batch = 4 * PAGE, 4
    gen = torch.Generator(device="cuda").manual_seed(3)
    (kc, ks), (vc, vs) = (quantized(torch.randn(kv, n, dim, generator=gen, device="cuda"), PAGE) for _ in range(2))
    cache = {"keys": kc, "values": vc, "key_scales": ks, "value_scales": vs}
    table = torch.tensor([[-1, 9, -1, 1 << 30], [0, 1, 2, 3], [0, 1, 2, -1], [-1, -1, -1, 3]], dtype=torch.int32, device="cuda")
    lengths = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    offsets = None if tokens == 1 else torch.arange(0, batch * tokens + 1, tokens, dtype=torch.int32, device="cuda")
    for bad in (math.nan, math.inf):
        q = torch.randn(batch, tokens, kv * group, dim, generator=gen, device="cuda").bfloat16()
        q[:, :, 1, 3] = bad
        got, lse = fp8_paged_attention(q.view(-1, kv * group, dim), cache, table, lengths, offsets=offsets, return_lse=True)
        got, lse = got.view(q.shape), lse.view(q.shape[:3])
        assert (got[0] == 0).all() and (lse[0] == -math.inf).all()
        assert got[1:, :, 1].isnan().all() and lse[1:, :, 1].isnan().all()
        others = [h for h in range(kv * group) if h != 1]
        assert got[1:, :, others].isfinite().all() and lse[1:, :, others].isfinite().all()
        got, lse = fp8_paged_attention(q.view(-1, kv * group, dim), cache, table, lengths, offsets=offsets, window=20,
                                       return_lse=True)
        got, lse = got.view(q.shape), lse.view(q.shape[:3])
        assert (got[2] == 0).all() and (lse[2] == -math.inf).all()
        assert got[3, :, 1].isnan().all() and got[3, :, others].isfinite().all()


@pytest.mark.parametrize("first", ["small", "large"])
@pytest.mark.parametrize("kv,group,dim,tokens", FORMS)
def test_logarithms_over_scales_far_apart(cuda_device, kv, group, dim, tokens, first):
    """Half of the pages have a value scale 2^100 times as large as the others': the sum of the exponentials counts all
    positions. Off by float32 sums of 64 exponentials a lane and page (2^-17 with room) and arguments of up to 2^8 (2^-15)."""
    n, batch = 40 * PAGE, 8
    gen = torch.Generator(device="cuda").manual_seed(7)
    kc, ks = quantized(torch.randn(kv, n, dim, generator=gen, device="cuda"), PAGE)
    vc, _ = quantized(torch.randn(kv, n, dim, generator=gen, device="cuda"), PAGE)
    vs = torch.full_like(ks, 127 - 64)
    vs[(0 if first == "large" else 1)::2] = 127 + 36
    cache = {"keys": kc, "values": vc, "key_scales": ks, "value_scales": vs}
    table = torch.arange(n // PAGE, dtype=torch.int32, device="cuda")[None].repeat(batch, 1)
    lengths = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    offsets = None if tokens == 1 else torch.arange(0, batch * tokens + 1, tokens, dtype=torch.int32, device="cuda")
    q = torch.randn(batch * tokens, kv * group, dim, generator=gen, device="cuda").bfloat16()
    _, lse = fp8_paged_attention(q, cache, table, lengths, offsets=offsets, return_lse=True)
    k = dequantized(kc, ks)
    for b in (0, batch - 1):
        rows = slice(b * tokens, (b + 1) * tokens)
        qs = q[rows].double().view(tokens, kv, group, dim)
        s = torch.einsum("nhgd,hjd->nhgj", qs, k) * dim ** -0.5
        seen = torch.arange(n, device="cuda")[None] <= n - tokens + torch.arange(tokens, device="cuda")[:, None]
        want = torch.logsumexp(torch.where(seen[:, None, None], s, torch.full_like(s, -math.inf)), dim=-1)
        es = 2.0 ** -18 * qs.abs().amax(dim=-1) * k.abs().sum(dim=-1).amax(dim=-1)[None, :, None] * dim ** -0.5
        off = (lse[rows].double() - want.reshape(tokens, -1)).abs()
        assert (off <= es.reshape(tokens, -1) + 2.0 ** -14).all(), float(off.max())


@pytest.mark.parametrize("power", list(range(20, 34)) + [60, 100])
@pytest.mark.parametrize("kv,group,dim,tokens", FORMS)
def test_scores_a_step_apart(cuda_device, kv, group, dim, tokens, power):
    """Scores so large that neighbours in float32 are as far apart as the weights' range reaches. The values are all one, in
    tiles of scale 2^-8 and 2^9 by turns, whose exponents move a score by a step or none: a result is one whatever
    the scores round to."""
    n, batch = 1024, 64 if tokens == 1 else 8
    k = torch.zeros(kv, n, dim, device="cuda")
    k[..., 0] = 256
    kc, ks = quantized(k, PAGE)
    ve = torch.where(torch.arange(n // PAGE, device="cuda") // 2 % 2 == 0, -8, 9)
    vc = torch.exp2(-ve.float())[:, None, None, None].expand(-1, kv, PAGE, dim).to(torch.float8_e4m3fn).view(torch.uint8)
    cache = {"keys": kc, "values": vc.contiguous(), "key_scales": ks,
             "value_scales": (127 + ve).to(torch.uint8)[:, None].expand(-1, kv).contiguous()}
    assert (dequantized(cache["values"], cache["value_scales"]) == 1).all()
    q = torch.zeros(batch * tokens, kv * group, dim, device="cuda", dtype=torch.bfloat16)
    q[..., 0] = 1 + torch.arange(q[..., 0].numel(), device="cuda").view(q.shape[:2]) % 128 / 128
    table = torch.arange(n // PAGE, dtype=torch.int32, device="cuda")[None].repeat(batch, 1)
    lengths = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    offsets = None if tokens == 1 else torch.arange(0, batch * tokens + 1, tokens, dtype=torch.int32, device="cuda")
    for sign in (1, -1):  # scores of 2^power to 2^(power + 1) in powers of two, of either sign
        got = fp8_paged_attention(sign * q, cache, table, lengths, offsets=offsets, scale=math.log(2) * 2.0 ** (power - 8))
        # f16 weights and their terms, sums, bf16: 2^-10 + 2^-12 + 2^-8 at most
        assert ((got.double() - 1).abs() < 2.0 ** -7).all(), (sign, float(got.min()), float(got.max()))
