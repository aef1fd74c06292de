"""Rotary positions, the append to a paged FP8 cache and attention over it in 64 bits, for the tests of these operators."""

from __future__ import annotations

import math

import torch

E4M3_MAX = 448.0
SMALLEST = -64  # exponent of a cache's smallest scale


def turned64(x, positions, radians, *, interleaved=False, magnitude=1.0, inverse=False):
    """x [T,H,D] with the first 2 * len(radians) dimensions turned, in float64."""
    pairs, out = len(radians), x.double().clone()
    # Positions and frequencies of a few hundred radians: the product's rounding in 64 bits is far below the tolerances.
    angle = positions.double().cpu()[:, None] * torch.tensor(radians, dtype=torch.float64)[None]
    cos, sin = angle.cos()[:, None].to(x.device), angle.sin()[:, None].to(x.device)
    if inverse:
        sin = -sin
    at = torch.arange(pairs, device=x.device)
    first, second = (2 * at, 2 * at + 1) if interleaved else (at, at + pairs)
    a, b = x.double()[..., first], x.double()[..., second]
    out[..., first], out[..., second] = magnitude * (a * cos - b * sin), magnitude * (a * sin + b * cos)
    return out


def turned_bound(x, rotary, magnitude, interleaved):
    """How far a rotation in float32 may be from the exact one, [T,H,rotary/2] for both values of a pair.

    In steps of 2^-24: the angle within an eighth of a turn is rounded twice (2 * 0.79), the polynomials are off by half
    a step and rounded at the end (1.5): 3.1 for a cosine or sine. A product adds its own rounding, the sum one and the
    magnitude one: at most 3.1 + 1 + 1 + 1 for each of |a| and |b|, and 8 with room for the second orders.
    """
    x = x.double().abs()[..., :rotary]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :rotary // 2], x[..., rotary // 2:])
    return 8 * 2.0 ** -24 * abs(magnitude) * (a + b)


def page_exponent(amax: float) -> int:
    """The smallest e with amax <= 448 * 2^e, at least -64."""
    if amax == 0:
        return SMALLEST
    mant, exp = math.frexp(amax)  # 448 = 0.875 * 2^9
    return max(exp - 9 + (mant > 0.875), SMALLEST)


def e4m3_rounded(v):
    """float64 rounded to E4M3: 4 significant bits, steps of 2^-9 below 2^-6, ties to even."""
    step = torch.exp2((torch.frexp(v)[1] - 1).clamp_min(-6).double() - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def append64(codes, scales, x, table, lengths, offsets):
    """The append of x [T,H,D] (float64) to a cache of values (float64 E4M3 numbers, exponents int) on the host.

    -> (values, exponents, unrounded): ``unrounded`` holds new tokens before their rounding and NaN elsewhere.
    """
    values, exps = codes.clone(), scales.clone()
    unrounded = torch.full_like(values, math.nan)
    page, pages = values.shape[2], values.shape[0]
    for b, length in enumerate(lengths):
        length = min(max(length, 0), page * len(table[b]))
        tokens = range(offsets[b], offsets[b + 1])
        places = {}
        for i, t in enumerate(tokens):
            column = (length + i) // page
            if column < len(table[b]) and 0 <= table[b][column] < pages:
                places.setdefault(table[b][column], []).append((t, (length + i) % page))
        for at, new in places.items():
            begun = new[0][1]
            rows, slots = x[[t for t, _ in new]], [s for _, s in new]
            for h in range(x.shape[1]):
                e = page_exponent(float(rows[:, h].abs().max()))
                if begun:
                    old = int(exps[at, h])
                    e = max(e, old)
                    values[at, h, :begun] = e4m3_rounded(values[at, h, :begun] * 2.0 ** (old - e))
                exps[at, h] = e
                unrounded[at, h, slots] = rows[:, h] * 2.0 ** -e
                values[at, h, slots] = e4m3_rounded(rows[:, h] * 2.0 ** -e)
    return values, exps, unrounded


def attention64(q, cache, table, lengths, offsets=None, window=0, scale=None):
    """Attention in float64 on q's device, its logarithms of sums, and how far the kernels' results may be off.

    The queries are exact but for what is below 2^-18 of the row's largest value, so a score is off by that times the
    keys, and by the float32 sums (2^-20 of the products' sum with room). The weights, scaled by their positions' value
    scales, are two E4M3 terms: off by 2^-8 of their value, or by 2^-14 of the row's largest where that is more and the
    weight not less. The result is rounded to bf16: 2^-8, or half the smallest step, 2^-133, which is what a result that
    is not zero in 64 bits alone may be off by.
    """
    dev, (tokens, heads, dim) = q.device, q.shape
    keys, values = (cache[n].view(torch.float8_e4m3fn).double() for n in ("keys", "values"))
    pages, kv, page, _ = keys.shape
    ke, ve = (cache[n].double() - 127 for n in ("key_scales", "value_scales"))
    ke, ve = (torch.where(e == 128, torch.full_like(e, math.nan), e) for e in (ke, ve))
    group, scale = heads // kv, dim ** -0.5 if scale is None else scale
    offsets = list(range(len(lengths) + 1)) if offsets is None else offsets
    out = torch.zeros(tokens, heads, dim, dtype=torch.float64, device=dev)
    lse = torch.full((tokens, heads), -math.inf, dtype=torch.float64, device=dev)
    bound, lse_bound = torch.zeros_like(out), torch.zeros_like(out[..., 0])
    for b, length in enumerate(lengths):
        n = offsets[b + 1] - offsets[b]
        length = min(max(length, 0), page * table.shape[1])
        if n <= 0 or length == 0:
            continue
        rows = table[b, :-(-length // page)].long()
        there = ((rows >= 0) & (rows < pages)).repeat_interleave(page)[:length]
        rows = rows.clamp(0, pages - 1)

        def gather(codes, exps):
            x = codes[rows] * torch.exp2(exps[rows])[..., None, None]
            return x.transpose(0, 1).reshape(kv, -1, dim)[:, :length]

        k, v = gather(keys, ke), gather(values, ve)
        e = ve[rows].transpose(0, 1).repeat_interleave(page, dim=1)[:, :length]
        qs = q[offsets[b]:offsets[b + 1]].double().view(n, kv, group, dim).permute(1, 2, 0, 3)  # [kv, group, n, dim]
        j, at = torch.arange(length, device=dev), length - n + torch.arange(n, device=dev)
        seen = (j[None] <= at[:, None]) & there[None]
        if window:
            seen &= j[None] > at[:, None] - window
        s = torch.einsum("hgnd,hjd->hgnj", qs, k) * scale
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        top = s.amax(dim=-1, keepdim=True)
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
        p = torch.exp(s - top)
        total = p.sum(dim=-1)
        some = total != 0
        safe = torch.where(some, total, torch.ones_like(total))
        bad = (seen[None, None] & torch.isnan(v).any(dim=-1)[:, None, None]).any(dim=-1)  # [kv, group, n]
        vv = torch.nan_to_num(v, nan=0.0)
        o = torch.einsum("hgnj,hjd->hgnd", p, vv) / safe[..., None]
        o = torch.where(bad[..., None], torch.full_like(o, math.nan), o)
        # The bounds.
        qmax, qabs = qs.abs().amax(dim=-1), qs.abs()
        ks, seen_k = k.abs().sum(dim=-1), torch.where(seen, 1.0, 0.0)
        es = 2.0 ** -18 * qmax * torch.nan_to_num(ks[:, None, None] * seen_k).amax(dim=-1) + \
            2.0 ** -20 * torch.nan_to_num(torch.einsum("hgnd,hjd->hgnj", qabs, k.abs()) * seen_k).amax(dim=-1)
        es = es * scale
        w = p * torch.exp2(torch.nan_to_num(e))[:, None, None]
        off = torch.maximum(2.0 ** -8 * w, torch.minimum(w, 2.0 ** -14 * w.amax(dim=-1, keepdim=True)))
        codes = vv.abs() * torch.exp2(-torch.nan_to_num(e))[..., None]
        ob = torch.einsum("hgnj,hjd->hgnd", off, codes) / safe[..., None]
        ob = ob + 2 * es[..., None] * torch.einsum("hgnj,hjd->hgnd", p, vv.abs()) / safe[..., None]
        ob = ob * (1 + 2.0 ** -7) + 2.0 ** -8 * o.abs() + 2.0 ** -134
        span = slice(offsets[b], offsets[b + 1])
        back = lambda x: x.permute(2, 0, 1, *range(3, x.ndim)).reshape(n, heads, *x.shape[3:])  # noqa: E731
        out[span], lse[span] = back(o), back(torch.where(some, top[..., 0] + torch.log(safe), torch.full_like(total, -math.inf)))
        # exponentials of 2^-17 or better, sums and logarithms in float32
        bound[span], lse_bound[span] = back(ob), back(es) + 2.0 ** -16
    lse_bound = lse_bound + 2.0 ** -22 * torch.where(lse.isfinite(), lse.abs(), torch.zeros_like(lse))
    return out, lse, bound, lse_bound


def make_cache(gen, pages, kv, page, dim, device, spread=3):
    """A cache of random codes and scales: no NaN codes, values of a few powers of two."""
    codes = lambda: (torch.randn(pages, kv, page, dim, generator=gen) * 40).clamp(-448, 448).to(torch.float8_e4m3fn) \
        .view(torch.uint8).to(device)  # noqa: E731
    scales = lambda: (127 - 5 + torch.randint(-spread, spread + 1, (pages, kv), generator=gen)).to(torch.uint8).to(device)  # noqa: E731
    return {"keys": codes(), "values": codes(), "key_scales": scales(), "value_scales": scales()}


def make_table(gen, lengths, page, pages, columns=None):
    """int32 page table of pages in random order: none is used twice."""
    columns = max([1] + [-(-n // page) for n in lengths]) if columns is None else columns
    order, at = torch.randperm(pages, generator=gen).tolist(), 0
    table = torch.full((len(lengths), columns), -1, dtype=torch.int32)
    for b, n in enumerate(lengths):
        for c in range(min(-(-n // page), columns)):
            table[b, c] = order[at]
            at += 1
    return table


def starts(counts):
    return [sum(counts[:b]) for b in range(len(counts) + 1)]
