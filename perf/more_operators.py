"""Cases for rotary positions, the append to a paged FP8 key/value cache and attention over that cache.

``run`` computes a case either in its plain form (elementary torch operations
in 32 bits, rotation angles and the cache's quantization in 64) or, with
``own`` true, through the framework's public functions. The cache holds E4M3
codes in pages, [pages, heads, page tokens, head size], with one power-of-two
scale (a UE8M0 byte) per page and head, for keys and for values.
"""

import math

import torch

own = False

E4M3_MAX = 448.0
SMALLEST = -64  # exponent of the cache's smallest scale
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}

# The most that a drawn case may have (the largest listed cases are at or above it).
MAX_SCORES = 2.0e9   # query heads x padded queries x padded context
MAX_CACHED = 5.5e8   # cached key values, padded
MAX_VALUES = 6.0e7   # values of a rotation or an append


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # A small decode batch's query heads: latency.
        {"name": "rotary_decode", "op": "rotary", "tokens": 8, "heads": 32, "dim": 128, "rotary": 128, "interleaved": False, "scaling": "none", "factor": 1.0, "far": 8192, "x": "bf16"},
        # The query heads of a prompt, with positions scaled for a long context.
        {"name": "rotary_prompt", "op": "rotary", "tokens": 8192, "heads": 32, "dim": 128, "rotary": 128, "interleaved": False, "scaling": "yarn", "factor": 8.0, "far": 65536, "x": "bf16"},
        # Interleaved pairs, part of the head, float32, far positions, odd counts.
        {"name": "rotary_odd", "op": "rotary", "tokens": 1777, "heads": 23, "dim": 96, "rotary": 72, "interleaved": True, "scaling": "linear", "factor": 4.0, "far": 1 << 20, "x": "f32"},
        # A decode step of 64 sequences: a token each, into pages that are partly filled.
        {"name": "append_decode", "op": "append", "batch": 64, "context": 4096, "queries": 1, "decoding": 0, "uneven": 0.7, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "rotary": 128, "interleaved": False, "scaling": "bands", "factor": 8.0, "x": "bf16"},
        # Prompts of up to 8192 tokens, from empty sequences.
        {"name": "append_prompt", "op": "append", "batch": 3, "context": 0, "queries": 8192, "decoding": 0, "uneven": 0.6, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "rotary": 128, "interleaved": False, "scaling": "none", "factor": 1.0, "x": "bf16"},
        # Small pages, an odd head size, ragged chunks that begin and end inside pages, float32.
        {"name": "append_odd", "op": "append", "batch": 11, "context": 700, "queries": 203, "decoding": 3, "uneven": 0.9, "heads": 15, "kv_heads": 5, "dim": 80, "page": 16, "rotary": 40, "interleaved": True, "scaling": "none", "factor": 1.0, "x": "f32"},
        # One token of one short conversation: latency.
        {"name": "attend_one", "op": "attention", "batch": 1, "context": 1000, "queries": 1, "decoding": 0, "uneven": 0.0, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "lse": False},
        # A decode step of 64 conversations of unequal length: streaming the cache.
        {"name": "attend_decode", "op": "attention", "batch": 64, "context": 8191, "queries": 1, "decoding": 0, "uneven": 0.5, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "lse": False},
        # One token over one very long context: few rows, a long axis.
        {"name": "attend_long", "op": "attention", "batch": 1, "context": 131071, "queries": 1, "decoding": 0, "uneven": 0.0, "heads": 64, "kv_heads": 8, "dim": 128, "page": 128, "window": 0, "lse": True},
        # Odd everything: head size 80, 6 query heads to a key head, small pages, a sliding window, a few tokens each.
        {"name": "attend_odd", "op": "attention", "batch": 13, "context": 3001, "queries": 5, "decoding": 4, "uneven": 0.9, "heads": 30, "kv_heads": 5, "dim": 80, "page": 16, "window": 1025, "lse": True},
        # A prompt of 8192 tokens.
        {"name": "attend_prompt", "op": "attention", "batch": 1, "context": 0, "queries": 8192, "decoding": 0, "uneven": 0.0, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "lse": False},
        # A serving step: chunks of two prompts over what they have cached, and 14 conversations that decode.
        {"name": "attend_mixed", "op": "attention", "batch": 16, "context": 7000, "queries": 512, "decoding": 14, "uneven": 0.6, "heads": 32, "kv_heads": 4, "dim": 64, "page": 32, "window": 0, "lse": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    kv = rng.choice([1, 2, 3, 4, 5, 8, 8, 16])
    return kv, kv * rng.choice([1, 2, 3, 4, 4, 6, 8, 8, 16])


def _rotation(rng, dim):
    scaling = rng.choice(["none", "none", "linear", "bands", "yarn"])
    return {"rotary": rng.choice([dim, dim, dim // 2, 2 * rng.randint(4, dim // 2)]), "interleaved": rng.random() < 0.4,
            "scaling": scaling, "factor": 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0, 32.0])}


def draw(rng):
    op = rng.choice(["rotary", "append", "attention", "attention"])
    for _ in range(1000):
        kv, heads = _heads(rng)
        dim, page = rng.choice([64, 80, 96, 112, 128, 128, 128]), rng.choice([16, 32, 64, 64, 128])
        if heads > 64:
            continue
        if op == "rotary":
            c = {"op": op, "tokens": _log_int(rng, 1, 16384), "heads": heads, "dim": dim, **_rotation(rng, dim),
                 "far": _log_int(rng, 1000, 1 << 21), "x": rng.choice(["bf16", "bf16", "f32"])}
            fits = c["tokens"] * heads * dim <= MAX_VALUES / 2
        else:
            batch, kind = _log_int(rng, 1, 128), rng.random()
            if kind < 0.5:  # a token of each sequence
                queries, context, decoding = 1, _log_int(rng, 1, 65536), 0
            else:  # prompts, chunks and mixtures
                queries = _log_int(rng, 2, 8192)
                context = 0 if rng.random() < 0.4 else _log_int(rng, 1, 16384)
                decoding = rng.randint(0, batch - 1) if rng.random() < 0.4 else 0
            c = {"op": op, "batch": batch, "context": context, "queries": queries, "decoding": decoding,
                 "uneven": round(rng.choice([0.0, rng.random()]), 3), "heads": heads, "kv_heads": kv, "dim": dim, "page": page}
            padded = batch * (context + queries)
            fits = padded * kv * dim <= MAX_CACHED
            if op == "append":
                c.update(_rotation(rng, dim), x=rng.choice(["bf16", "bf16", "f32"]))
                fits = fits and batch * queries * (heads + 2 * kv) * dim <= 4 * MAX_VALUES
                fits = fits and batch * queries * kv * dim <= MAX_VALUES / 2
            else:
                c.update(window=rng.choice([0, 0, 0, _log_int(rng, 16, 8192)]), lse=rng.random() < 0.5)
                fits = fits and padded * heads * queries <= MAX_SCORES
        if fits:
            return c
    raise RuntimeError("no case within the limits")


def _spread(b, by):
    return (b + 1) * by % 1.0


def _new_tokens(c):
    """New tokens of each sequence: the last `decoding` ones have one."""
    return [1 if b >= c["batch"] - c["decoding"] else max(1, round(c["queries"] * (1.0 - c["uneven"] * _spread(b, 0.7548777))))
            for b in range(c["batch"])]


def _contexts(c):
    """Tokens of each sequence before the new ones."""
    return [round(c["context"] * (1.0 - c["uneven"] * _spread(b, 0.618034))) for b in range(c["batch"])]


def work(case):
    c, size = case, {"bf16": 2, "f32": 4}
    if c["op"] == "rotary":
        n = c["tokens"] * c["heads"]
        return {"bytes": 2 * n * c["dim"] * size[c["x"]] + 4 * c["tokens"], "flops": 3 * n * c["rotary"]}
    new, before = _new_tokens(c), _contexts(c)
    if c["op"] == "append":
        n = sum(new) * c["kv_heads"]
        return {"bytes": 2 * n * c["dim"] * (size[c["x"]] + 1), "flops": n * (3 * c["rotary"] + 4 * c["dim"])}
    seen, pairs = 0, 0
    for n, past in zip(new, before):
        total, window = past + n, c["window"] or past + n
        seen += min(total, window + n - 1)
        full = max(0, min(n, window - past))  # queries that see all before them: i + past + 1 positions
        pairs += full * (past + 1) + full * (full - 1) // 2 + (n - full) * window
    return {"bytes": 2 * seen * c["kv_heads"] * c["dim"] + 4 * sum(new) * c["heads"] * c["dim"],
            "flops": 4 * pairs * c["heads"] * c["dim"]}


# --------------------------------------------------------------------------- inputs
ROPE_BASE, ROPE_ORIGINAL = 500000.0, 8192


def _frequencies(c):
    """Radians per position of each pair (Python floats), and the factor of the rotated values."""
    r, factor = c["rotary"], c["factor"]
    plain = [ROPE_BASE ** (-2.0 * i / r) for i in range(r // 2)]
    if c["scaling"] == "linear":
        return [f / factor for f in plain], 1.0
    if c["scaling"] == "bands":  # low frequencies divided, high ones kept, linear in between
        low, high = 1.0, 4.0
        blend = [min(1.0, max(0.0, (ROPE_ORIGINAL * f / (2.0 * math.pi) - low) / (high - low))) for f in plain]
        return [(1.0 - s) * f / factor + s * f for f, s in zip(plain, blend)], 1.0
    if c["scaling"] == "yarn":  # a ramp over the pairs, between those that turn 32 times and once in the original context
        def pair(turns):
            return r * math.log(ROPE_ORIGINAL / (turns * 2.0 * math.pi)) / (2.0 * math.log(ROPE_BASE))

        first, last = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), r - 1)
        ramp = [min(1.0, max(0.0, (i - first) / max(last - first, 0.001))) for i in range(r // 2)]
        return [f * (1.0 - s) + f / factor * s for f, s in zip(plain, ramp)], 0.1 * math.log(factor) + 1.0
    return plain, 1.0


def _hidden(shape, gen, dev):
    """Normal values with a few larger channels, as projections give them."""
    x = torch.randn(shape, generator=gen, device=dev)
    gain = torch.rand(shape[-1], generator=gen, device=dev)
    return x * torch.where(gain > 0.97, 6.0, 1.0)


def _starts(counts):
    return torch.tensor([sum(counts[:b]) for b in range(len(counts) + 1)], dtype=torch.int32)


def _cache(c, totals, gen, dev):
    """Page table int32 [B, most pages], and key and value codes and scales of a cache that holds the sequences."""
    used = [-(-t // c["page"]) for t in totals]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=gen, device=dev).int().cpu()
    table = torch.zeros((c["batch"], max(used)), dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    state = {"table": table.to(dev)}
    shape = (pages, c["kv_heads"], c["page"], c["dim"])
    for name in ("keys", "values"):
        codes = torch.empty(shape, dtype=torch.uint8, device=dev)
        scales = torch.empty(shape[:2], dtype=torch.uint8, device=dev)
        gain = torch.where(torch.rand(c["dim"], generator=gen, device=dev) > 0.97, 6.0, 1.0)
        for p in range(0, pages, 1024):
            x = torch.randn((min(1024, pages - p), *shape[1:]), generator=gen, device=dev) * gain
            mant, exp = torch.frexp(x.abs().amax(dim=(2, 3)))
            e = exp - 9 + (mant > 0.875).int()
            codes[p:p + 1024] = (x * torch.exp2(-e.float())[:, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
            scales[p:p + 1024] = (e + 127).to(torch.uint8)
        state[name], state[name[:-1] + "_scales"] = codes, scales
    return state


def _inputs(case, seed):
    """The case's data on the GPU, made from the seed alone."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    c = case
    if c["op"] == "rotary":
        x = _hidden((c["tokens"], c["heads"] * c["dim"]), gen, dev).to(DTYPES[c["x"]])
        positions = torch.randint(0, c["far"], (c["tokens"],), generator=gen, device=dev, dtype=torch.int32)
        return {"x": x.view(c["tokens"], c["heads"], c["dim"]), "positions": positions}
    new, before = _new_tokens(c), _contexts(c)
    state = _cache(c, [n + p for n, p in zip(new, before)], gen, dev)
    state["offsets"] = _starts(new).to(dev)
    state["before"] = torch.tensor(before, dtype=torch.int32, device=dev)
    state["lengths"] = state["before"] + torch.tensor(new, dtype=torch.int32, device=dev)
    if c["op"] == "append":
        # Keys and values are views of a projection's output, which has the query heads first.
        h, k, d = c["heads"], c["kv_heads"], c["dim"]
        qkv = _hidden((sum(new), (h + 2 * k) * d), gen, dev).to(DTYPES[c["x"]])
        state["k"] = qkv[:, h * d:(h + k) * d].view(-1, k, d)
        state["v"] = qkv[:, (h + k) * d:].view(-1, k, d)
    else:
        state["q"] = _hidden((sum(new), c["heads"] * c["dim"]), gen, dev).to(torch.bfloat16).view(-1, c["heads"], c["dim"])
    return state


def prepare(case, seed):
    state = {"case": dict(case), **_inputs(case, seed)}
    if case["op"] != "attention":
        frequencies, magnitude = _frequencies(case)
        state["frequencies"] = torch.tensor(frequencies, dtype=torch.float64, device="cuda")
        state["magnitude"] = magnitude
    else:
        new = _new_tokens(case)
        state["most"], state["ragged"] = max(new), max(new) > 1  # a scheduler knows how many tokens it hands out
    if own:
        # A user's program keeps the rotation's frequencies and the cache from when the model was loaded.
        if case["op"] != "attention":
            from mambo_b200.kernels.rotary import prepare_rotary_fields

            state["rope"] = prepare_rotary_fields(
                case["rotary"], base=ROPE_BASE, interleaved=case["interleaved"],
                scaling=None if case["scaling"] == "none" else case["scaling"], factor=case["factor"],
                original_length=ROPE_ORIGINAL, device="cuda")
        if case["op"] != "rotary":
            state["cache"] = {name: state[name] for name in ("keys", "values", "key_scales", "value_scales")}
    return state


# --------------------------------------------------------------------------- plain forms
def _rotated(x, positions, state, c, angles_as):
    """x [T,H,D] with its first `rotary` dimensions rotated; cosines and sines from angles in 64 bits."""
    r = c["rotary"]
    angle = positions.double()[:, None] * state["frequencies"]
    cos, sin = (angle.cos() * state["magnitude"]).to(angles_as), (angle.sin() * state["magnitude"]).to(angles_as)
    cos, sin, x = cos[:, None], sin[:, None], x.to(angles_as)
    if c["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([turned, x[..., r:]], dim=-1)


def _exponent(amax):
    """The smallest e with amax <= 448 * 2^e; SMALLEST at least and for zero."""
    mant, exp = torch.frexp(amax)  # amax = mant * 2^exp, 448 = 0.875 * 2^9
    e = exp - 9 + (mant > 0.875).int()
    return torch.where(amax > 0, e, torch.full_like(e, SMALLEST)).clamp(SMALLEST, 127)


def _store(x, codes, scales, page, slot, tokens_of_page, begun):
    """Quantizes x [T,H,D] into its pages: a page's scale grows where a new token needs it, and its older codes with it."""
    pages, heads, size, dim = codes.shape
    amax = torch.zeros((pages, heads), dtype=x.dtype, device=x.device)
    amax = amax.scatter_reduce(0, page[:, None].expand(-1, heads), x.abs().amax(dim=-1), "amax")
    old = scales.int() - 127
    e = _exponent(amax)
    e = torch.where(begun[:, None] > 0, torch.maximum(e, old), e)
    e = torch.where(tokens_of_page[:, None] > 0, e, old)
    at = torch.nonzero((tokens_of_page > 0) & (begun > 0)).flatten()
    was = codes[at].view(torch.float8_e4m3fn).float() * torch.exp2((old - e)[at].float())[:, :, None, None]
    keep = torch.arange(size, device=x.device)[None, :] < begun[at][:, None]
    codes[at] = torch.where(keep[:, None, :, None], was.to(torch.float8_e4m3fn).view(torch.uint8), codes[at])
    scaled = (x * torch.exp2(-e[page].to(x.dtype))[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).float()
    codes[page[:, None], torch.arange(heads, device=x.device)[None, :], slot[:, None]] = \
        scaled.to(torch.float8_e4m3fn).view(torch.uint8)
    scales.copy_((e + 127).to(torch.uint8))


def _stored(state):
    return {"keys": state["keys"].view(torch.float8_e4m3fn), "key_scales": state["key_scales"].view(torch.float8_e8m0fnu),
            "values": state["values"].view(torch.float8_e4m3fn), "value_scales": state["value_scales"].view(torch.float8_e8m0fnu)}


def _append(state, c):
    offsets, before = state["offsets"].long(), state["before"].long()
    token = torch.arange(state["k"].shape[0], device=offsets.device)
    seq = torch.searchsorted(offsets[1:].contiguous(), token, right=True)
    position = before[seq] + token - offsets[seq]
    page, slot = state["table"].long()[seq, position // c["page"]], position % c["page"]
    count = torch.zeros(state["keys"].shape[0], dtype=torch.long, device=page.device)
    tokens_of_page = count.scatter_add(0, page, torch.ones_like(page))
    begun = count.scatter(0, page, torch.full_like(page, c["page"])).scatter_reduce(0, page, slot, "amin")  # older tokens
    _store(_rotated(state["k"], position, state, c, torch.float64), state["keys"], state["key_scales"], page, slot,
           tokens_of_page, begun)
    _store(state["v"].double(), state["values"], state["value_scales"], page, slot, tokens_of_page, begun)
    return _stored(state)


def _gathered(codes, scales, table, dtype):
    """Cached values [B, H, positions, D]."""
    b, n = table.shape
    _, heads, size, dim = codes.shape
    x = codes[table].view(torch.float8_e4m3fn).to(dtype) * torch.exp2((scales.int() - 127)[table].to(dtype))[..., None, None]
    return x.permute(0, 2, 1, 3, 4).reshape(b, heads, n * size, dim)


def _seen(offsets, lengths, most, positions, window):
    """Truth of [B, most queries, positions]: which positions a query sees."""
    count = offsets[1:] - offsets[:-1]
    query = torch.arange(most, device=offsets.device)
    at = (lengths - count)[:, None, None] + query[None, :, None]
    j = torch.arange(positions, device=offsets.device)[None, None, :]
    seen = (j <= at) & (query[None, :, None] < count[:, None, None])
    return seen & (j > at - window) if window else seen


def _attention(state, c):
    offsets, lengths, table = state["offsets"].long(), state["lengths"].long(), state["table"].long()
    q, kv, most, d = state["q"], c["kv_heads"], state["most"], c["dim"]
    token = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(offsets[1:].contiguous(), token, right=True)
    local = token - offsets[seq]
    rows = q.new_zeros((c["batch"], most, c["heads"], d), dtype=torch.float32)
    rows[seq, local] = q.float()
    group = c["heads"] // kv
    rows = rows.view(c["batch"], most, kv, group, d).permute(0, 2, 3, 1, 4).reshape(c["batch"], kv, group * most, d)
    s = rows @ _gathered(state["keys"], state["key_scales"], table, torch.float32).transpose(2, 3)
    s = s.view(c["batch"], kv, group, most, -1).mul_(d ** -0.5)
    s.masked_fill_(~_seen(offsets, lengths, most, s.shape[-1], c["window"])[:, None, None], -math.inf)
    top = s.amax(dim=-1, keepdim=True)
    top = torch.where(top > -math.inf, top, torch.zeros_like(top))
    p = s.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    o = p.view(c["batch"], kv, group * most, -1) @ _gathered(state["values"], state["value_scales"], table, torch.float32)
    o = o.view(c["batch"], kv, group, most, d) / torch.where(total > 0, total, torch.ones_like(total))
    out = o.permute(0, 3, 1, 2, 4).reshape(c["batch"], most, c["heads"], d)[seq, local].to(torch.bfloat16)
    if not c["lse"]:
        return {"out": out}
    lse = (top + total.log())[..., 0].permute(0, 3, 1, 2).reshape(c["batch"], most, c["heads"])
    return {"out": out, "lse": lse[seq, local]}


def _plain(state):
    c = state["case"]
    if c["op"] == "rotary":
        return _rotated(state["x"], state["positions"], state, c, torch.float32).to(state["x"].dtype)
    return _append(state, c) if c["op"] == "append" else _attention(state, c)


# --------------------------------------------------------------------------- the framework's calls
def _own(state):
    from mambo_b200.kernels import attention_fp8, rotary

    c = state["case"]
    if c["op"] == "rotary":
        return rotary.launch_rotary(state["x"], state["positions"], state["rope"])
    if c["op"] == "append":
        offsets = state["offsets"] if c["queries"] > 1 else None
        attention_fp8.launch_fp8_kv_append(state["cache"], state["k"], state["v"], state["table"], state["before"],
                                           offsets=offsets, rope=state["rope"])
        return _stored(state)
    answer = attention_fp8.fp8_paged_attention(
        state["q"], state["cache"], state["table"], state["lengths"], offsets=state["offsets"] if state["ragged"] else None,
        window=c["window"], return_lse=c["lse"])
    return {"out": answer[0], "lse": answer[1]} if c["lse"] else {"out": answer}


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------------- 64 bits
def _e4m3_rounded(v):
    """float64 values rounded to E4M3: 4 significant bits, steps of 2^-9 below 2^-6, ties to even."""
    step = torch.exp2((torch.frexp(v)[1] - 1).clamp_min(-6).double() - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_turned(x, positions, c):
    frequencies, magnitude = _frequencies(c)
    r, out = c["rotary"], x.double().clone()
    angle = positions.double()[:, None, None] * torch.tensor(frequencies, dtype=torch.float64, device=x.device)
    at = torch.arange(r // 2, device=x.device)
    first, second = (2 * at, 2 * at + 1) if c["interleaved"] else (at, at + r // 2)
    z = torch.complex(out[..., first], out[..., second]) * torch.polar(torch.full_like(angle, magnitude), angle)
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_store(codes, scales, x, table, before, offsets, page):
    """The cache's codes (as numbers) and scales after the append, page by page."""
    value, scale = codes.view(torch.float8_e4m3fn).double(), torch.exp2(scales.double() - 127)
    for b, past in enumerate(before):
        new = x[offsets[b]:offsets[b + 1]]
        first, n = past // page, new.shape[0]
        blocks = -(-(past + n) // page) - first
        rows = torch.zeros((blocks * page, *x.shape[1:]), dtype=torch.float64, device=x.device)
        rows[past - first * page:past - first * page + n] = new
        rows = rows.view(blocks, page, *x.shape[1:]).transpose(1, 2)
        at = table[b, first:first + blocks].long()
        amax = rows.abs().amax(dim=(2, 3))
        need = torch.where(amax > 0, torch.ceil(torch.log2(amax / E4M3_MAX)), torch.full_like(amax, SMALLEST)).clamp(SMALLEST, 127)
        need = torch.exp2(need)
        if past % page:
            need[0] = torch.maximum(need[0], scale[at[0]])
            value[at[0], :, :past % page] = _e4m3_rounded(value[at[0], :, :past % page] * (scale[at[0]] / need[0])[:, None, None])
        scale[at] = need
        coded = _e4m3_rounded(rows / need[:, :, None, None])
        slot = torch.arange(blocks * page, device=x.device).view(blocks, page) + first * page
        fresh = ((slot >= past) & (slot < past + n))[:, None, :, None]
        value[at] = torch.where(fresh, coded, value[at])
    return value, scale


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    if c["op"] == "rotary":
        return _exact_turned(s["x"], s["positions"], c)
    new, before = _new_tokens(c), _contexts(c)
    offsets = _starts(new).tolist()
    if c["op"] == "append":
        position = torch.cat([torch.arange(p, p + n, device=s["k"].device) for p, n in zip(before, new)])
        keys = _exact_store(s["keys"], s["key_scales"], _exact_turned(s["k"], position, c), s["table"], before, offsets, c["page"])
        values = _exact_store(s["values"], s["value_scales"], s["v"].double(), s["table"], before, offsets, c["page"])
        return {"keys": keys[0], "key_scales": keys[1], "values": values[0], "value_scales": values[1]}
    group, out, lse = c["heads"] // c["kv_heads"], [], []
    for b, (n, past) in enumerate(zip(new, before)):
        pages = s["table"][b, :-(-(past + n) // c["page"])].long()
        at, j = past + torch.arange(n, device=pages.device)[:, None], torch.arange(past + n, device=pages.device)[None, :]
        hidden = (j > at) | (j <= at - c["window"]) if c["window"] else j > at
        q = s["q"][offsets[b]:offsets[b + 1]].double()
        o = torch.empty_like(q)
        z = torch.empty(q.shape[:2], dtype=torch.float64, device=q.device)
        for h in range(c["heads"]):
            k, v = (s[name][pages, h // group].view(torch.float8_e4m3fn).double().mul_(torch.exp2(s[name[:-1] + "_scales"][pages, h // group].double() - 127)[:, None, None]).flatten(0, 1)[:past + n]
                    for name in ("keys", "values"))
            score = (q[:, h] @ k.t() / math.sqrt(c["dim"])).masked_fill_(hidden, -math.inf)
            z[:, h] = torch.logsumexp(score, dim=1)
            o[:, h] = torch.exp(score - z[:, h, None]) @ v
        out.append(o)
        lse.append(z)
    answer = {"out": torch.cat(out)}
    return {**answer, "lse": torch.cat(lse)} if c["lse"] else answer
