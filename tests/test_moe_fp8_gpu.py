"""Expert router, combine and the experts' path against plain float64 computations."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mambo_b200 import _lib
from mambo_b200.kernels.fp8_block import fp8_block_grouped_linear, prepare_fp8_block_fields
from mambo_b200.kernels.moe_fp8 import fp8_moe_experts, launch_moe_combine, launch_moe_route
from test_fp8_block_gpu import frob, make_weight, make_x, quantize64, weight64

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert _lib.device_status()[0] == 0


def route_ref(logits, top, scoring="softmax", bias=None, renormalize=True, scale=1.0):
    """ids from float32 scores (the selection's own precision), weights in float64."""
    l32 = np.where(np.isnan(logits), -np.inf, np.minimum(logits, np.finfo(np.float32).max)).astype(np.float32)
    masked = np.isneginf(l32)
    l = l32.astype(np.float64)
    with np.errstate(all="ignore"):
        if scoring == "softmax":
            mx = np.where(masked.all(axis=1), 0, np.where(masked, -np.inf, l).max(axis=1))
            p = np.where(masked, 0, np.exp(l - mx[:, None]))
            p = p / np.where(p.sum(axis=1) > 0, p.sum(axis=1), 1)[:, None]
            key = l32.copy()
        else:
            p = 1 / (1 + np.exp(-l))
            key = (np.float32(1) / (np.float32(1) + torch.exp(-torch.from_numpy(l32).cuda()).cpu().numpy()))
    if bias is not None:
        key = key + bias
    key = np.where(masked, -np.inf, key)
    ids = np.argsort(-key, axis=1, kind="stable")[:, :top]
    none = np.take_along_axis(masked, ids, 1)
    w = np.where(none, 0, np.take_along_axis(p, ids, 1))
    if renormalize:
        t = w.sum(axis=1, keepdims=True)
        w = w / np.where(t > 0, t, 1)
    ids = np.where(none, -1, ids)
    t, e = logits.shape
    flat = np.where(ids < 0, e, ids).reshape(-1)
    order = np.argsort(flat, kind="stable")
    pos = np.empty(t * top, dtype=np.int64)
    pos[order] = np.arange(t * top)
    offsets = np.searchsorted(flat[order], np.arange(e + 1))
    rows = np.where(flat[order] == e, -1, order)
    pos = np.where(flat == e, -1, pos).reshape(t, top)
    return ids, w * scale, offsets, pos, rows


def check_route(route, ref):
    for name, r in zip(("ids", "offsets", "positions", "rows"), (ref[0], ref[2], ref[3], ref[4])):
        assert np.array_equal(route[name].cpu().numpy(), r), name
    # exp, one division and at most 33 additions in FP32: 40 roundings of 2^-24.
    assert np.allclose(route["weights"].cpu().numpy(), ref[1], rtol=40 * 2.0 ** -24, atol=1e-30)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (1, 64, 6), (3, 8, 8), (16, 64, 6), (127, 33, 4), (128, 256, 8),
                                   (129, 256, 8), (1000, 60, 3), (2048, 512, 10), (300, 1024, 32)])
def test_route(cuda_device, t, e, k, scoring):
    rng = np.random.default_rng(t + e)
    logits = rng.standard_normal((t, e)).astype(np.float32)
    bias = (0.1 * rng.standard_normal(e)).astype(np.float32) if scoring == "sigmoid" else None
    r = launch_moe_route(torch.from_numpy(logits).to(cuda_device), k, scoring=scoring,
                         bias=None if bias is None else torch.from_numpy(bias).to(cuda_device), scale=2.5)
    check_route(r, route_ref(logits, k, scoring, bias, scale=2.5))


def test_route_ties_bf16_and_strides(cuda_device):
    rng = np.random.default_rng(0)
    logits = rng.integers(-2, 3, size=(200, 70)).astype(np.float32)  # many equal scores
    lg = torch.from_numpy(logits).to(cuda_device)
    ref = route_ref(logits, 5, renormalize=False)
    check_route(launch_moe_route(lg, 5, renormalize=False), ref)
    check_route(launch_moe_route(lg.bfloat16(), 5, renormalize=False), ref)
    wide = torch.zeros(200, 99, device=cuda_device)
    wide[:, 11:81] = lg
    check_route(launch_moe_route(wide[:, 11:81], 5, renormalize=False), ref)
    check_route(launch_moe_route(lg.t().contiguous().t(), 5, renormalize=False), ref)


def test_route_masks(cuda_device):
    """Masked experts, rows with nothing left, lowest values, infinities and NaN."""
    rng = np.random.default_rng(5)
    logits = rng.standard_normal((12, 40)).astype(np.float32)
    logits[0, :] = -np.inf
    logits[1, :] = np.nan
    logits[2, 3:] = -np.inf
    logits[3, ::2] = np.nan
    logits[4, :] = np.finfo(np.float32).min
    logits[5, 1:] = np.finfo(np.float32).min
    logits[6, 7] = np.inf
    logits[7, 7], logits[7, 9] = np.inf, np.inf
    logits[8, :] = -200.0
    for scoring in ("softmax", "sigmoid"):
        r = launch_moe_route(torch.from_numpy(logits).to(cuda_device), 6, scoring=scoring)
        ref = route_ref(logits, 6, scoring)
        if scoring == "sigmoid":
            # exp(200) is infinite in FP32: those weights are exactly 0 there.
            ref[1][8] = 0
            ref[1][4] = 0
            ref[1][5, 1:] = 0
            ref[1][5, 0] = 1
        check_route(r, ref)
    empty = launch_moe_route(torch.empty(0, 40, device=cuda_device), 6)
    assert empty["ids"].shape == (0, 6) and (empty["offsets"] == 0).all()


@pytest.mark.parametrize("h", [1, 37, 64, 2056])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_combine(cuda_device, h, dtype):
    rng = np.random.default_rng(h)
    t, e, k = 50, 16, 3
    logits = rng.standard_normal((t, e)).astype(np.float32)
    logits[7] = -np.inf
    logits[8, 1:] = -np.inf
    r = launch_moe_route(torch.from_numpy(logits).to(cuda_device), k)
    y = torch.from_numpy(rng.standard_normal((t * k, h)).astype(np.float32)).to(dtype)
    ids, w, _, pos, _ = route_ref(logits, k)
    y64 = y.double().numpy()
    ref = (np.where(pos[:, :, None] >= 0, y64[np.maximum(pos, 0)], 0) * w[:, :, None]).sum(axis=1)
    out = launch_moe_combine(y.to(cuda_device), r, out_dtype=torch.float32)
    assert np.allclose(out.cpu().numpy(), ref, rtol=1e-5, atol=1e-5)
    assert (out[7] == 0).all()
    out16 = launch_moe_combine(y.to(cuda_device), r)
    assert np.allclose(out16.double().cpu().numpy(), ref, rtol=2.0 ** -8, atol=1e-5)


def experts_ref(x, route, gu, gus, down, downs):
    """The path in float64 from the definition (route: route_ref's)."""
    ids, w = route[0], route[1]
    t, h = x.shape
    i, half = gu.shape[1] // 2, gus.shape[1] // 2
    xq = quantize64(x.astype(np.float64), 32)[0]
    out = np.zeros((t, h))
    for e in range(gu.shape[0]):
        tok, j = np.nonzero(ids == e)
        if len(tok) == 0:
            continue
        g = xq[tok] @ weight64(gu[e, :i], gus[e, :half]).T
        u = xq[tok] @ weight64(gu[e, i:], gus[e, half:]).T
        hq = quantize64(g / (1 + np.exp(-g)) * u, 32)[0]
        np.add.at(out, tok, w[tok, j][:, None] * (hq @ weight64(down[e], downs[e]).T))
    return out


def make_experts(e, h, i, seed):
    gu, _ = make_weight(2 * i, h, seed, experts=e)
    rng = np.random.default_rng(seed + 1)
    # Small enough that silu sees ordinary values.
    gus = (2.0 ** rng.uniform(-13, -11, size=(e, 2 * -(-i // 128), -(-h // 128)))).astype(np.float32)
    down, downs = make_weight(h, i, seed + 2, experts=e)
    return gu, gus, down, downs


# The E4M3 codes of h come from FP32 sums: a sum that is off by 1e-6 of its size moves a code (by 2^-4 of the value at
# most) when it lies that near to a rounding boundary, about one in 2e4, 5e-4 in the norm; bf16 rows add 2^-9.
EXPERTS_F32_TOL = 2e-3
EXPERTS_BF16_TOL = 2.0 ** -8 + EXPERTS_F32_TOL


@pytest.mark.parametrize("t,e,k,h,i", [(1, 8, 2, 128, 64), (1, 4, 1, 256, 128), (5, 8, 3, 200, 100), (32, 8, 2, 512, 384),
                                       (64, 16, 4, 384, 192), (300, 8, 3, 256, 320), (77, 32, 6, 1000, 136),
                                       (600, 4, 2, 640, 448), (2, 64, 8, 1024, 33)])
def test_experts(cuda_device, t, e, k, h, i):
    gu, gus, down, downs = make_experts(e, h, i, t + i)
    dev = cuda_device
    wg = prepare_fp8_block_fields(torch.from_numpy(gu).to(dev), torch.from_numpy(gus).to(dev), gate_up=True)
    wd = prepare_fp8_block_fields(torch.from_numpy(down).to(dev), torch.from_numpy(downs).to(dev))
    rng = np.random.default_rng(t)
    logits = rng.standard_normal((t, e)).astype(np.float32)
    if t > 4:
        logits[2] = -np.inf  # a token without experts
        logits[3, 1:] = -np.inf  # and one with a single one
    x = make_x(t, h, 3).bfloat16()
    route = launch_moe_route(torch.from_numpy(logits).to(dev), k)
    ref = experts_ref(x.float().numpy(), route_ref(logits, k), gu, gus, down, downs)
    out = fp8_moe_experts(x.to(dev), route, wg, wd, out_dtype=torch.float32)
    assert frob(out.cpu(), ref) < EXPERTS_F32_TOL
    assert torch.equal(out, fp8_moe_experts(x.to(dev), route, wg, wd, out_dtype=torch.float32))
    if t > 4:
        assert (out[2] == 0).all()
    out16 = fp8_moe_experts(x.to(dev), route, wg, wd)
    assert out16.dtype == torch.bfloat16 and frob(out16.float().cpu(), ref) < EXPERTS_BF16_TOL
    outf = fp8_moe_experts(x.float().to(dev), route, wg, wd, out_dtype=torch.float32)
    assert torch.equal(out, outf)


def test_experts_from_the_parts(cuda_device):
    """The layer put together from the public parts gives the same down rows and sum."""
    t, e, k, h, i = 40, 8, 2, 256, 128
    dev = cuda_device
    gu, gus, down, downs = make_experts(e, h, i, 4)
    wg = prepare_fp8_block_fields(torch.from_numpy(gu).to(dev), torch.from_numpy(gus).to(dev), gate_up=True)
    plain = prepare_fp8_block_fields(torch.from_numpy(gu).to(dev), torch.from_numpy(gus).to(dev))
    wd = prepare_fp8_block_fields(torch.from_numpy(down).to(dev), torch.from_numpy(downs).to(dev))
    x = make_x(t, h, 6).to(dev)
    route = launch_moe_route(torch.randn(t, e, generator=torch.Generator().manual_seed(0)).to(dev), k)
    xs = x[(route["rows"] // k).long()]
    a = fp8_block_grouped_linear(xs, route["offsets"], plain, act_group=32, out_dtype=torch.float32)
    hid = a[:, :i] / (1 + torch.exp(-a[:, :i])) * a[:, i:]
    y = fp8_block_grouped_linear(hid, route["offsets"], wd, act_group=32, out_dtype=torch.float32)
    out = launch_moe_combine(y, route, out_dtype=torch.float32)
    whole = fp8_moe_experts(x, route, wg, wd, out_dtype=torch.float32)
    assert frob(whole.cpu(), out.cpu()) < EXPERTS_F32_TOL


def test_refusals(cuda_device):
    dev = cuda_device
    gu, gus, down, downs = make_experts(4, 256, 128, 1)
    wg = prepare_fp8_block_fields(torch.from_numpy(gu).to(dev), torch.from_numpy(gus).to(dev), gate_up=True)
    wd = prepare_fp8_block_fields(torch.from_numpy(down).to(dev), torch.from_numpy(downs).to(dev))
    x, logits = torch.zeros(6, 256, device=dev), torch.zeros(6, 4, device=dev)
    r = launch_moe_route(logits, 2)
    r5 = launch_moe_route(torch.zeros(6, 5, device=dev), 2)
    bad = [
        lambda: launch_moe_route(logits, 0), lambda: launch_moe_route(logits, 5), lambda: launch_moe_route(logits.half(), 1),
        lambda: launch_moe_route(logits, 2, scoring="relu"), lambda: launch_moe_route(logits[0], 2),
        lambda: launch_moe_route(logits, 2, bias=torch.zeros(3, device=dev)), lambda: launch_moe_route(logits.cpu(), 2),
        lambda: launch_moe_route(torch.zeros(1, 2000, device=dev), 2), lambda: fp8_moe_experts(x[:5], r, wg, wd),
        lambda: fp8_moe_experts(x[:, :128], r, wg, wd), lambda: fp8_moe_experts(x, r, wd, wd),
        lambda: fp8_moe_experts(x, r, wg, wg), lambda: fp8_moe_experts(x, r5, wg, wd),
        lambda: fp8_moe_experts(x.half(), r, wg, wd), lambda: fp8_moe_experts(x, r, wg, wd, out_dtype=torch.float16),
        lambda: launch_moe_combine(x.half(), r), lambda: launch_moe_combine(x, r, out=torch.zeros(5, 256, device=dev)),
        lambda: fp8_moe_experts(x, {**r, "ids": r["ids"].long()}, wg, wd),
    ]
    for n, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {n} was accepted")
    with pytest.raises(TypeError):
        fp8_moe_experts(x, r, gu, wd)


@pytest.mark.parametrize("t,e,k,h,i", [(1, 8, 2, 4096, 64), (3, 8, 2, 4096, 64), (5, 4, 1, 256, 4096), (40, 2, 1, 2304, 130)])
def test_experts_split_along_k(cuda_device, t, e, k, h, i):
    """Few tiles of many K blocks: several CTAs share a tile, also where its epilogue forms the hidden activations."""
    gu, gus, down, downs = make_experts(e, h, i, t + i)
    dev = cuda_device
    wg = prepare_fp8_block_fields(torch.from_numpy(gu).to(dev), torch.from_numpy(gus).to(dev), gate_up=True)
    wd = prepare_fp8_block_fields(torch.from_numpy(down).to(dev), torch.from_numpy(downs).to(dev))
    logits = np.random.default_rng(t).standard_normal((t, e)).astype(np.float32)
    x = torch.zeros(t, h + 3, device=dev)
    x[:, 1:1 + h] = make_x(t, h, 3).to(dev) * 0.5
    x = x[:, 1:1 + h]
    route = launch_moe_route(torch.from_numpy(logits).to(dev), k)
    ref = experts_ref(x.cpu().numpy(), route_ref(logits, k), gu, gus, down, downs)
    out = fp8_moe_experts(x, route, wg, wd, out_dtype=torch.float32)
    assert frob(out.cpu(), ref) < EXPERTS_F32_TOL
    for _ in range(3):
        assert torch.equal(out, fp8_moe_experts(x, route, wg, wd, out_dtype=torch.float32))


def test_experts_in_a_graph(cuda_device):
    """Route and experts captured once and replayed on new inputs: nothing goes through the host."""
    dev = cuda_device
    t, e, k, h, i = 6, 16, 2, 256, 128
    gu, gus, down, downs = make_experts(e, h, i, 4)
    wg = prepare_fp8_block_fields(torch.from_numpy(gu).to(dev), torch.from_numpy(gus).to(dev), gate_up=True)
    wd = prepare_fp8_block_fields(torch.from_numpy(down).to(dev), torch.from_numpy(downs).to(dev))
    x, logits = torch.zeros(t, h, device=dev, dtype=torch.bfloat16), torch.zeros(t, e, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fp8_moe_experts(x, launch_moe_route(logits, k), wg, wd)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = fp8_moe_experts(x, launch_moe_route(logits, k), wg, wd)
    for seed in range(3):
        gen = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(t, h, generator=gen))
        logits.copy_(torch.randn(t, e, generator=gen))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, fp8_moe_experts(x, launch_moe_route(logits, k), wg, wd))


def test_example_layer(cuda_device):
    """The example's layer gives the sum of its shared and routed experts, computed in float64."""
    import sys

    from conftest import ROOT

    sys.path.insert(0, str(ROOT / "examples"))
    from fp8_expert_layer import ExpertLayer, random_fp8_weight

    hidden, features, experts, top = 256, 128, 8, 2
    layer = ExpertLayer(hidden, features, experts, top, seed=3)
    gen = torch.Generator(device="cuda").manual_seed(3)
    router = torch.randn((experts, hidden), generator=gen, device="cuda") / hidden ** 0.5
    plain = []
    for shape in ((2 * features, hidden), (hidden, features), (experts, 2 * features, hidden), (experts, hidden, features)):
        v, s = random_fp8_weight(shape, gen)
        plain.append((v.view(torch.uint8).cpu().numpy(), s.cpu().numpy()))
    x = torch.randn(20, hidden, device=cuda_device).bfloat16()
    xq = quantize64(x.double().cpu().numpy(), 128)[0]
    a = xq @ weight64(*plain[0]).T
    g, u = a[:, :features], a[:, features:]
    shared = quantize64(g / (1 + np.exp(-g)) * u, 128)[0] @ weight64(*plain[1]).T
    logits = (x.float() @ router.t()).cpu().numpy()
    routed = experts_ref(x.float().cpu().numpy(), route_ref(logits, top), *plain[2], *plain[3])
    # The shared hidden activations pass through bf16 here: two roundings of 2^-8 and the codes they move (2^-4 of
    # about 2^-8 / 2^-4 of them), under 2e-2 in the norm.
    assert frob(layer(x).float().cpu(), shared + routed) < 2e-2
