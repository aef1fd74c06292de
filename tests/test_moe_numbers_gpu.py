"""Numbers of the routed experts and the grouped product that the smaller tests leave open.

Tolerances. One rounding to bf16 is uniform over a step of 2^-7 of the value's power of two, so its error is at most
2^-7 / sqrt(12) = 2.26e-3 of the norm; two independent ones add up in squares to 3.19e-3. An FP32 sum that is off by
1e-6 of its size moves about one E4M3 code of the hidden activations in 2e4 by 2^-4 at most: 5e-4 of the norm.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mambo_b200 import _lib
from mambo_b200.kernels.fp8_block import fp8_block_grouped_linear, fp8_block_linear, prepare_fp8_block_fields
from mambo_b200.kernels.moe_fp8 import fp8_moe_experts, launch_moe_route
from test_fp8_block_gpu import F32_TOL, check, frob, make_weight, make_x, quantize64, weight64
from test_moe_fp8_gpu import experts_ref, make_experts, route_ref

pytestmark = pytest.mark.gpu

ROUNDING = 2.0 ** -7 / 12 ** 0.5
CODES = 5e-4


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert _lib.device_status()[0] == 0


def on(dev, *arrays):
    return [torch.from_numpy(a).to(dev) for a in arrays]


def prepared_experts(dev, gu, gus, down, downs):
    return prepare_fp8_block_fields(*on(dev, gu, gus), gate_up=True), prepare_fp8_block_fields(*on(dev, down, downs))


@pytest.mark.parametrize("t,e,k,h,i", [(1, 16, 6, 512, 256), (20, 8, 2, 640, 384), (400, 8, 4, 384, 256)])
def test_roundings_of_a_bf16_result(cuda_device, t, e, k, h, i):
    """A bf16 result carries two roundings, a float32 one that is rounded afterwards a single one."""
    parts = make_experts(e, h, i, t)
    wg, wd = prepared_experts(cuda_device, *parts)
    logits = np.random.default_rng(t).standard_normal((t, e)).astype(np.float32)
    x = make_x(t, h, 4).bfloat16()
    route = launch_moe_route(torch.from_numpy(logits).to(cuda_device), k)
    ref = experts_ref(x.float().numpy(), route_ref(logits, k), *parts)
    one = fp8_moe_experts(x.to(cuda_device), route, wg, wd, out_dtype=torch.float32).bfloat16()
    two = fp8_moe_experts(x.to(cuda_device), route, wg, wd)
    assert frob(one.float().cpu(), ref) < (ROUNDING ** 2 + CODES ** 2) ** 0.5
    assert frob(two.float().cpu(), ref) < (2 * ROUNDING ** 2 + CODES ** 2) ** 0.5


def experts_on_gpu(x, ids, weights, gu, gus, down, downs, tokens):
    """experts_ref for some tokens, on the GPU in float64."""
    half, i = gus.shape[1] // 2, gu.shape[1] // 2
    xq = torch.from_numpy(quantize64(x[tokens].astype(np.float64), 32)[0]).cuda()
    out = torch.zeros(len(tokens), x.shape[1], dtype=torch.float64, device="cuda")
    for e in range(gu.shape[0]):
        tok, j = np.nonzero(ids[tokens] == e)
        if len(tok):
            g = xq[tok] @ torch.from_numpy(weight64(gu[e, :i], gus[e, :half])).cuda().T
            u = xq[tok] @ torch.from_numpy(weight64(gu[e, i:], gus[e, half:])).cuda().T
            hq = torch.from_numpy(quantize64((g / (1 + torch.exp(-g)) * u).cpu().numpy(), 32)[0]).cuda()
            y = hq @ torch.from_numpy(weight64(down[e], downs[e])).cuda().T
            out.index_add_(0, torch.from_numpy(tok).cuda(), torch.from_numpy(weights[tokens][tok, j]).cuda()[:, None] * y)
    return out.cpu().numpy()


@pytest.mark.parametrize("t,e,k,h,i,skew", [(5000, 16, 4, 512, 384, False), (3000, 8, 2, 1024, 200, True),
                                            (1024, 64, 1, 384, 128, True)])
def test_experts_many_tokens(cuda_device, t, e, k, h, i, skew):
    """Many waves of tiles; with skew one expert has every token."""
    parts = make_experts(e, h, i, k)
    wg, wd = prepared_experts(cuda_device, *parts)
    rng = np.random.default_rng(e)
    logits = rng.standard_normal((t, e)).astype(np.float32)
    if skew:
        logits[:, 3] = 50.0
    x = make_x(t, h, 8).bfloat16()
    route = launch_moe_route(torch.from_numpy(logits).to(cuda_device), k)
    ids, weights = route_ref(logits, k)[:2]
    out = fp8_moe_experts(x.to(cuda_device), route, wg, wd, out_dtype=torch.float32)
    tokens = np.sort(rng.permutation(t)[:400])
    ref = experts_on_gpu(x.float().numpy(), ids, weights, *parts, tokens)
    got = out.cpu().numpy()[tokens]
    assert frob(got, ref) < CODES + F32_TOL
    # No token is off as a whole (a moved code or two weigh more in one row than in all).
    assert (np.linalg.norm(got - ref, axis=1) < 2.0 ** -5 * np.linalg.norm(ref, axis=1)).all()
    assert torch.equal(out, fp8_moe_experts(x.to(cuda_device), route, wg, wd, out_dtype=torch.float32))


def test_grouped_many_rows(cuda_device):
    counts, n, k = [900, 0, 2500, 1, 40, 3000, 192, 193, 700], 520, 640
    offsets = np.concatenate([[0], np.cumsum(counts)])
    codes, scales = make_weight(n, k, 31, experts=len(counts))
    w = prepare_fp8_block_fields(*on(cuda_device, codes, scales))
    x = make_x(int(offsets[-1]), k, 12).bfloat16()
    out = fp8_block_grouped_linear(x.to(cuda_device), torch.tensor(offsets, dtype=torch.int32, device=cuda_device), w,
                                   out_dtype=torch.float32)
    xq = quantize64(x.double().numpy(), 128)[0]
    check(out, np.concatenate([xq[offsets[e]:offsets[e + 1]] @ weight64(codes[e], scales[e]).T for e in range(len(counts))]))


@pytest.mark.parametrize("rows", [2, 24, 500])
def test_grouped_special_values(cuda_device, rows):
    """NaN and infinity stay in their row, a NaN weight code in its expert and column."""
    experts, n, k = 3, 200, 300
    codes, scales = make_weight(n, k, 4, experts=experts)
    codes[2, 7, 100] = 0x7F
    first = rows // 2
    offsets = torch.tensor([0, first, first, rows], dtype=torch.int32, device=cuda_device)
    w = prepare_fp8_block_fields(*on(cuda_device, codes, scales))
    x = make_x(rows, k, 8)
    bad_rows = {0: float("nan"), rows - 1: float("inf")} if rows > 2 else {0: float("nan")}
    for r, v in bad_rows.items():
        x[r, 290 % k] = v
    got = fp8_block_grouped_linear(x.to(cuda_device), offsets, w, out_dtype=torch.float32).cpu().numpy()
    expect_nan = np.zeros((rows, n), dtype=bool)
    expect_nan[list(bad_rows)] = True
    expect_nan[first:, 7] = True
    assert np.array_equal(np.isnan(got), expect_nan) and np.isfinite(got[~expect_nan]).all()
    xq = quantize64(np.nan_to_num(x.double().numpy(), nan=0.0, posinf=0.0), 128)[0]
    clean = np.where(codes == 0x7F, 0, codes)
    ref = np.concatenate([xq[:first] @ weight64(clean[0], scales[0]).T, xq[first:] @ weight64(clean[2], scales[2]).T])
    assert frob(np.where(expect_nan, 0, got), np.where(expect_nan, 0, ref)) < F32_TOL


@pytest.mark.parametrize("t", [1, 2, 9, 40, 700])
@pytest.mark.parametrize("what", ["nan", "inf", "overflow"])
def test_experts_special_values(cuda_device, what, t):
    """NaN, infinity and hidden activations past FP32 give NaN to their tokens; the others' values do not change."""
    e, k, h, i = 6, 2, 320, 160
    gu, gus, down, downs = make_experts(e, h, i, 5)
    rng = np.random.default_rng(t)
    logits = rng.standard_normal((t, e)).astype(np.float32)
    if t == 1:
        logits[0, 4] = 9.0
    ids = route_ref(logits, k)[0]
    x = make_x(t, h, 3)
    plain = fp8_moe_experts(x.to(cuda_device), launch_moe_route(torch.from_numpy(logits).to(cuda_device), k),
                            *prepared_experts(cuda_device, gu, gus, down, downs), out_dtype=torch.float32).cpu().numpy()
    bad = np.zeros(t, dtype=bool)
    if what == "overflow":
        gus = gus.copy()
        gus[4] *= np.float32(2.0 ** 100)  # gate and up of expert 4 near 2^100: their product is infinite
        bad = (ids == 4).any(axis=1)
    else:
        bad[t // 2] = True
        x[t // 2, 77] = float(what)
    out = fp8_moe_experts(x.to(cuda_device), launch_moe_route(torch.from_numpy(logits).to(cuda_device), k),
                          *prepared_experts(cuda_device, gu, gus, down, downs), out_dtype=torch.float32).cpu().numpy()
    assert bad.any()
    assert np.isnan(out[bad]).all()
    assert np.array_equal(out[~bad], plain[~bad])


def test_wide_scales_of_every_row(cuda_device):
    """Activation scales over the UE8M0 range, every row checked.

    A row of 2^-126 has products down to 2^-127 * 2^-9 * 2^-9 times the weight scale, below the smallest normal number;
    sums of such may lose up to 2^-126 an addition, K of them, times the weight scale of the block.
    """
    m, n, k = 9, 256, 640
    codes, _ = make_weight(n, k, 6)
    scales = np.array([[2.0 ** -60, -3.7, 0.0, 2.0 ** 40, 1.0], [1e-20, 1e20, 5.0, -2.0 ** -30, 0.3]], dtype=np.float32)
    w = prepare_fp8_block_fields(*on(cuda_device, codes, scales))
    x = make_x(m, k, 3) * torch.tensor([2.0 ** e for e in (-100, -60, -20, 0, 10, 20, 25, -126, 1)])[:, None]
    got = fp8_block_linear(x.to(cuda_device), w, out_dtype=torch.float32).double().cpu().numpy()
    ref = quantize64(x.double().numpy(), 128)[0] @ weight64(codes, scales).T
    lost = 128 * 2.0 ** -126 * np.repeat(np.abs(scales.astype(np.float64)).sum(axis=1), 128)
    for r in range(m):
        for half in (slice(0, 128), slice(128, 256)):
            assert np.linalg.norm(got[r, half] - ref[r, half]) < F32_TOL * np.linalg.norm(ref[r, half]) \
                + np.linalg.norm(lost[half]), (r, half)


def test_example_layer_seeded(cuda_device):
    """The example's layer on given inputs: three roundings to bf16 (shared, routed rows, their sums) and moved codes.

    The shared and the routed half are rounded each (the routed one twice) and their sum once more: at most
    sqrt(3) roundings of the larger norms; a code of either half moves as above.
    """
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
    x = torch.randn(200, hidden, generator=torch.Generator().manual_seed(11)).bfloat16().to(cuda_device)
    xq = quantize64(x.double().cpu().numpy(), 128)[0]
    a = xq @ weight64(*plain[0]).T
    g, u = a[:, :features], a[:, features:]
    shared = quantize64(g / (1 + np.exp(-g)) * u, 128)[0] @ weight64(*plain[1]).T
    logits = (x.float() @ router.t()).cpu().numpy()
    routed = experts_ref(x.float().cpu().numpy(), route_ref(logits, top), *plain[2], *plain[3])
    norm = np.linalg.norm
    bound = ((norm(shared) ** 2 + 2 * norm(routed) ** 2 + norm(shared + routed) ** 2) * ROUNDING ** 2) ** 0.5 \
        + CODES * (norm(shared) + norm(routed))
    assert norm(layer(x).double().cpu().numpy() - shared - routed) < bound
