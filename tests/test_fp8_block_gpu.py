"""FP8 block-scaled linear, plain and grouped by expert, against float64 products of the same codes.

Tolerances. The quantizer's codes and scales are exact (the scale is a power
of two), so the product is compared on identical operands: products of two
E4M3 values are exact in FP32, and an FP32 sum of K of them, in any order,
is within K * 2^-24 of the sum of magnitudes; rounding errors of a sum of
random signs grow with sqrt(K) at most, and the relative Frobenius error stays
below sqrt(K) * 2^-23 plus the one rounding of the scale product (2^-24 per
block): 2e-5 for K up to 28672. A bf16 output has to equal the float32 output
of the same call, rounded once, bit for bit.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mambo_b200 import _lib
from mambo_b200.kernels.fp8_block import fp8_block_grouped_linear, fp8_block_linear, launch_fp8_block_matmul, \
    launch_quantize_fp8_block, prepare_fp8_block_fields
from mambo_b200.kernels.quantize_fp8 import launch_quantize_fp8

pytestmark = pytest.mark.gpu

F32_TOL = 2e-5


def e4m3_table() -> np.ndarray:
    b = np.arange(256)
    exp, man = (b >> 3) & 15, b & 7
    v = np.where(exp == 0, man * 2.0 ** -9, (8 + man) * 2.0 ** (exp - 10.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b & 128, -v, v)


def quantize64(x: np.ndarray, group: int):
    """(values, e) of x [M,K] from the definition: values / 2^e rounded to E4M3, ties to even, times 2^e."""
    m, k = x.shape
    g = -(-k // group)
    p = np.zeros((m, g * group))
    p[:, :k] = x
    p = p.reshape(m, g, group)
    amax = np.abs(p).max(axis=2)
    mant, exp = np.frexp(amax)  # amax = mant * 2^exp, 448 = 0.875 * 2^9
    e = np.where(amax == 0, 0, np.clip(exp - 9 + (mant > 0.875), -127, 127))
    v = p * 2.0 ** -e[:, :, None].astype(np.float64)
    step = 2.0 ** (np.maximum(np.frexp(v)[1] - 1, -6) - 3.0)
    v = np.clip(np.rint(v / step) * step, -448, 448)
    return (v * 2.0 ** e[:, :, None].astype(np.float64)).reshape(m, -1)[:, :k], e


def make_weight(n, k, seed, experts=None):
    rng = np.random.default_rng(seed)
    shape = (n, k) if experts is None else (experts, n, k)
    codes = rng.integers(0, 256, size=shape, dtype=np.uint8)
    codes[(codes & 127) == 127] = 0x38
    blocks = (-(-n // 128), -(-k // 128))
    scales = (2.0 ** rng.uniform(-9, -5, size=blocks if experts is None else (experts, *blocks))).astype(np.float32)
    return codes, scales


def weight64(codes, scales):
    n, k = codes.shape
    s = np.repeat(np.repeat(scales.astype(np.float64), 128, axis=0), 128, axis=1)[:n, :k]
    return e4m3_table()[codes] * s


def make_x(m, k, seed):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((m, k)).astype(np.float32)
    x[:, rng.permutation(k)[: max(1, k // 100)]] *= 40.0
    return torch.from_numpy(x)


def prepared(dev, codes, scales, **kw):
    return prepare_fp8_block_fields(torch.from_numpy(codes).to(dev), torch.from_numpy(scales).to(dev), **kw)


def frob(a, b):
    a, b = np.asarray(a, dtype=np.float64), np.asarray(b, dtype=np.float64)
    return float(np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-300))


def check(out, ref, tol=F32_TOL):
    assert out.dtype == torch.float32
    got = out.double().cpu().numpy()
    assert got.shape == ref.shape
    assert frob(got, ref) < tol
    # No row or column is off as a whole.
    for axis in (0, 1):
        num, den = np.linalg.norm(got - ref, axis=axis), np.linalg.norm(ref, axis=axis)
        assert (num <= 4 * tol * np.maximum(den, 1e-3 * den.max())).all()


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert _lib.device_status()[0] == 0


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 31), (2, 128), (5, 129), (1, 4096), (7, 1000), (130, 2500)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantizer_is_exact(cuda_device, m, k, group, dtype):
    x = make_x(m, k, m * 7 + k).to(dtype)
    x[0, :] *= 2.0 ** -20
    values, scales = launch_quantize_fp8_block(x.to(cuda_device), group=group)
    ref, e = quantize64(x.double().numpy(), group)
    assert np.array_equal(scales.cpu().numpy().astype(int) - 127, e)
    got = e4m3_table()[values.cpu().numpy()] * np.repeat(2.0 ** e.astype(np.float64), group, axis=1)[:, :k]
    assert np.array_equal(got, ref)
    if group == 32 and k % 32 == 0:
        v2, s2 = launch_quantize_fp8(x.to(cuda_device))
        assert torch.equal(values, v2) and torch.equal(scales, s2)


def test_quantizer_special_values(cuda_device):
    x = torch.zeros(5, 256)
    x[1, 5], x[2, 130], x[3, 0] = float("inf"), float("nan"), 2.0 ** -140
    x[4, 128:] = 448.0 * 2.0 ** 3
    v, s = launch_quantize_fp8_block(x.to(cuda_device))
    assert s.cpu().tolist() == [[127, 127], [255, 127], [127, 255], [0, 127], [127, 130]]
    assert (v.cpu()[0] == 0).all() and (v.cpu()[4, 128:] == 0x7E).all()


SHAPES = [(1, 128, 128), (1, 1, 1), (2, 100, 37), (1, 4096, 4096), (8, 1000, 520), (16, 256, 2048), (17, 384, 1024),
          (31, 129, 257), (32, 512, 4096), (33, 640, 384), (64, 300, 900), (65, 1024, 512), (100, 77, 3001),
          (128, 2048, 256), (129, 256, 640), (240, 512, 512), (241, 130, 1500), (300, 1000, 1000), (513, 896, 768),
          (1000, 1152, 640)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear(cuda_device, m, n, k):
    codes, scales = make_weight(n, k, n * 3 + k)
    w = prepared(cuda_device, codes, scales)
    w64 = weight64(codes, scales)
    for dtype, group in ((torch.bfloat16, 128), (torch.float32, 32), (torch.bfloat16, 32)):
        x = make_x(m, k, m + n + k).to(dtype)
        out = fp8_block_linear(x.to(cuda_device), w, act_group=group, out_dtype=torch.float32)
        check(out, quantize64(x.double().numpy(), group)[0] @ w64.T)
        out16 = fp8_block_linear(x.to(cuda_device), w, act_group=group)
        assert out16.dtype == torch.bfloat16 and torch.equal(out16, out.bfloat16())


@pytest.mark.parametrize("m,n,k", [(1, 14336, 4096), (8, 28672, 8192), (4, 4096, 28672), (48, 8192, 4096)])
def test_linear_long(cuda_device, m, n, k):
    """Many K blocks and row tiles: ranges that cross tiles, tiles shared by several CTAs."""
    codes, scales = make_weight(n, k, 11)
    w = prepared(cuda_device, codes, scales)
    x = make_x(m, k, 5).bfloat16()
    ref = quantize64(x.double().numpy(), 128)[0] @ weight64(codes, scales).T
    out = [fp8_block_linear(x.to(cuda_device), w, out_dtype=torch.float32) for _ in range(3)]
    check(out[0], ref)
    # The same sums in the same order on every call, whichever CTA arrives last.
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])


@pytest.mark.parametrize("m,n,k", [(1, 256, 512), (50, 200, 300), (200, 512, 1024)])
def test_prequantized_equals_fused(cuda_device, m, n, k):
    codes, scales = make_weight(n, k, 3)
    w = prepared(cuda_device, codes, scales)
    x = make_x(m, k, 9).to(cuda_device)
    for group in (32, 128):
        v, s = launch_quantize_fp8_block(x, group=group)
        a = launch_fp8_block_matmul(v, s, w)
        b = fp8_block_linear(x, w, act_group=group, out_dtype=torch.float32)
        assert torch.equal(a, b)


def test_strides_alignment_and_out(cuda_device):
    m, n, k = 37, 260, 520
    codes, scales = make_weight(n, k, 21)
    dev = cuda_device
    wide = torch.zeros(n + 3, k + 5, dtype=torch.uint8, device=dev)
    wide[2:2 + n, 3:3 + k] = torch.from_numpy(codes).to(dev)
    w = prepare_fp8_block_fields(wide[2:2 + n, 3:3 + k].view(torch.float8_e4m3fn), torch.from_numpy(scales).to(dev).t().contiguous().t())
    wt = prepare_fp8_block_fields(torch.from_numpy(codes).to(dev).t().contiguous().t(), torch.from_numpy(scales).to(dev))
    assert torch.equal(w["packed"], wt["packed"]) and torch.equal(w["scales"], wt["scales"])
    ref = None
    for dtype in (torch.bfloat16, torch.float32):
        x = make_x(m, k, 2).to(dtype)
        ref = quantize64(x.double().numpy(), 128)[0] @ weight64(codes, scales).T
        xs = torch.zeros(m, k + 7, dtype=dtype, device=dev)
        xs[:, 3:3 + k] = x.to(dev)
        check(fp8_block_linear(xs[:, 3:3 + k], w, out_dtype=torch.float32), ref)
        check(fp8_block_linear(x.to(dev).t().contiguous().t(), w, out_dtype=torch.float32), ref)
    out = torch.full((m, n + 9), 7.0, device=dev)
    res = fp8_block_linear(x.to(dev), w, out=out[:, 5:5 + n])
    assert res.data_ptr() == out[:, 5:5 + n].data_ptr()
    check(res, ref)
    assert (out[:, :5] == 7).all() and (out[:, 5 + n:] == 7).all()
    # On a stream that is not the current one.
    side = torch.cuda.Stream()
    xg = x.to(dev)
    side.wait_stream(torch.cuda.current_stream())
    res = fp8_block_linear(xg, w, out_dtype=torch.float32, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    check(res, ref)


def test_special_values(cuda_device):
    """NaN and infinity stay in their row; a NaN weight code stays in its column; zeros give zeros."""
    m, n, k = 20, 200, 300
    codes, scales = make_weight(n, k, 4)
    codes[7, 100] = 0x7F
    w = prepared(cuda_device, codes, scales)
    x = make_x(m, k, 8)
    x[3, 5], x[4, 290], x[9] = float("nan"), float("inf"), 0.0
    out = fp8_block_linear(x.to(cuda_device), w, out_dtype=torch.float32).cpu()
    bad = torch.isnan(out)
    assert bad[3].all() and bad[4].all() and bad[:, 7].all()
    keep_rows = [r for r in range(m) if r not in (3, 4)]
    keep_cols = [c for c in range(n) if c != 7]
    good = out[keep_rows][:, keep_cols]
    assert torch.isfinite(good).all()
    assert (out[9, keep_cols] == 0).all()
    x2 = x.clone()
    x2[3], x2[4] = 0, 0
    ref = (quantize64(x2.double().numpy(), 128)[0] @ weight64(np.where(codes == 0x7F, 0, codes), scales).T)
    check(good, ref[keep_rows][:, keep_cols])


def test_wide_scales(cuda_device):
    """Activation scales over the UE8M0 range and block scales of any sign and size, zero included."""
    m, n, k = 9, 256, 640
    codes, _ = make_weight(n, k, 6)
    scales = np.array([[2.0 ** -60, -3.7, 0.0, 2.0 ** 40, 1.0], [1e-20, 1e20, 5.0, -2.0 ** -30, 0.3]], dtype=np.float32)
    w = prepared(cuda_device, codes, scales)
    x = make_x(m, k, 3) * torch.tensor([2.0 ** e for e in (-100, -60, -20, 0, 10, 20, 25, -126, 1)])[:, None]
    out = fp8_block_linear(x.to(cuda_device), w, out_dtype=torch.float32)
    ref = quantize64(x.double().numpy(), 128)[0] @ weight64(codes, scales).T
    got = out.double().cpu().numpy()
    for r in range(m - 2):
        assert frob(got[r, 128:], ref[r, 128:]) < F32_TOL and frob(got[r, :128], ref[r, :128]) < F32_TOL


def test_graph_capture_and_empty(cuda_device):
    n, k = 512, 1024
    codes, scales = make_weight(n, k, 13)
    w = prepared(cuda_device, codes, scales)
    x = make_x(5, k, 1).bfloat16().to(cuda_device)
    ref = fp8_block_linear(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fp8_block_linear(x, w)  # the stream's workspace exists before the capture
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = fp8_block_linear(x, w)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref)
    assert fp8_block_linear(x[:0], w).shape == (0, n)
    assert launch_quantize_fp8_block(x[:0])[0].shape == (0, k)


def _grouped_ref(x, offsets, codes, scales, group):
    xq = quantize64(x.double().numpy(), group)[0]
    return np.concatenate([xq[offsets[e]:offsets[e + 1]] @ weight64(codes[e], scales[e]).T
                           for e in range(len(offsets) - 1)])


GROUPED = [
    ([5], 128, 256), ([0, 3, 0, 1, 0], 200, 300), ([1] * 33, 128, 128), ([0, 0, 0, 70], 300, 512),
    ([16, 17, 15, 0, 129, 1, 64], 256, 640), ([300, 0, 2, 500, 33], 384, 384), ([8] * 64, 130, 257),
    ([1000, 7], 512, 256), ([0] * 40 + [2] + [0] * 60 + [9] * 3, 256, 512), ([241, 239, 480, 16], 640, 1100),
]


@pytest.mark.parametrize("counts,n,k", GROUPED, ids=range(len(GROUPED)))
def test_grouped(cuda_device, counts, n, k):
    offsets = np.concatenate([[0], np.cumsum(counts)])
    codes, scales = make_weight(n, k, 17, experts=len(counts))
    w = prepared(cuda_device, codes, scales)
    off = torch.tensor(offsets, dtype=torch.int32, device=cuda_device)
    for dtype, group in ((torch.bfloat16, 128), (torch.float32, 32)):
        x = make_x(int(offsets[-1]), k, 23).to(dtype)
        out = fp8_block_grouped_linear(x.to(cuda_device), off, w, act_group=group, out_dtype=torch.float32)
        check(out, _grouped_ref(x, offsets, codes, scales, group))
        out16 = fp8_block_grouped_linear(x.to(cuda_device), off, w, act_group=group)
        assert out16.dtype == torch.bfloat16 and torch.equal(out16, out.bfloat16())


def test_grouped_equals_single(cuda_device):
    """Each segment as one linear of its own gives the same sums (the K split differs, so not the same bits)."""
    counts, n, k = [40, 0, 3, 200], 256, 1024
    offsets = np.concatenate([[0], np.cumsum(counts)])
    codes, scales = make_weight(n, k, 5, experts=4)
    w = prepared(cuda_device, codes, scales)
    x = make_x(243, k, 2).to(cuda_device)
    out = fp8_block_grouped_linear(x, torch.tensor(offsets, dtype=torch.int32, device=cuda_device), w, out_dtype=torch.float32)
    for e, c in enumerate(counts):
        if c:
            one = fp8_block_linear(x[offsets[e]:offsets[e + 1]], prepared(cuda_device, codes[e], scales[e]), out_dtype=torch.float32)
            assert frob(out[offsets[e]:offsets[e + 1]].cpu(), one.cpu()) < F32_TOL


def test_grouped_bad_offsets_stay_in_bounds(cuda_device):
    """Offsets that decrease, are negative or pass the rows are clamped: covered rows only, nothing else written."""
    n, k, rows = 128, 256, 20
    codes, scales = make_weight(n, k, 5, experts=3)
    w = prepared(cuda_device, codes, scales)
    x = make_x(rows, k, 2).to(cuda_device)
    for off in ([0, 5, 2, 20], [-7, 4, 900, 30], [3, 3, 3, 10], [0, 0, 0, 0], [20, 20, 20, 20]):
        guard = torch.full((rows + 8, n), 3.0, device=cuda_device)
        fp8_block_grouped_linear(x, torch.tensor(off, dtype=torch.int32, device=cuda_device), w, out=guard[4:4 + rows])
        torch.cuda.synchronize()
        assert (guard[:4] == 3).all() and (guard[4 + rows:] == 3).all()
    guard = torch.full((rows, n), 3.0, device=cuda_device)
    off = np.array([2, 5, 5, 9])
    fp8_block_grouped_linear(x, torch.tensor(off, dtype=torch.int32, device=cuda_device), w, out=guard)
    assert (guard[:2] == 3).all() and (guard[9:] == 3).all()
    xq = quantize64(x.double().cpu().numpy(), 128)[0]
    check(guard[2:5], xq[2:5] @ weight64(codes[0], scales[0]).T)
    check(guard[5:9], xq[5:9] @ weight64(codes[2], scales[2]).T)


def test_refusals(cuda_device):
    codes, scales = make_weight(256, 256, 1)
    c, s = torch.from_numpy(codes).to(cuda_device), torch.from_numpy(scales).to(cuda_device)
    w = prepare_fp8_block_fields(c, s)
    x = torch.zeros(4, 256, device=cuda_device)
    bad = [
        lambda: prepare_fp8_block_fields(c.int(), s), lambda: prepare_fp8_block_fields(c, s[:1]),
        lambda: prepare_fp8_block_fields(c, s.double()), lambda: prepare_fp8_block_fields(c[:255], s, gate_up=True),
        lambda: prepare_fp8_block_fields(c, s[None]), lambda: fp8_block_linear(x.half(), w),
        lambda: fp8_block_linear(x[:, :128], w), lambda: fp8_block_linear(x, w, act_group=64),
        lambda: fp8_block_linear(x, w, out_dtype=torch.float16), lambda: fp8_block_linear(x.cpu(), w),
        lambda: fp8_block_linear(x, w, out=torch.zeros(4, 255, device=cuda_device)),
        lambda: fp8_block_linear(x, w, out=torch.zeros(256, 4, device=cuda_device).t()),
        lambda: launch_quantize_fp8_block(x, group=16), lambda: launch_fp8_block_matmul(x, x, w),
        lambda: launch_fp8_block_matmul(x.byte(), x.byte()[:, :3], w),
        lambda: fp8_block_grouped_linear(x, torch.zeros(3, dtype=torch.int32, device=cuda_device), w),
        lambda: fp8_block_grouped_linear(x, torch.zeros(2, dtype=torch.int64, device=cuda_device), w),
        lambda: fp8_block_linear(x, prepare_fp8_block_fields(c, s, gate_up=True)),
        lambda: fp8_block_linear(x, prepare_fp8_block_fields(c[None].repeat(2, 1, 1), s[None].repeat(2, 1, 1))),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was accepted")
    with pytest.raises(TypeError):
        fp8_block_linear(x, c)


@pytest.mark.parametrize("m,n,k", [(192, 256, 128), (193, 300, 200), (385, 4100, 256), (2000, 3000, 640),
                                   (4096, 1030, 384), (200, 512, 8192), (100, 130, 6000), (1, 20000, 300), (2, 9000, 777)])
def test_linear_waves_and_splits(cuda_device, m, n, k):
    """Several waves of pair tiles, pair tiles split along K, row groups past a block of 8, one and two tokens."""
    codes, scales = make_weight(n, k, m + 1)
    w = prepared(cuda_device, codes, scales)
    x = make_x(m, k, n).bfloat16()
    ref = quantize64(x.double().numpy(), 128)[0] @ weight64(codes, scales).T
    out = fp8_block_linear(x.to(cuda_device), w, out_dtype=torch.float32)
    check(out, ref)
    assert torch.equal(out, fp8_block_linear(x.to(cuda_device), w, out_dtype=torch.float32))
    assert torch.equal(out.bfloat16(), fp8_block_linear(x.to(cuda_device), w))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [1, 2])
def test_one_and_two_tokens_equal_the_quantizer(cuda_device, m, dtype):
    """The product's own quantization of one or two tokens gives what the quantizer gives, whatever the rows' alignment."""
    n, k = 300, 1003
    codes, scales = make_weight(n, k, 2)
    w = prepared(cuda_device, codes, scales)
    wide = torch.zeros(m, k + 9, dtype=dtype, device=cuda_device)
    wide[:, 5:5 + k] = make_x(m, k, 1).to(dtype).to(cuda_device)
    x = wide[:, 5:5 + k]
    for group in (32, 128):
        v, s = launch_quantize_fp8_block(x, group=group)
        assert torch.equal(fp8_block_linear(x, w, act_group=group, out_dtype=torch.float32), launch_fp8_block_matmul(v, s, w))
    off = torch.tensor([0, 0, m], dtype=torch.int32, device=cuda_device)
    w2 = prepared(cuda_device, np.stack([codes, codes]), np.stack([scales, scales]))
    assert torch.equal(fp8_block_grouped_linear(x, off, w2), fp8_block_linear(x, w))


def test_more_than_2_31_elements(cuda_device):
    """Output and weight offsets past 32 bits."""
    dev = cuda_device
    codes, scales = make_weight(8192, 128, 3)
    w = prepared(dev, codes, scales)
    m = 300_000
    x = torch.randn(m, 128, device=dev, dtype=torch.bfloat16)
    out = fp8_block_linear(x, w)
    assert out.numel() > 2 ** 31
    for a in (0, 131_072, m - 40):
        # Which tokens share a tile does not change a sum of one K block.
        assert torch.equal(out[a:a + 40], fp8_block_linear(x[a:a + 40].contiguous(), w))
    del out, x
    experts, n, k = 40, 8192, 8192
    big = torch.randint(0, 120, (experts, n, k), dtype=torch.uint8, device=dev)
    s = torch.full((experts, 64, 64), 2.0 ** -8, device=dev)
    wg = prepare_fp8_block_fields(big, s)
    x = torch.randn(experts * 3, k, device=dev, dtype=torch.bfloat16)
    off = torch.arange(experts + 1, dtype=torch.int32, device=dev) * 3
    out = fp8_block_grouped_linear(x, off, wg, out_dtype=torch.float32)
    for e in (0, 39):
        one = fp8_block_linear(x[3 * e:3 * e + 3], prepare_fp8_block_fields(big[e], s[e]), out_dtype=torch.float32)
        assert frob(out[3 * e:3 * e + 3].cpu(), one.cpu()) < F32_TOL
