"""A feed-forward layer with a shared FP8 expert and routed FP8 experts, on the framework's FP8 block operators.

    python examples/fp8_expert_layer.py [--tokens 4 512] [--hidden 2048] [--features 1408] [--experts 64] [--top 6]

Random weights in the form FP8 checkpoints have (E4M3 values, one float32 scale
per 128 x 128 block) are prepared once; each call then runs

    h = silu(x Wg^T) * (x Wu^T)        fp8_block_linear (the shared expert)
    shared = h Wd^T                    fp8_block_linear
    route = top experts of x Wr^T      launch_moe_route
    routed = sum of their outputs      fp8_moe_experts

and is timed as a CUDA graph.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from mambo_b200.kernels.fp8_block import fp8_block_linear, prepare_fp8_block_fields  # noqa: E402
from mambo_b200.kernels.moe_fp8 import fp8_moe_experts, launch_moe_route  # noqa: E402


def random_fp8_weight(shape: tuple[int, ...], gen: torch.Generator) -> tuple[torch.Tensor, torch.Tensor]:
    """Normal weights [..., N, K] as E4M3 values and block scales (N and K multiples of 128)."""
    n, k = shape[-2:]
    w = torch.randn(shape, generator=gen, device="cuda") / k ** 0.5
    blocks = w.view(*shape[:-2], n // 128, 128, k // 128, 128)
    scales = blocks.abs().amax(dim=(-3, -1)) / 448.0
    values = (blocks / scales[..., :, None, :, None]).view(shape).to(torch.float8_e4m3fn)
    return values, scales


class ExpertLayer:
    def __init__(self, hidden: int, features: int, experts: int, top: int, seed: int = 0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.top = top
        self.router = torch.randn((experts, hidden), generator=gen, device="cuda") / hidden ** 0.5
        self.shared_up = prepare_fp8_block_fields(*random_fp8_weight((2 * features, hidden), gen))
        self.shared_down = prepare_fp8_block_fields(*random_fp8_weight((hidden, features), gen))
        self.gate_up = prepare_fp8_block_fields(*random_fp8_weight((experts, 2 * features, hidden), gen), gate_up=True)
        self.down = prepare_fp8_block_fields(*random_fp8_weight((experts, hidden, features), gen))

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        # float32 until it is quantized again: rounded to bf16 first, one E4M3 code in twenty would be another.
        gate, up = fp8_block_linear(x, self.shared_up, out_dtype=torch.float32).chunk(2, dim=1)
        shared = fp8_block_linear(torch.nn.functional.silu(gate) * up, self.shared_down)
        route = launch_moe_route(x.float() @ self.router.t(), self.top)
        return shared + fp8_moe_experts(x, route, self.gate_up, self.down)


def time_us(layer: ExpertLayer, x: torch.Tensor, reps: int = 20) -> float:
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        layer(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            layer(x)
        for _ in range(3):
            graph.replay()
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record(stream)
        for _ in range(reps):
            graph.replay()
        end.record(stream)
    end.synchronize()
    return start.elapsed_time(end) * 1e3 / reps


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--tokens", type=int, nargs="+", default=[1, 16, 512])
    ap.add_argument("--hidden", type=int, default=2048)
    ap.add_argument("--features", type=int, default=1408)
    ap.add_argument("--experts", type=int, default=64)
    ap.add_argument("--top", type=int, default=6)
    args = ap.parse_args()
    layer = ExpertLayer(args.hidden, args.features, args.experts, args.top)
    for tokens in args.tokens:
        x = torch.randn((tokens, args.hidden), device="cuda", dtype=torch.bfloat16)
        out = layer(x)
        assert out.shape == x.shape and torch.isfinite(out).all()
        print(f"{tokens:6d} tokens  {time_us(layer, x):9.1f} us  output rms {out.float().square().mean().sqrt():.3f}")


if __name__ == "__main__":
    main()
