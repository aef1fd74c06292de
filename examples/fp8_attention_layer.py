"""An attention layer over a paged FP8 key/value cache, on the framework's FP8 block operators.

    python examples/fp8_attention_layer.py [--hidden 4096] [--heads 32] [--kv-heads 8] [--context 4096] [--batch 16]

Random weights in the form FP8 checkpoints have are prepared once; each step then runs

    q, k, v = x Wqkv^T                 fp8_block_linear
    q turned by its positions          launch_rotary
    k turned, k and v to their pages   launch_fp8_kv_append
    attention over the cache           fp8_paged_attention
    out = attention Wo^T               fp8_block_linear

first on a prompt of every sequence, then on single tokens, which are timed as a CUDA graph.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
sys.path.insert(0, str(Path(__file__).resolve().parent))

from fp8_expert_layer import random_fp8_weight  # noqa: E402
from mambo_b200.kernels.attention_fp8 import fp8_paged_attention, launch_fp8_kv_append, prepare_fp8_kv_cache  # noqa: E402
from mambo_b200.kernels.fp8_block import fp8_block_linear, prepare_fp8_block_fields  # noqa: E402
from mambo_b200.kernels.rotary import launch_rotary, prepare_rotary_fields  # noqa: E402


class AttentionLayer:
    def __init__(self, hidden: int, heads: int, kv_heads: int, head_dim: int, batch: int, most: int, page: int = 64,
                 seed: int = 0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.sizes = (heads, kv_heads, head_dim)
        self.qkv = prepare_fp8_block_fields(*random_fp8_weight(((heads + 2 * kv_heads) * head_dim, hidden), gen))
        self.out = prepare_fp8_block_fields(*random_fp8_weight((hidden, heads * head_dim), gen))
        self.rope = prepare_rotary_fields(head_dim, base=500000.0)
        columns = -(-most // page)
        self.cache = prepare_fp8_kv_cache(batch * columns, kv_heads, page, head_dim)
        self.table = torch.randperm(batch * columns, generator=gen, device="cuda").int().view(batch, columns)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")

    def __call__(self, x: torch.Tensor, positions: torch.Tensor, offsets: torch.Tensor | None = None) -> torch.Tensor:
        """x [T, hidden]: the next tokens of every sequence, those of sequence b from ``offsets[b]`` on."""
        heads, kv_heads, dim = self.sizes
        parts = fp8_block_linear(x, self.qkv).view(len(x), heads + 2 * kv_heads, dim)
        q, k, v = parts.split([heads, kv_heads, kv_heads], dim=1)
        q = launch_rotary(q, positions, self.rope)
        launch_fp8_kv_append(self.cache, k, v, self.table, self.lengths, offsets=offsets, rope=self.rope)
        self.lengths += 1 if offsets is None else offsets[1:] - offsets[:-1]
        attended = fp8_paged_attention(q, self.cache, self.table, self.lengths, offsets=offsets)
        return fp8_block_linear(attended.view(len(x), heads * dim), self.out)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("hidden", 4096), ("heads", 32), ("kv-heads", 8), ("head-dim", 128), ("context", 4096), ("batch", 16),
                        ("steps", 20)):
        ap.add_argument(f"--{name}", type=int, default=value)
    args = ap.parse_args()
    layer = AttentionLayer(args.hidden, args.heads, args.kv_heads, args.head_dim, args.batch, args.context + args.steps + 8)
    x = torch.randn(args.batch * args.context, args.hidden, device="cuda", dtype=torch.bfloat16)
    offsets = torch.arange(args.batch + 1, device="cuda", dtype=torch.int32) * args.context
    out = layer(x, torch.arange(args.context, device="cuda").repeat(args.batch), offsets)
    assert out.shape == x.shape and torch.isfinite(out).all()
    stream, token = torch.cuda.Stream(), x[:args.batch].clone()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        layer(token, layer.lengths)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = layer(token, layer.lengths)
        for _ in range(3):
            graph.replay()
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record(stream)
        for _ in range(args.steps):
            graph.replay()
        end.record(stream)
    end.synchronize()
    assert torch.isfinite(out).all()
    print(f"{args.batch} sequences of {args.context} tokens: {start.elapsed_time(end) * 1e3 / args.steps:.1f} us a decode step, "
          f"output rms {out.float().square().mean().sqrt():.3f}")


if __name__ == "__main__":
    main()
