"""Takes packed prompts through a random 8-bit attention block into a 4-bit cache, then answers tokens from there in a CUDA graph;
prints the time of the prompts and of a step:

    python examples/prompt_s8.py --batch 8 --prompt 1024
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from my_own_cnn_b200 import KV4Cache  # noqa: E402
from my_own_cnn_b200.decoder import random_block_s8  # noqa: E402


def main() -> None:
    ap = argparse.ArgumentParser(description="Packed prompts and tokens through a random 8-bit attention block.")
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=1024, help="tokens of the longest prompt")
    ap.add_argument("--steps", type=int, default=64)
    a = ap.parse_args()
    dtype, hidden, heads, kv_heads, d, page = torch.bfloat16, 4096, 32, 8, 128, 64
    block = random_block_s8(hidden, heads, kv_heads, d, dtype, a.prompt + a.steps + 1)
    per = -(-(a.prompt + a.steps) // page)
    cache = KV4Cache.empty(a.batch * per, kv_heads, page, d)
    table = torch.arange(a.batch * per, dtype=torch.int32, device="cuda").view(a.batch, per)
    lengths = torch.tensor([a.prompt * (i + 1) // a.batch for i in range(a.batch)], device="cuda")
    starts = torch.cat([lengths.new_zeros(1), lengths.cumsum(0)]).int()
    sequence = torch.repeat_interleave(torch.arange(a.batch, device="cuda"), lengths)
    positions = (torch.arange(int(starts[-1]), device="cuda") - starts[sequence]).int()
    slots = sequence * (per * page) + positions
    x = torch.randn(int(starts[-1]), hidden, device="cuda").to(dtype)
    residual = torch.randn_like(x)

    def timed(work, times):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        for _ in range(times):
            work()
        end.record()
        end.synchronize()
        return 1000 * start.elapsed_time(end) / times

    block.prompt(x, residual.clone(), positions, starts, cache, slots)  # modules are loaded by the first call
    us = timed(lambda: block.prompt(x, residual.clone(), positions, starts, cache, slots), 10)
    print(f"{a.batch} prompts, {x.shape[0]} tokens: {us:.0f} us, {x.shape[0] / us:.1f} M tokens/s through one block")

    lens = lengths.int()
    token, carried = torch.randn(a.batch, hidden, device="cuda").to(dtype), torch.randn(a.batch, hidden, device="cuda").to(dtype)

    def step():
        at = torch.arange(a.batch, device="cuda") * (per * page) + lens
        here = lens.clone()
        lens.add_(1)
        out, _ = block.forward(token, carried, cache, here, at, table, lens)
        token.copy_(out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # workspaces are made before the capture
        step()
    torch.cuda.current_stream().wait_stream(side)
    lens.copy_(lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    us = timed(graph.replay, a.steps)
    print(f"{a.batch} sequences: {us:.1f} us a step, {a.batch / us * 1e6:.0f} tokens/s through one block")


if __name__ == "__main__":
    main()
