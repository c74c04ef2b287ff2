"""Answers tokens with a random 4-bit attention block, captured in a CUDA graph, and prints the time of a step:

    python examples/decode_w4.py --batch 8 --context 4096
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from my_own_cnn_b200 import KV4Cache, kv4_append  # noqa: E402
from my_own_cnn_b200.decoder import random_block  # noqa: E402


def main() -> None:
    ap = argparse.ArgumentParser(description="Answer tokens with a random 4-bit attention block.")
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--context", type=int, default=4096, help="tokens in the cache when timing starts")
    ap.add_argument("--steps", type=int, default=64)
    a = ap.parse_args()
    dtype, hidden, heads, kv_heads, d, page = torch.bfloat16, 4096, 32, 8, 128, 64
    block = random_block(hidden, heads, kv_heads, d, dtype, a.context + a.steps + 1)
    per = -(-(a.context + a.steps) // page)
    cache = KV4Cache.empty(a.batch * per, kv_heads, page, d)
    table = torch.arange(a.batch * per, dtype=torch.int32, device="cuda").view(a.batch, per)
    first = torch.arange(a.context, device="cuda")
    for i in range(a.batch):  # a context of random keys and values
        kv = torch.randn(a.context, 2 * kv_heads, d, device="cuda").to(dtype)
        kv4_append(cache, kv[:, :kv_heads], kv[:, kv_heads:], i * per * page + first)
    lens = torch.full((a.batch,), a.context, dtype=torch.int32, device="cuda")
    x = torch.randn(a.batch, 1, hidden, device="cuda").to(dtype)

    def step():
        slots = torch.arange(a.batch, device="cuda") * (per * page) + lens
        positions = lens.clone()
        lens.add_(1)
        x.copy_(block.forward(x, cache, positions, slots, table, lens))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # workspaces are made before the capture
        step()
    torch.cuda.current_stream().wait_stream(side)
    lens.fill_(a.context)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(a.steps):
        graph.replay()
    end.record()
    end.synchronize()
    us = 1000 * start.elapsed_time(end) / a.steps
    print(f"batch {a.batch}, context {a.context}: {us:.1f} us a step, {a.batch / us * 1e6:.0f} tokens/s through one block")


if __name__ == "__main__":
    main()
