"""The 8-bit attention block: packed prompts into the 4-bit cache, then tokens from there."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import my_own_cnn_b200 as b2q
from my_own_cnn_b200.decoder import random_block_s8
from tests import s8_ref
from tests.lowbit_ref import norm_rope

pytestmark = pytest.mark.gpu
HIDDEN, H, HK, D, PAGE = 320, 6, 2, 64, 16


def values(rows):
    return rows.codes[:, :rows.k].double() * rows.scales.double()[:, None]


def plain(block, x, residual, positions, attend):
    """The block in 64 bits: its first rounding to 8 bits as the format says, the second one of the plain attention's rows."""
    codes, scales, h = s8_ref.rows(x, block.norm, residual, block.eps)
    qkv = ((codes * scales[:, None]) @ values(block.wqkv).t()).view(-1, H + 2 * HK, D)
    q = norm_rope(qkv[:, :H], block.q_norm.double(), block.table, positions, block.eps, False)
    k = norm_rope(qkv[:, H:H + HK], block.k_norm.double(), block.table, positions, block.eps, False)
    o = attend(q, k, qkv[:, H + HK:]).reshape(-1, H * D)
    top = o.abs().amax(-1, keepdim=True)
    return ((o * 127 / top).round() * top / 127) @ values(block.wo).t(), h


def softmax(q, k, v, seen):
    a = torch.einsum("ihrd,jhd->hrij", q.view(q.shape[0], HK, H // HK, D), k) * D ** -0.5
    a = a.masked_fill(~seen, -float("inf")).softmax(-1)
    return torch.einsum("hrij,jhd->ihrd", a, v).reshape(q.shape[0], H * D)


# A value that moves by a share d of a step changes its code in a share d of the cases, by a whole step: the mean square is d steps, not
# d^2.  A step is about 4 / 127 of a row's root mean square.  fp32: d of 1e-5 steps and less, (1e-5)^1/2 4 / 127 = 1e-4.  bf16: roundings
# of projection, norm, weights and result, 4 x 2^-9 / 3^1/2 in all 0.5 % or 0.15 of a step, 0.15^1/2 4 / 127 = 1.2 %.
BOUND = {torch.float32: 1e-3, torch.bfloat16: 2.0 ** -6}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompts_then_tokens(dtype):
    block = random_block_s8(HIDDEN, H, HK, D, dtype, positions=256)
    lengths = [37, 0, 90, 1]
    per = 8
    cache = b2q.KV4Cache.empty(len(lengths) * per, HK, PAGE, D, 32)
    table = torch.randperm(len(lengths) * per, device="cuda").int().view(len(lengths), per)
    starts = torch.tensor([0] + lengths, device="cuda").cumsum(0).int()
    sequence = torch.repeat_interleave(torch.arange(len(lengths), device="cuda"), torch.tensor(lengths, device="cuda"))
    positions = (torch.arange(sum(lengths), device="cuda") - starts[sequence]).int()

    def slots_of(seq, pos):
        return table[seq, pos.long() // PAGE].long() * PAGE + pos.long() % PAGE

    g = torch.Generator(device="cuda").manual_seed(3)
    x, residual = (torch.randn(sum(lengths), HIDDEN, generator=g, device="cuda").to(dtype) for _ in range(2))
    kept = residual.clone()
    y, total = block.prompt(x, kept, positions, starts, cache, slots_of(sequence, positions))
    b2q.device_error()
    seen = (sequence[:, None] == sequence) & (positions[None] <= positions[:, None])
    want, h = plain(block, x, residual, positions, lambda q, k, v: softmax(q, k, v, seen))
    assert total is kept and torch.equal(total, h)
    assert (y.double() - want).norm() / want.norm() < BOUND[dtype]
    # without a residual, and without a cache
    y2, x2 = block.prompt(x, None, positions, starts)
    want, _ = plain(block, x, None, positions, lambda q, k, v: softmax(q, k, v, seen))
    assert x2 is x and (y2.double() - want).norm() / want.norm() < BOUND[dtype]

    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    seq = torch.arange(len(lengths), device="cuda")
    for _ in range(3):
        at = lens.clone()
        lens += 1
        x, residual = (torch.randn(len(lengths), HIDDEN, generator=g, device="cuda").to(dtype) for _ in range(2))
        kept = residual.clone()
        y, total = block.forward(x, kept, cache, at, slots_of(seq, at), table, lens)
        b2q.device_error()

        def attend(q, k, v):
            rows = []
            for i in range(len(lengths)):
                n = int(lens[i])
                kv = b2q.kv4_read(cache, slots_of(torch.full((n,), i, device="cuda"), torch.arange(n, device="cuda")))
                rows.append(softmax(q[i:i + 1], kv[0].double(), kv[1].double(), torch.ones(1, n, dtype=torch.bool, device="cuda")))
            return torch.cat(rows)

        want, h = plain(block, x, residual, at, attend)
        assert torch.equal(total, h)
        assert (y.double() - want).norm() / want.norm() < BOUND[dtype]


def test_block_in_a_graph_and_on_a_stream():
    block = random_block_s8(HIDDEN, H, HK, D, torch.bfloat16, positions=256)
    x = torch.randn(100, HIDDEN, device="cuda").bfloat16()
    positions, starts = torch.arange(100, device="cuda").int(), torch.tensor([0, 60, 100], device="cuda").int()
    eager, _ = block.prompt(x, None, positions, starts)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    other, _ = block.prompt(x, None, positions, starts, stream=s)
    s.synchronize()
    assert torch.equal(eager, other)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out, _ = block.prompt(x, None, positions, starts)
    starts.copy_(torch.tensor([0, 100, 100]))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, block.prompt(x, None, positions, starts)[0])


def test_projections_that_do_not_fit():
    b = random_block_s8(HIDDEN, H, HK, D, torch.float32, positions=8)
    with pytest.raises(RuntimeError, match="do not fit"):
        b2q.S8Attention(b.norm, b.wqkv, b.wo, None, None, None, H + 1, HK, D)
    with pytest.raises(RuntimeError, match="do not fit"):
        b2q.S8Attention(b.norm[:300], b.wqkv, b.wo, None, None, None, H, HK, D)


def test_example_runs():
    root = Path(__file__).resolve().parents[1]
    r = subprocess.run([sys.executable, str(root / "examples" / "prompt_s8.py"), "--batch", "3", "--prompt", "96", "--steps", "4"],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert "tokens/s" in r.stdout
