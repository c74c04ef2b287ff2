"""The 4-bit attention block: its operators together, token by token."""
import pytest
import torch

import my_own_cnn_b200 as b2q
from my_own_cnn_b200.decoder import random_block
from lowbit_ref import norm_rope, w4_values

pytestmark = pytest.mark.gpu


def setup(dtype, batch=3, page=16, pages=6):
    block = random_block(320, 6, 2, 64, dtype, positions=128, group=32)
    cache = b2q.KV4Cache.empty(batch * pages, 2, page, 64, 32)
    table = torch.randperm(batch * pages, device="cuda").int().view(batch, pages)
    return block, cache, table


def place(table, page, at):
    return table.long().gather(1, at // page) * page + at % page


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tq", [1, 3])
def test_block_answers_tokens(dtype, tq):
    """Several steps against 64 bits over the values that the cache holds.  In fp32 every operator is within about 1e-6
    of its size; in bf16 four roundings of 2^-9 (projection, norm, attention, output) meet, 2^-7 in all."""
    block, cache, table = setup(dtype)
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    wqkv, wo = w4_values(block.wqkv), w4_values(block.wo)
    for step in range(12):
        x = torch.randn(3, tq, 320, generator=g, device="cuda").to(dtype)
        at = lens.long()[:, None] + torch.arange(tq, device="cuda")
        lens += tq
        slots = place(table, 16, at).flatten()
        y = block.forward(x, cache, at.int().flatten(), slots, table, lens)
        qkv = (x.double().view(3 * tq, 320) @ wqkv.t()).view(3 * tq, 10, 64)
        q = norm_rope(qkv[:, :6], block.q_norm.double(), block.table, at.flatten(), 1e-6, False).view(3, tq, 2, 3, 64)
        n = int(lens[0])
        seen = torch.arange(n, device="cuda").expand(3, n)
        k, v = b2q.kv4_read(cache, place(table, 16, seen).flatten())
        k, v = k.double().view(3, n, 2, 64), v.double().view(3, n, 2, 64)
        a = torch.einsum("bihrd,bthd->bihrt", q, k) / 8
        hidden = torch.arange(n, device="cuda") > (n - tq + torch.arange(tq, device="cuda"))[:, None]
        a = a.masked_fill(hidden[None, :, None, None], -float("inf")).softmax(-1)
        o = torch.einsum("bihrt,bthd->bihrd", a, v).reshape(3 * tq, 384)
        want = (o @ wo.t()).view(3, tq, 320)
        off = (y.double() - want).norm() / want.norm()
        assert off < (1e-5 if dtype == torch.float32 else 2.0 ** -7), (step, float(off))


def test_block_in_a_graph_and_on_a_stream():
    block, cache, table = setup(torch.bfloat16)
    other = b2q.KV4Cache.empty(18, 2, 16, 64, 32)
    s = torch.cuda.Stream()
    x = torch.randn(3, 1, 320, device="cuda").bfloat16()
    at = torch.zeros(3, 1, dtype=torch.int64, device="cuda")
    positions, slots = at.int().flatten(), place(table, 16, at).flatten()
    lens = torch.ones(3, dtype=torch.int32, device="cuda")
    s.wait_stream(torch.cuda.current_stream())
    first = block.forward(x, other, positions, slots, table, lens, stream=s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        y = block.forward(x, cache, positions, slots, table, lens)
    g.replay()
    assert torch.equal(y, first)
    for step in range(1, 20):
        x.copy_(torch.randn(3, 1, 320, device="cuda"))
        at += 1
        positions.copy_(at.flatten())
        slots.copy_(place(table, 16, at).flatten())
        lens += 1
        g.replay()
        assert torch.equal(y, block.forward(x, other, positions, slots, table, lens)), step


def test_block_refuses_projections_that_do_not_fit():
    block, _, _ = setup(torch.float32)
    with pytest.raises(RuntimeError, match="do not fit"):
        b2q.W4Attention(block.wqkv, block.wo, None, None, None, 5, 2, 64)


def test_block_takes_tokens_in_any_layout():
    block, cache, table = setup(torch.bfloat16)
    x = torch.randn(320, 2, 3, device="cuda").bfloat16().permute(2, 1, 0)
    at = torch.arange(2, device="cuda").expand(3, 2)
    args = cache, at.int().flatten(), place(table, 16, at).flatten(), table, torch.full((3,), 2, dtype=torch.int32, device="cuda")
    assert torch.equal(block.forward(x, *args), block.forward(x.contiguous(), *args))
