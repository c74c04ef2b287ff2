"""The softmax weights of the 4-bit cache's attention: every token's counts to the type's own precision, however small it or its
values are beside others', and every token's values reach the output.

Bounds, of a row's relative size (root of the sum of squares over its channels).
  * fp32: a score is off by four roundings of 2^-24 of it (its product, two factors, the reference), and its weight by as much;
    ex2 is within 2^-22, three bf16 terms hold 24 bits, the sums and the output round to 2^-24: 2^-24 (8 + 4 max |score|) where
    a score is one product.  Where it is a sum over d channels (of size about one), d / 16 + 2 truncations of 2^-23 of the
    adder come instead: 2^-23 (d / 16 + 2) + 2^-21.
  * 16-bit: two bf16 terms leave 2^-18 of a weight; up to 128 additions to one sum truncate at 2^-24 each: together below e = 2^-16.
    Beside the definition's value rounded once, an element differs by one unit in the last place (at most 2 u of it) where the
    definition lies within e of a tie, so the root mean square of what differs is at most sqrt(2 u e)."""
import pytest
import torch

import my_own_cnn_b200 as b2q
from lowbit_ref import UNIT

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def normal(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda")


def held(k, v, group, page=64):
    """A cache of one head with these keys and values [n, d] in order, its table and length, and the values that it holds."""
    n, d = k.shape
    pages = -(-n // page)
    c = b2q.KV4Cache.empty(pages, 1, page, d, group)
    slots = torch.arange(n, device="cuda")
    b2q.kv4_append(c, k[:, None].contiguous(), v[:, None].contiguous(), slots)
    kk, vv = b2q.kv4_read(c, slots)
    return c, torch.arange(pages, device="cuda").int()[None], torch.tensor([n], device="cuda").int(), kk[:, 0].double(), vv[:, 0].double()


def definition(q, k, v, scale):
    a = scale * (q.double() @ k.t())
    return torch.softmax(a, -1) @ v, float(a.abs().max())


def apart(got, want):
    """The largest relative distance of a row."""
    return float(((got.double() - want).norm(dim=-1) / want.norm(dim=-1)).max())


@pytest.mark.parametrize("d,group", [(64, 32), (128, 64), (256, 64)])
@pytest.mark.parametrize("rows", [1, 12])
@pytest.mark.parametrize("n", [512, 2048, 9000])
@pytest.mark.parametrize("nats", [4.0, 8.0, 10.0, 12.0, 16.0])
def test_a_token_that_outweighs_the_rest(nats, n, rows, d, group):
    """The first token takes most of the weight and holds small values, as a sequence's first token often does."""
    k, v = torch.zeros(n, d, device="cuda"), normal(2, n, d)
    k[0, 0] = nats
    v[0] *= 2.0 ** -12
    c, table, lens, kk, vv = held(k, v, group)
    q = torch.zeros(1, 1, rows, d, device="cuda")
    q[..., 0] = 8.0
    out = b2q.kv4_attention(q, c, table, lens, scale=0.125)
    want, top = definition(q[0, 0], kk, vv, 0.125)
    assert apart(out[0, 0], want) <= 2.0 ** -24 * (8 + 4 * top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d,group", [(64, 32), (128, 32), (128, 64), (256, 64)])
@pytest.mark.parametrize("e", [0, 7, 14, 20, 60])
def test_groups_of_channels_of_different_size(dtype, d, group, e):
    """Each group's values by themselves, one group 2^e times as large as the others."""
    n, rows = 4096, 3
    k, v = normal(1, n, d), normal(2, n, d)
    v[:, :group] *= 2.0 ** e
    c, table, lens, kk, vv = held(k, v, group)
    q = normal(3, 1, 1, rows, d).to(dtype)
    out = b2q.kv4_attention(q, c, table, lens, scale=d ** -0.5)[0, 0]
    want, _ = definition(q[0, 0], kk, vv, d ** -0.5)
    bound = 2.0 ** -23 * (d / 16 + 2) + 2.0 ** -21 if dtype == torch.float32 else UNIT[dtype] + 2.0 ** -16
    for g in range(0, d, group):
        assert apart(out[:, g:g + group], want[:, g:g + group]) <= bound, g


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,group", [(64, 32), (64, 64), (128, 64), (256, 32)])
@pytest.mark.parametrize("n,rows", [(37, 40), (512, 5), (2000, 3), (20000, 4)])
def test_outputs_are_the_definition_rounded_once(dtype, n, rows, d, group):
    k, v = normal(1, n, d), normal(2, n, d)
    c, table, lens, kk, vv = held(k, v, group)
    q = normal(3, 1, 1, rows, d).to(dtype)
    out = b2q.kv4_attention(q, c, table, lens, scale=d ** -0.5)[0, 0]
    want, _ = definition(q[0, 0], kk, vv, d ** -0.5)
    if dtype == torch.float32:
        assert apart(out, want) <= 2.0 ** -23 * (d / 16 + 2) + 2.0 ** -21
    else:
        once = want.to(dtype).double()
        assert float((out.double() - once).norm() / once.norm()) <= (2 * UNIT[dtype] * 2.0 ** -16) ** 0.5


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 48])
def test_every_tokens_values_reach_the_output(dtype, page):
    """Equal scores, and in every channel another sixteenth of the tokens holds the value 15, the rest 0: a tile, warp, block or
    part left out takes a fiftieth or more from some channel's mean, and one token takes a thousandth."""
    n, d = 1500, 64
    t = torch.arange(n, device="cuda")
    v = torch.stack([((t * (2 * i + 1)) % 16 == i % 16).float() * 15 for i in range(d)], 1)
    c, table, lens, kk, vv = held(torch.zeros(n, d, device="cuda"), v, 64, page)
    q = normal(4, 1, 1, 2, d).to(dtype)
    out = b2q.kv4_attention(q, c, table, lens)[0, 0]
    want = vv.mean(0).expand(2, d)
    bound = 2.0 ** -21 if dtype == torch.float32 else 2.0 ** -16 + UNIT[dtype]
    assert float(((out.double() - want).abs() / want.abs().clamp(min=1e-9)).max()) <= bound


@pytest.mark.parametrize("dtype", TYPES)
def test_scales_of_either_sign(dtype):
    """A cache that was written elsewhere may hold negative scales."""
    n, d = 300, 64
    c, table, lens, kk, vv = held(normal(1, n, d), normal(2, n, d), 32)
    c.v_params[:, :, ::3, 1] |= 0x8000
    vv[:, 32:] *= torch.where(torch.arange(n, device="cuda") % 64 % 3 == 0, -1.0, 1.0)[:, None]
    q = normal(3, 1, 1, 2, d).to(dtype)
    out = b2q.kv4_attention(q, c, table, lens)[0, 0]
    want, _ = definition(q[0, 0], kk, vv, d ** -0.5)
    assert apart(out, want) <= (2.0 ** -20 if dtype == torch.float32 else UNIT[dtype] + 2.0 ** -16)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,mean", [(64, 0.0), (64, 1.0), (128, 1.0)])
def test_long_sums_do_not_drift(dtype, d, mean):
    """Sequences that one block each adds up from end to end (more units than blocks; they share their pages): with every tile's
    sum rounded once to 2^-24, 4096 tiles in four warps are off by 2^-24 sqrt(1024) of the sum at most likely, below e."""
    n, b = 131072, 640
    k, v = normal(1, n, d), normal(2, n, d) + mean
    c, table, lens, kk, vv = held(k, v, 64)
    q = normal(3, b, 1, 1, d).to(dtype)
    out = b2q.kv4_attention(q, c, table.expand(b, -1).contiguous(), lens.expand(b).contiguous(), scale=d ** -0.5)[::16, 0, 0]
    want, _ = definition(q[::16, 0, 0], kk, vv, d ** -0.5)
    if dtype == torch.float32:
        assert apart(out, want) <= 2.0 ** -23 * (d / 16 + 2) + 2.0 ** -20
    else:
        once = want.to(dtype).double()
        assert float((out.double() - once).norm() / once.norm()) <= (2 * UNIT[dtype] * 2.0 ** -16) ** 0.5
