"""NaN and infinities in queries and caches: shown by the rows and channels that meet them, and by no others."""
import pytest
import torch

import my_own_cnn_b200 as b2q
from lowbit_ref import cache_values

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
NAN, INF = 0x7FC0, 0x7F80  # scale words with a zero point of 0


def normal(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda")


def held(n, heads, d, group, page=16):
    c = b2q.KV4Cache.empty(-(-n // page), heads, page, d, group)
    slots = torch.arange(n, device="cuda")
    b2q.kv4_append(c, normal(1, n, heads, d), normal(2, n, heads, d), slots)
    return c, torch.arange(c.pages, device="cuda").int()[None], torch.tensor([n], device="cuda").int()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,group", [(64, 32), (128, 64), (256, 64)])
@pytest.mark.parametrize("n", [1, 50, 5000])
def test_nan_queries(dtype, d, group, n):
    c, table, lens = held(n, 2, d, group)
    q = normal(3, 1, 1, 6, d).to(dtype)
    want, sums = b2q.kv4_attention(q, c, table, lens, return_lse=True)
    q[0, 0, 1, 3] = q[0, 0, 4] = float("nan")
    out, lse = b2q.kv4_attention(q, c, table, lens, return_lse=True)
    bad = torch.tensor([1, 4], device="cuda")
    good = torch.tensor([0, 2, 3, 5], device="cuda")
    assert out[0, 0, bad].isnan().all() and lse[0, 0, bad].isnan().all()
    assert torch.equal(out[0, 0, good], want[0, 0, good]) and torch.equal(lse[0, 0, good], sums[0, 0, good])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("n,at", [(33, 32), (60, 40), (97, 96), (5000, 2500), (4129, 4128)])
def test_a_nan_key(dtype, d, n, at):
    """Wherever its token lies: alone in its tile, beside others, in one part of many.  Rows that come before it are finite."""
    c, table, lens = held(n, 1, d, 32)
    tq = n - at + 1  # the first row sees the tokens before it
    q = normal(3, 1, min(tq, 3), 2, d).to(dtype)
    if tq > 3:
        lens.fill_(at + 2)
    want, sums = b2q.kv4_attention(q, c, table, lens, return_lse=True)
    c.k_params[at // 16, 0, at % 16, 1] = NAN
    out, lse = b2q.kv4_attention(q, c, table, lens, return_lse=True)
    first = int(lens) - q.shape[1]  # tokens that come before the rows' own
    for i in range(q.shape[1]):
        if first + i + 1 > at:
            assert out[0, i].isnan().all() and lse[0, i].isnan().all()
        else:
            assert torch.equal(out[0, i], want[0, i]) and torch.equal(lse[0, i], sums[0, i])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("word", [NAN, INF, INF | 0x8000, INF | 5 << 16])
@pytest.mark.parametrize("d,group", [(64, 32), (128, 64), (256, 64)])
@pytest.mark.parametrize("n,at", [(1, 0), (60, 40), (3000, 1500)])
def test_value_scales(dtype, d, group, n, at, word):
    """The sum of one term (code - zero) * scale that is infinite or NaN and of finite ones, channel by channel."""
    c, table, lens = held(n, 1, d, group)
    q = normal(3, 1, 1, 3, d).to(dtype)
    want, sums = b2q.kv4_attention(q, c, table, lens, return_lse=True)
    c.v_params[at // 16, 0, at % 16, 1] = word
    out, lse = b2q.kv4_attention(q, c, table, lens, return_lse=True)
    value, _ = cache_values(c.v_codes[at // 16, 0, at % 16], c.v_params[at // 16, 0, at % 16], group)
    other = torch.ones(d, dtype=torch.bool, device="cuda")
    other[group:2 * group] = False
    assert torch.equal(out[..., other], want[..., other]) and torch.equal(lse, sums)
    value = value[group:2 * group].to(dtype).expand(3, group)
    assert not value.isfinite().any()
    assert torch.equal(out[0, 0, :, group:2 * group].nan_to_num(1.0, 3.0, -3.0), value.nan_to_num(1.0, 3.0, -3.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("word", [NAN, INF])
def test_value_scales_that_a_row_does_not_see(dtype, word):
    c, table, lens = held(50, 1, 64, 32)
    q = normal(3, 1, 4, 2, 64).to(dtype)
    want = b2q.kv4_attention(q, c, table, lens)
    c.v_params[48 // 16, 0, 48 % 16, 0] = word
    out = b2q.kv4_attention(q, c, table, lens)
    assert torch.equal(out[:, :2], want[:, :2]) and torch.equal(out[..., 32:], want[..., 32:])
    assert not out[:, 2:, :, :32].isfinite().any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("d,group", [(64, 32), (64, 64), (128, 32), (128, 64), (256, 32), (256, 64)])
def test_append_keeps_what_is_not_finite(dtype, bad, d, group):
    """Its group of channels reads back as NaN, wherever in the group it lies; all other groups as without it."""
    t = d + 3  # a token for each channel, one with a whole group of them, and two without
    c = b2q.KV4Cache.empty(-(-t // 16), 2, 16, d, group)
    clean = b2q.KV4Cache.empty(c.pages, 2, 16, d, group)
    slots = torch.arange(t, device="cuda")
    k, v = normal(1, t, 2, d).to(dtype), normal(2, t, 2, d).to(dtype)
    b2q.kv4_append(clean, k, v, slots)
    want = b2q.kv4_read(clean, slots, dtype)
    i = torch.arange(d, device="cuda")
    hit = torch.zeros(t, 2, d, dtype=torch.bool, device="cuda")
    hit[i, 1, i] = True
    hit[d, 0, :group] = True
    for x in (k, v):
        x[hit] = bad
    b2q.kv4_append(c, k, v, slots)
    groups = hit.unflatten(-1, (-1, group)).any(-1, keepdim=True).expand(t, 2, d // group, group).flatten(-2)
    for got, x in zip(b2q.kv4_read(c, slots, dtype), want):
        assert got[groups].isnan().all() and torch.equal(got[~groups], x[~groups])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_attention_shows_what_was_appended(dtype, what, bad):
    c, table, lens = held(50, 2, 64, 32)
    q = normal(3, 1, 3, 4, 64).to(dtype)
    want, sums = b2q.kv4_attention(q, c, table, lens, return_lse=True)
    slot = torch.tensor([48], device="cuda")  # the last row but one's own token
    k, v = b2q.kv4_read(c, slot)
    (k if what == "k" else v)[..., 5] = bad
    b2q.kv4_append(c, k, v, slot)
    out, lse = b2q.kv4_attention(q, c, table, lens, return_lse=True)
    assert torch.equal(out[:, 0], want[:, 0]) and torch.equal(lse[:, 0], sums[:, 0])
    assert out[:, 1:, :, :32].isnan().all() and lse[:, 1:].isnan().all() == (what == "k")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,group", [(64, 32), (128, 64), (256, 32)])
def test_read_of_any_word(dtype, d, group):
    """(code - zero) * scale to the bit for every code and zero point, with scales that are finite, infinite and NaN."""
    c = b2q.KV4Cache.empty(4, 1, 64, d, group)
    scales = torch.tensor([0x3F80, 0x3DCD, 0xBE01, 0x0080, 0x7F00, INF, INF | 0x8000, NAN], device="cuda")
    for i, (codes, params) in enumerate(((c.k_codes, c.k_params), (c.v_codes, c.v_params))):
        codes.copy_(((torch.arange(codes.numel(), device="cuda") * (97 + 2 * i)) % 256).view_as(codes))
        at = torch.arange(params.numel(), device="cuda").view_as(params)
        params.copy_(scales[at % 8] | (at // 8 % 16) << 16)
    slots = torch.arange(256, device="cuda")
    for got, codes, params in zip(b2q.kv4_read(c, slots, dtype), (c.k_codes, c.v_codes), (c.k_params, c.v_params)):
        want = cache_values(codes.flatten(0, 2), params.flatten(0, 2), group)[0].to(torch.float32).to(dtype)
        assert torch.equal(got[:, 0].isnan(), want.isnan())
        assert torch.equal(got[:, 0][~want.isnan()], want[~want.isnan()])
