"""The 4-bit paged cache and its attention on the GPU: codes bit for bit, attention against 64 bits."""
import pytest
import torch

import my_own_cnn_b200 as b2q
from lowbit_ref import attention, cache_values, cache_words, quantize4, within

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def gen(seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def poisoned(pages, heads, page, d, group):
    """A cache whose every place holds NaN scales until it is written."""
    c = b2q.KV4Cache.empty(pages, heads, page, d, group)
    for x in (c.k_codes, c.v_codes):
        x.fill_(0xA7)
    for x in (c.k_params, c.v_params):
        x.fill_(0x7FC0)
    return c


def filled(lens, heads, page, d, group, seed=0, spare=2):
    """A cache with `lens` tokens per sequence in scattered pages, and its block table."""
    g = gen(seed)
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + spare
    c = poisoned(pages, heads, page, d, group)
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((len(lens), max(counts + [1])), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n]
        at += n
    slots = torch.cat([table[i, :counts[i]].long().repeat_interleave(page)[:n] * page
                       + torch.arange(n, device="cuda") % page for i, n in enumerate(lens)]) if sum(lens) else None
    if slots is not None:
        size = torch.rand(heads, 1, generator=g, device="cuda") + 0.5
        k, v = (torch.randn(len(slots), heads, d, generator=g, device="cuda") * size for _ in range(2))
        b2q.kv4_append(c, k, v, slots)
    return c, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,group", [(64, 32), (64, 64), (128, 32), (128, 64), (256, 32), (256, 64)])
@pytest.mark.parametrize("t,heads,page", [(1, 1, 1), (3, 2, 5), (67, 3, 16), (300, 1, 64)])
def test_append_and_read_bit_for_bit(dtype, d, group, t, heads, page):
    g = gen(t)
    pages = -(-t // page) + 2
    c = poisoned(pages, heads, page, d, group)
    before = [x.clone() for x in (c.k_codes, c.k_params, c.v_codes, c.v_params)]
    fused = (torch.randn(t, 2 * heads, d, generator=g, device="cuda") * 3).to(dtype)
    k, v = fused[:, :heads], fused[:, heads:]
    # groups that are zero, of one sign, constant, tiny, huge
    special = [0.0, 1e-42 if dtype == torch.float32 else 0.0, 5.0, -2.5]
    for i, s in enumerate(special):
        if i < t:
            k[i, 0, :group] = s
    v[0, 0, :group] = v[0, 0, :group].abs() + 1
    if t > 4:
        v[4, 0] *= 1e3
        v[3, 0, :group] *= 1e-3
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:t]
    if t > 2:
        slots[2] = -1
    b2q.kv4_append(c, k, v, slots)
    rk, rv = b2q.kv4_read(c, slots, dtype)
    assert b2q.last_path() == "kv4-cache"
    kept = (slots >= 0).cpu()
    pg, at = slots.cpu()[kept] // page, slots.cpu()[kept] % page
    for x, r, codes, params, old_codes, old_params in ((k, rk, c.k_codes, c.k_params, before[0], before[1]),
                                                       (v, rv, c.v_codes, c.v_params, before[2], before[3])):
        cd, s, z = quantize4(x.cpu()[kept], group)
        want_codes, want_params = old_codes.cpu(), old_params.cpu()
        want_codes[pg, :, at] = cd[..., 0::2] | (cd[..., 1::2] << 4)
        want_params[pg, :, at] = cache_words(s, z)
        assert torch.equal(codes.cpu(), want_codes) and torch.equal(params.cpu(), want_params)
        values, _ = cache_values(want_codes[pg, :, at], want_params[pg, :, at], group)
        assert torch.equal(r.cpu()[kept], values.float().to(dtype)) and (r.cpu()[~kept] == 0).all()
        # each value is within half a step (a step more at the range's end, where the scale was rounded down)
        step = s.repeat_interleave(group, -1)
        assert ((values - x.cpu()[kept].double()).abs() <= 0.5625 * step + 1e-37).all()


def test_append_views_and_channels_apart():
    c, other = poisoned(3, 2, 16, 64, 32), poisoned(3, 2, 16, 64, 32)
    x = torch.randn(64, 2, 9, device="cuda").permute(2, 1, 0)
    store = torch.randn(9, 2, 67, device="cuda")
    slots = torch.arange(9, device="cuda")
    b2q.kv4_append(c, x, store[..., 3:], slots)
    b2q.kv4_append(other, x.contiguous(), store[..., 3:].contiguous(), slots)
    assert torch.equal(c.k_codes, other.k_codes) and torch.equal(c.v_codes, other.v_codes)
    assert torch.equal(c.k_params, other.k_params) and torch.equal(c.v_params, other.v_params)


def run(c, table, lens, tq, hq, dtype, seed=9, scale=None):
    b, d = len(lens), c.head_dim
    q = torch.randn(b, tq, hq, d, generator=gen(seed), device="cuda").to(dtype)
    out, lse = b2q.kv4_attention(q, c, table, lens, scale=scale, return_lse=True)
    assert b2q.last_path() == "kv4-attention"
    want, wl, ob, lb = attention(q, c, table, lens, d ** -0.5 if scale is None else scale, dtype)
    within(out, want, ob + (2.0 ** -25 if dtype == torch.float16 else 0))
    within(lse, wl, lb)
    return q, out, lse


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,group", [(64, 32), (64, 64), (128, 32), (128, 64), (256, 32), (256, 64)])
@pytest.mark.parametrize("hk,ratio,tq", [(1, 1, 1), (2, 4, 1), (3, 5, 2), (1, 8, 3), (2, 3, 7)])
def test_attention(dtype, d, group, hk, ratio, tq):
    c, table, lens = filled([37, 1, 0, 200, 16, 3], hk, 16, d, group)
    run(c, table, lens, tq, hk * ratio, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [1, 3, 16, 48, 100, 128])
def test_attention_page_sizes_and_long_sequences(dtype, page):
    c, table, lens = filled([1500, 0, 129, 64, 65, 63, 2047], 2, page, 64, 32, seed=page)
    run(c, table, lens, 1, 8, dtype)
    run(c, table, lens, 2, 2, dtype)


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 511, 512, 513, 4095, 4097])
def test_attention_lengths(length):
    c, table, lens = filled([length], 1, 32, 128, 64, seed=length)
    run(c, table, lens, 1, 4, torch.bfloat16)


@pytest.mark.parametrize("page", [16, 32])
@pytest.mark.parametrize("d,hk,ratio,tq", [(64, 2, 3, 1), (128, 1, 9, 1), (256, 1, 5, 3)])
def test_attention_many_sequences(d, hk, ratio, tq, page):
    """More sequences than a warp counts at a time, most of them short, some empty, a few split over several blocks."""
    lens = [(0, 7, 1, 130, 33, 64, 300)[i % 7] for i in range(75)]
    lens[40], lens[71] = 3000, 1500
    c, table, n = filled(lens, hk, page, d, 32, seed=d)
    run(c, table, n, tq, hk * ratio, torch.float16)


@pytest.mark.parametrize("d,ratio", [(64, 4), (128, 4), (128, 16), (256, 8)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_long_context(dtype, d, ratio):
    c, table, n = filled([20000], 1, 64, d, 64, seed=d + ratio)
    run(c, table, n, 1, ratio, dtype)


def test_attention_wide_table():
    """A table with room for many more pages than the lengths name."""
    c, table, lens = filled([500, 40], 2, 32, 64, 64)
    wide = torch.full((2, 5000), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    q = torch.randn(2, 1, 4, 64, generator=gen(6), device="cuda")
    want, _, ob, _ = attention(q, c, table, lens, 0.125, torch.float32)
    within(b2q.kv4_attention(q, c, wide, lens), want, ob)


def test_attention_many_rows_of_a_head():
    c, table, lens = filled([90, 5], 1, 16, 64, 64)
    run(c, table, lens, 9, 11, torch.float16)
    run(c, table, lens, 40, 3, torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_peaked_and_flat_scores(dtype):
    """Scores of hundreds: nearly all the weight on one token, a maximum that comes late; and all alike."""
    c, table, lens = filled([700, 300], 2, 64, 128, 64, seed=3)
    run(c, table, lens, 1, 4, dtype, scale=8.0)
    run(c, table, lens, 1, 4, dtype, scale=0.0)
    run(c, table, lens, 1, 4, dtype, scale=-0.3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kscale,vscale", [(1e-6, 1e3), (1e4, 1e-6), (1.0, 1e-12)])
def test_attention_scales_of_any_size(dtype, kscale, vscale):
    if dtype == torch.float16 and vscale < 1:
        pytest.skip("the values lie below fp16's range")
    pages, page, d = 8, 16, 64
    c = poisoned(pages, 1, page, d, 32)
    n = 100
    k, v = torch.randn(n, 1, d, generator=gen(1), device="cuda"), torch.randn(n, 1, d, generator=gen(2), device="cuda")
    b2q.kv4_append(c, k * kscale, v * vscale, torch.arange(n, device="cuda"))
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    run(c, table, torch.tensor([n], dtype=torch.int32, device="cuda"), 1, 2, dtype, scale=0.1 / kscale)


def test_attention_views_of_queries_and_tables():
    c, table, lens = filled([70, 33, 16], 2, 16, 128, 64)
    big = torch.randn(3, 2, 4 + 5, 128 + 1, generator=gen(4), device="cuda").bfloat16()
    q = big[:, :, 2:6, 1:]
    wide = torch.full((3, table.shape[1] + 6), -7, dtype=torch.int32, device="cuda")
    wide[:, 1:1 + table.shape[1]] = table
    want = b2q.kv4_attention(q.contiguous(), c, table, lens)
    assert torch.equal(b2q.kv4_attention(q, c, wide[:, 1:1 + table.shape[1]], lens), want)
    apart = q.contiguous().permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)
    assert torch.equal(b2q.kv4_attention(apart, c, table, lens), want)
    out = torch.empty_like(want)
    assert b2q.kv4_attention(q, c, table, lens, out=out) is out and torch.equal(out, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,group", [(64, 32), (128, 64), (256, 64)])
def test_log_sums_are_fp32(dtype, d, group):
    """One token: the log-sum is its score, d / 16 additions that may truncate at 2^-23, and the scaling after them."""
    c, table, lens = filled([1] * 60, 2, 16, d, group)
    q = torch.randn(60, 1, 6, d, generator=gen(14), device="cuda").to(dtype)
    _, lse = b2q.kv4_attention(q, c, table, lens, return_lse=True)
    k, _ = b2q.kv4_read(c, table[:, 0].long() * 16)
    want = (q.double().view(60, 2, 3, d) * k.double()[:, :, None]).sum(-1).view(60, 1, 6) * d ** -0.5
    assert (lse.double() - want).norm() <= 2.0 ** -23 * (d / 16 + 2) * want.norm()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_attention_hides_what_a_row_does_not_see(dtype, what, bad):
    """A token with an infinite or NaN channel is met by its own row and later ones, not by the rows before it."""
    c, table, lens = filled([50], 2, 16, 64, 32)
    q = torch.randn(1, 3, 4, 64, generator=gen(13), device="cuda").to(dtype)
    want = b2q.kv4_attention(q, c, table, lens)
    slot = (table[0, 48 // 16].long() * 16 + 48 % 16).view(1)  # the last row but one's own token
    k, v = b2q.kv4_read(c, slot)
    (k if what == "k" else v)[..., 5] = bad
    b2q.kv4_append(c, k, v, slot)
    out = b2q.kv4_attention(q, c, table, lens)
    assert torch.equal(out[:, 0], want[:, 0])
    if what == "v" and bad == bad:  # not hidden from those that see it (an infinite key may give a score of -inf, weight 0)
        assert not out[:, 1:].isfinite().all(-1).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("length", [40, 9000])
def test_attention_output_at_any_element(dtype, length):
    c, table, lens = filled([length], 2, 16, 64, 32)
    q = torch.randn(1, 1, 6, 64, generator=gen(6), device="cuda").to(dtype)
    want = b2q.kv4_attention(q, c, table, lens)
    for at in range(1, 9):
        store = torch.full((q.numel() + 16,), 7.0, dtype=dtype, device="cuda")
        out = store[at:at + q.numel()].view(q.shape)
        b2q.kv4_attention(q, c, table, lens, out=out)
        assert torch.equal(out, want) and (store[:at] == 7).all() and (store[at + q.numel():] == 7).all()


def test_a_graph_outlives_larger_calls_on_its_stream():
    c, table, lens = filled([3000], 1, 16, 64, 64)
    q = torch.randn(1, 1, 4, 64, generator=gen(7), device="cuda").bfloat16()
    big, big_table, big_lens = filled([2000] * 40, 4, 16, 256, 64)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    want = b2q.kv4_attention(q, c, table, lens, stream=s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        y = b2q.kv4_attention(q, c, table, lens)
    b2q.kv4_attention(torch.zeros(40, 1, 32, 256, device="cuda"), big, big_table, big_lens, stream=s)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(3):
            g.replay()
            b2q.kv4_attention(torch.zeros(40, 1, 32, 256, device="cuda"), big, big_table, big_lens)
    torch.cuda.synchronize()
    assert torch.equal(y, want)


def test_a_stream_without_scratch_is_not_captured():
    c, table, lens = filled([100], 1, 16, 64, 64)
    q = torch.randn(1, 1, 4, 64, generator=gen(8), device="cuda")
    s = torch.cuda.Stream(priority=-1)
    s.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=s):
            b2q.kv4_attention(q, c, table, lens)
    y = b2q.kv4_attention(q, c, table, lens, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(y, b2q.kv4_attention(q, c, table, lens))


def test_attention_repeats_and_streams_and_graph():
    c, table, lens = filled([3000, 100, 0], 2, 64, 128, 64)
    q = torch.randn(3, 1, 8, 128, generator=gen(5), device="cuda").half()
    want = b2q.kv4_attention(q, c, table, lens)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = [b2q.kv4_attention(q, c, table, lens, stream=s) for _ in range(4)]
    here = [b2q.kv4_attention(q, c, table, lens) for _ in range(4)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, want) for x in got + here)
    with torch.cuda.stream(s):
        b2q.kv4_attention(q, c, table, lens)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        y = b2q.kv4_attention(q, c, table, lens)
    lens[1] = 64  # a shorter sequence in the replay
    g.replay()
    assert torch.equal(y, b2q.kv4_attention(q, c, table, lens))


def test_offsets_past_32_bits():
    """A cache of over 2^32 code bytes: the last pages are written, read back and attended to."""
    heads, page, d = 8, 128, 256
    pages = (1 << 32) // (heads * page * d // 2) + 9
    c = b2q.KV4Cache.empty(pages, heads, page, d, 64)
    assert c.k_codes.numel() > 1 << 32
    n = 300
    order = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device="cuda")
    slots = order[0].long().repeat_interleave(page)[:n] * page + torch.arange(n, device="cuda") % page
    k, v = (torch.randn(n, heads, d, generator=gen(i), device="cuda").bfloat16() for i in (1, 2))
    b2q.kv4_append(c, k, v, slots)
    small = b2q.KV4Cache.empty(3, heads, page, d, 64)
    b2q.kv4_append(small, k, v, torch.arange(n, device="cuda"))
    for a, b in zip(b2q.kv4_read(c, slots), b2q.kv4_read(small, torch.arange(n, device="cuda"))):
        assert torch.equal(a, b)
    q = torch.randn(1, 1, 16, d, generator=gen(3), device="cuda").bfloat16()
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    line = torch.arange(3, dtype=torch.int32, device="cuda")[None]
    assert torch.equal(b2q.kv4_attention(q, c, order, lens), b2q.kv4_attention(q, small, line, lens))


@pytest.mark.parametrize("page", [16, 32])
def test_values_out_of_range_are_reported_and_left_out(page):
    c, table, lens = filled([40, 20], 1, page, 64, 64)
    b2q.device_error()
    k = torch.randn(2, 1, 64, device="cuda")
    before = c.k_codes.clone()
    b2q.kv4_append(c, k, k, torch.tensor([-1, c.pages * page], device="cuda"))
    with pytest.raises(b2q.B200QError, match="slot"):
        b2q.device_error()
    assert torch.equal(c.k_codes, before)
    rk, _ = b2q.kv4_read(c, torch.tensor([c.pages * page + 5, 0], device="cuda"))
    with pytest.raises(b2q.B200QError, match="slot"):
        b2q.device_error()
    assert (rk[0] == 0).all()
    q = torch.randn(2, 1, 2, 64, device="cuda")
    want = b2q.kv4_attention(q, c, table, lens)
    b2q.device_error()
    for bad, message in ((c.pages, "page"), (-1, "page")):
        t = table.clone()
        t[0, 1] = bad
        out = b2q.kv4_attention(q, c, t, lens)
        with pytest.raises(b2q.B200QError, match=message):
            b2q.device_error()
        assert out.isfinite().all() and torch.equal(out[1], want[1])
    for bad in (table.shape[1] * page + 1, -3):
        n = lens.clone()
        n[0] = bad
        out = b2q.kv4_attention(q, c, table, n)
        with pytest.raises(b2q.B200QError, match="length"):
            b2q.device_error()
        assert (out[0] == 0).all() and torch.equal(out[1], want[1])
    b2q.device_error()


def test_nothing_to_do():
    c, table, lens = filled([5], 1, 16, 64, 64)
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    b2q.kv4_append(c, torch.zeros(0, 1, 64, device="cuda"), torch.zeros(0, 1, 64, device="cuda"), none)
    assert b2q.kv4_read(c, none)[0].shape == (0, 1, 64)
    assert b2q.kv4_attention(torch.zeros(0, 1, 2, 64, device="cuda"), c, table[:0], lens[:0]).shape == (0, 1, 2, 64)
    empty = torch.zeros(1, 0, dtype=torch.int32, device="cuda")
    out, lse = b2q.kv4_attention(torch.ones(1, 2, 2, 64, device="cuda"), c, empty, torch.zeros_like(lens), return_lse=True)
    assert (out == 0).all() and (lse == -float("inf")).all()


def test_refusals():
    c, table, lens = filled([5], 2, 16, 64, 64)
    k = torch.zeros(3, 2, 64, device="cuda")
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="k and v must be"):
        b2q.kv4_append(c, k[..., :32], k[..., :32], slots)
    with pytest.raises(TypeError, match="v must be"):
        b2q.kv4_append(c, k, k.half(), slots)
    with pytest.raises(TypeError, match="slots"):
        b2q.kv4_append(c, k, k, slots.int())
    with pytest.raises(RuntimeError, match="slots"):
        b2q.kv4_append(c, k, k, slots[:2])
    with pytest.raises(TypeError, match="dtype"):
        b2q.kv4_read(c, slots, torch.float64)
    q = torch.zeros(1, 1, 4, 64, device="cuda")
    with pytest.raises(RuntimeError, match="do not divide"):
        b2q.kv4_attention(q[:, :, :3], c, table, lens)
    with pytest.raises(RuntimeError, match="q must be"):
        b2q.kv4_attention(q[..., :32], c, table, lens)
    with pytest.raises(TypeError, match="lens"):
        b2q.kv4_attention(q, c, table, lens.long())
    with pytest.raises(RuntimeError, match="block_table"):
        b2q.kv4_attention(q, c, table[:, None], lens)
    with pytest.raises(RuntimeError, match="out must be"):
        b2q.kv4_attention(q, c, table, lens, out=q.half())
    with pytest.raises(RuntimeError, match="cache codes"):
        b2q.KV4Cache(c.k_codes[0], c.k_params, c.v_codes, c.v_params)
    with pytest.raises(RuntimeError, match="same cache shapes"):
        b2q.KV4Cache(c.k_codes, c.k_params, c.v_codes[:1], c.v_params)
    with pytest.raises(RuntimeError, match="4-bit caches"):
        b2q.KV4Cache.empty(1, 1, 16, 96)
