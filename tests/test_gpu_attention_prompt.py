"""prompt_attention against softmax in 64 bits, sequence by sequence and head by head."""
import math

import pytest
import torch

import my_own_cnn_b200 as b2q
from tests import s8_ref
from tests.lowbit_ref import UNIT, within

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def starts_of(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).cuda()


def make(tq, tk, hq, hk, d, dtype, seed=0, fused=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if fused:
        assert tq == tk
        x = torch.randn(tq, hq + 2 * hk, d, generator=g, device="cuda").to(dtype)
        return x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    return [torch.randn(n, h, d, generator=g, device="cuda").to(dtype) for n, h in ((tq, hq), (tk, hk), (tk, hk))]


def check(q, k, v, starts, k_starts=None, scale=None, out=None, lse=None):
    d = q.shape[2]
    if out is None:
        out, lse = b2q.prompt_attention(q, k, v, starts, k_starts, scale, return_lse=True)
        b2q.device_error()
    want, want_lse, ob, lb = s8_ref.attention(q, k, v, starts, starts if k_starts is None else k_starts,
                                              d ** -0.5 if scale is None else scale, q.dtype)
    rows = ~want_lse.isnan()
    within(out.cpu()[rows], want[rows], ob[rows])
    within(lse.cpu()[rows], want_lse[rows], lb[rows])
    return out, lse


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 80, 256, 40, 72, 1, 33])
def test_head_sizes(cuda_lib, dtype, d):
    q, k, v = make(300, 300, 4, 2, d, dtype, d)
    check(q, k, v, starts_of([131, 1, 0, 168]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hk", [(1, 1), (6, 2), (5, 1), (7, 7), (8, 1), (12, 3), (130, 1)])
def test_grouped_heads(cuda_lib, dtype, hq, hk):
    q, k, v = make(150, 150, hq, hk, 64, dtype, hq, fused=True)
    check(q, k, v, starts_of([77, 73]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 2, 15, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 192, 255, 256, 257, 300, 383, 384, 385, 640])
def test_lengths(cuda_lib, dtype, n):
    q, k, v = make(n, n, 4, 2, 128, dtype, n, fused=True)
    check(q, k, v, starts_of([n]))


@pytest.mark.parametrize("dtype", TYPES)
def test_keys_of_an_earlier_part_and_rows_that_see_none(cuda_lib, dtype):
    lq, lk = [3, 64, 1, 0, 130, 20, 50, 7, 200], [3, 200, 400, 9, 131, 5, 0, 6, 70]
    q, k, v = make(sum(lq), sum(lk), 8, 2, 64, dtype)
    out, lse = check(q, k, v, starts_of(lq), starts_of(lk))
    none = slice(sum(lq[:6]), sum(lq[:7]))  # no keys at all
    assert (out[none] == 0).all() and (lse[none] == -math.inf).all()
    first = sum(lq[:5])  # 20 queries, 5 keys: the first 15 see none
    assert (out[first:first + 15] == 0).all() and (lse[first:first + 15] == -math.inf).all() and lse[first + 15].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b", [33, 100, 257])
def test_many_sequences(cuda_lib, dtype, b):
    lens = [(i * 7919 + 3) % 23 if i % 5 else 0 for i in range(b)]
    lens[b // 2] = 270
    q, k, v = make(sum(lens), sum(lens), 4, 4, 64, dtype)
    check(q, k, v, starts_of(lens))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_outside_the_sequences_stay(cuda_lib, dtype):
    """Rows before the first sequence and behind the last one hold NaN in q, k and v, and their outputs are left as they were."""
    q, k, v = make(400, 400, 4, 2, 64, dtype)
    for x in (q, k, v):
        x[:11] = math.nan
        x[311:] = math.inf
    starts = torch.tensor([11, 90, 90, 311], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 3.0)
    got, lse = b2q.prompt_attention(q, k, v, starts, out=out, return_lse=True)
    assert got is out
    check(q, k, v, starts, out=out, lse=lse)
    assert (out[:11] == 3).all() and (out[311:] == 3).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_what_is_masked_has_no_part(cuda_lib, dtype):
    """NaN and infinities in keys and values reach the rows that see them, and no others."""
    n, hq, hk, d = 290, 4, 2, 64
    for place in (289, 200, 128, 5):
        q, k, v = make(n, n, hq, hk, d, dtype, place)
        clean, clean_lse = b2q.prompt_attention(q, k, v, starts_of([150, 140]) if place < 150 else starts_of([n]), return_lse=True)
        starts = starts_of([150, 140]) if place < 150 else starts_of([n])
        most = float(v.abs().max())
        v[place, 0, 7] = math.nan
        v[place, 1, 9] = math.inf
        out, lse = b2q.prompt_attention(q, k, v, starts, return_lse=True)
        end = 150 if place < 150 else n
        sees = torch.zeros(n, dtype=torch.bool, device="cuda")
        sees[place:end] = True
        assert out[sees, :2, 7].isnan().all() and (out[sees, 2:, 9] == math.inf).all()
        hit = torch.zeros_like(out, dtype=torch.bool)
        hit[sees, :2, 7] = True
        hit[sees, 2:, 9] = True
        # two roundings of the results, one of the weights, another order of sums
        unit = 3 * UNIT[dtype] + (n / 4 + 16) * 2.0 ** -22
        assert (out[~hit].double() - clean[~hit].double()).abs().max() < most * unit
        within(lse, clean_lse, torch.full_like(lse, 2.0 ** -16))
        # a key: its score is NaN
        q, k, v = make(n, n, hq, hk, d, dtype, place)
        k[place, 0, 3] = math.nan
        out, lse = b2q.prompt_attention(q, k, v, starts, return_lse=True)
        assert out[sees, :2].isnan().all() and lse[sees, :2].isnan().all()
        assert torch.equal(out[~sees], clean[~sees]) and torch.equal(out[:, 2:], clean[:, 2:])
        # a query
        q, k, v = make(n, n, hq, hk, d, dtype, place)
        q[place, 1] = math.nan
        out, lse = b2q.prompt_attention(q, k, v, starts, return_lse=True)
        assert out[place, 1].isnan().all() and lse[place, 1].isnan()
        out[place, 1], lse[place, 1] = clean[place, 1], clean_lse[place, 1]
        assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lq", [2500, 40])
def test_what_is_seen_and_not_finite(cuda_lib, dtype, lq):
    """NaN and infinities early in a long prompt (all of its rows, or the last 40 over the same keys): the results that see them, no
    others, with the log-sums and without."""
    n, hq, hk, d = 2500, 8, 2, 64
    q, k, v = make(n, n, hq, hk, d, dtype, 3)
    ends = starts_of([lq]), starts_of([n])
    call = lambda **kw: b2q.prompt_attention(q[n - lq:], k, v, *ends, **kw)
    clean, clean_lse = call(return_lse=True)
    most = float(v.abs().max())
    unit = 3 * UNIT[dtype] + (n / 4 + 16) * 2.0 ** -22  # as above
    v[3, 0, 5] = math.nan
    v[4, 1, 6], v[900, 1, 6], v[70, 1, 40] = math.inf, -math.inf, -math.inf
    out, lse = call(return_lse=True)
    at = torch.arange(n - lq, n, device="cuda")
    assert out[at >= 3, :4, 5].isnan().all() and out[at >= 900, 4:, 6].isnan().all()
    assert (out[(at >= 4) & (at < 900), 4:, 6] == math.inf).all() and (out[at >= 70, 4:, 40] == -math.inf).all()
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[at >= 3, :4, 5] = True
    hit[at >= 4, 4:, 6] = True
    hit[at >= 70, 4:, 40] = True
    assert (out[~hit].double() - clean[~hit].double()).abs().max() < most * unit
    within(lse, clean_lse, torch.full_like(lse, 2.0 ** -16))
    assert torch.equal(call().view(torch.uint8), out.view(torch.uint8))
    # keys: a NaN, and an infinity in one channel, whose sign in the scores is the query's
    k[1200, 1, 2] = math.nan
    k[700, 0, 9] = math.inf
    out, lse = call(return_lse=True)
    up = (q[n - lq:, :4, 9] > 0) & (at >= 700)[:, None]
    down = (q[n - lq:, :4, 9] < 0) & (at >= 700)[:, None]
    assert out[at >= 1200, 4:].isnan().all() and lse[at >= 1200, 4:].isnan().all()
    assert out[:, :4][up].isnan().all() and (lse[:, :4][up] == math.inf).all()
    sees = out[:, :4][down]
    assert sees[:, 5].isnan().all() and sees[:, :5].isfinite().all() and lse[:, :4][down].isfinite().all()
    assert torch.equal(call().isnan(), out.isnan())


@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores_and_scales(cuda_lib, dtype):
    """Rows whose weight lies on one key, maxima that grow along the row, a scale of zero, a negative one."""
    n = 400
    q, k, v = make(n, n, 2, 2, 128, dtype)
    grow = torch.linspace(0.0, 8.0, n, device="cuda")[:, None, None]
    k2 = (k.float() * grow).to(dtype)
    for keys, scale in ((k2, 0.5), (k2.flip(0).contiguous(), 0.5), (k, 0.0), (k, -0.3), (k, 1e-3)):
        check(q, keys, v, starts_of([n]), scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_alike_values_come_back(cuda_lib, dtype):
    """Whatever the weights, an average of one value is that value, up to the two sums' roundings."""
    q, k, v = make(700, 700, 2, 1, 128, dtype)
    v.fill_(1.25)
    out = b2q.prompt_attention(q, k, v, starts_of([700]))
    unit = {torch.float32: (700 / 4 + 16) * 2.0 ** -22, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}[dtype]
    assert (out.double() - 1.25).abs().max() <= 1.25 * unit


def test_views_and_strides(cuda_lib):
    for dtype in TYPES:
        wide = make(200, 200, 8, 8, 160, dtype)
        starts = starts_of([120, 80])
        cut = [x[:, ::2, 16:80] for x in wide]     # heads and channels apart
        check(*cut, starts)
        odd = [x[:, 1:5, 3:67] for x in wide]      # not aligned
        check(*odd, starts)
        turned = [x.transpose(0, 1).contiguous().transpose(0, 1)[..., :64] for x in wide]  # heads outermost
        check(*turned, starts)
        apart = [x[..., ::2] for x in wide]        # channels apart
        check(*apart, starts)
        q = wide[0][:, :4, :64]
        one = wide[1][:, :1, :64].expand(200, 4, 64)  # one key head for all, by a stride of zero
        check(q, one, one, starts)


def test_bad_starts_are_reported(cuda_lib):
    q, k, v = make(100, 100, 2, 2, 64, torch.float16)
    good, _ = check(q, k, v, starts_of([40, 30, 30]))
    for bad in ([0, 40, 39, 39], [0, 40, 70, 101], [-1, 40, 70, 100], [0, 2 ** 31 - 1, 70, 100]):
        out = torch.full_like(q, 3.0)
        b2q.prompt_attention(q, k, v, torch.tensor(bad, dtype=torch.int32, device="cuda"), out=out)
        with pytest.raises(b2q.B200QError, match="starts"):
            b2q.device_error()
        ok = [i for i in range(3) if 0 <= bad[i] <= bad[i + 1] <= 100]
        for i in ok:
            if [bad[i], bad[i + 1]] in ([0, 40], [40, 70], [70, 100]):
                assert torch.equal(out[bad[i]:bad[i + 1]], good[bad[i]:bad[i + 1]])
        covered = torch.zeros(100, dtype=torch.bool, device="cuda")
        for i in ok:
            covered[bad[i]:bad[i + 1]] = True
        assert (out[~covered] == 3).all()
    b2q.device_error()


def test_nothing_to_do_and_refusals(cuda_lib):
    q, k, v = make(10, 10, 2, 2, 64, torch.float16)
    s = starts_of([10])
    assert b2q.prompt_attention(q[:0], k[:0], v[:0], starts_of([0])).shape == (0, 2, 64)
    assert b2q.prompt_attention(q, k, v, starts_of([])).shape == (10, 2, 64)
    out, lse = b2q.prompt_attention(q, k[:0], v[:0], s, starts_of([0]), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    with pytest.raises(RuntimeError, match="divide"):
        b2q.prompt_attention(make(10, 10, 3, 2, 64, torch.float16)[0], k, v, s)
    with pytest.raises(RuntimeError, match="starts of the keys"):
        b2q.prompt_attention(q[:9], k, v, s)
    with pytest.raises(RuntimeError, match="256"):
        b2q.prompt_attention(*make(10, 10, 2, 2, 257, torch.float16), s)
    with pytest.raises(RuntimeError, match="finite"):
        b2q.prompt_attention(q, k, v, s, scale=math.inf)
    with pytest.raises(TypeError):
        b2q.prompt_attention(q, k.float(), v, s)
    with pytest.raises(TypeError):
        b2q.prompt_attention(q, k, v, s.long())
    with pytest.raises(RuntimeError, match="k_starts"):
        b2q.prompt_attention(q, k, v, s, starts_of([5, 5]))
    with pytest.raises(RuntimeError, match="channels"):
        b2q.prompt_attention(q, k, v[:, :1], s)
    with pytest.raises(RuntimeError, match="out"):
        b2q.prompt_attention(q, k, v, s, out=torch.empty(10, 2, 63, device="cuda", dtype=torch.float16))


@pytest.mark.parametrize("dtype", TYPES)
def test_streams_and_graphs(cuda_lib, dtype):
    """A captured call takes other lengths in a replay."""
    q, k, v = make(500, 500, 8, 2, 128, dtype, fused=True)
    starts = starts_of([100, 300, 100])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out, lse = b2q.prompt_attention(q, k, v, starts, return_lse=True, stream=side)
    side.synchronize()
    check(q, k, v, starts, out=out, lse=lse)
    again = torch.empty_like(out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _, lse = b2q.prompt_attention(q, k, v, starts, out=again, return_lse=True)
    for lens in ([500, 0, 0], [1, 1, 498], [200, 150, 150]):
        starts.copy_(starts_of(lens))
        g.replay()
        check(q, k, v, starts, out=again, lse=lse)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_call_repeats_bit_for_bit(cuda_lib, dtype):
    q, k, v = make(900, 900, 8, 2, 128, dtype)
    starts = starts_of([600, 300])
    first = b2q.prompt_attention(q, k, v, starts, return_lse=True)
    for _ in range(3):
        again = b2q.prompt_attention(q, k, v, starts, return_lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 80, 256])
@pytest.mark.parametrize("lq,lk", [([28], [3138]), ([3, 20, 0, 1], [3000, 1500, 700, 5000]), ([1, 1, 64], [4096, 10, 65]), ([70], [7000]),
                                   ([30, 5], [3, 2500])])
def test_few_rows_over_many_keys(cuda_lib, dtype, d, lq, lk):
    """The keys are cut into parts whose sums a second kernel joins: parts that end inside a sequence, that a row does not see, that are empty."""
    q, k, v = make(sum(lq), sum(lk), 4, 1, d, dtype, d)
    out, lse = check(q, k, v, starts_of(lq), starts_of(lk))
    again = b2q.prompt_attention(q, k, v, starts_of(lq), starts_of(lk), return_lse=True)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_parts_leave_other_rows_and_masked_values_out(cuda_lib, dtype):
    lq, lk = [5, 16], [2600, 3000]
    q, k, v = make(30, sum(lk) + 9, 4, 2, 64, dtype)
    starts = torch.tensor([2, 7, 23], dtype=torch.int32, device="cuda")
    k_starts = torch.tensor([4, 2604, 5604], dtype=torch.int32, device="cuda")
    for x in (k, v):
        x[:4] = math.nan
        x[5604:] = math.inf
    clean = torch.full_like(q, 3.0)
    _, clean_lse = b2q.prompt_attention(q, k, v, starts, k_starts, out=clean, return_lse=True)
    check(q, k, v, starts, k_starts, out=clean, lse=clean_lse)
    assert (clean[:2] == 3).all() and (clean[23:] == 3).all()
    most = float(v[4:5604].abs().max())
    v[2603, 0, 7] = math.nan   # the first sequence's last key: its last row alone sees it
    v[4000, 1, 9] = -math.inf  # all rows of the second
    out = torch.full_like(q, 3.0)
    b2q.prompt_attention(q, k, v, starts, k_starts, out=out)
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[6, :2, 7] = True
    hit[7:23, 2:, 9] = True
    assert out[6, :2, 7].isnan().all() and (out[7:23, 2:, 9] == -math.inf).all()
    unit = 3 * UNIT[dtype] + (3000 / 4 + 16) * 2.0 ** -22
    assert (out[~hit].double() - clean[~hit].double()).abs().max() < most * unit


@pytest.mark.parametrize("dtype", TYPES)
def test_parts_in_a_graph_beside_cache_attention(cuda_lib, dtype):
    """The parts' counters are the stream's scratch, which the cache attention uses too: both find it as they left it."""
    q, k, v = make(12, 4000, 4, 2, 64, dtype)
    starts, k_starts = starts_of([8, 4]), starts_of([2500, 1500])
    cache = b2q.KV4Cache.empty(80, 2, 64, 64, 32)
    b2q.kv4_append(cache, k, v, torch.arange(4000, device="cuda"))
    table, lens = torch.arange(80, device="cuda").int().view(2, 40), torch.tensor([2500, 1500], device="cuda").int()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = b2q.kv4_attention(q[:2, None], cache, table, lens)
        out, lse = b2q.prompt_attention(q, k, v, starts, k_starts, return_lse=True)
        second = b2q.kv4_attention(q[:2, None], cache, table, lens)
    side.synchronize()
    # bit for bit: the second sequence's last 60 places were not written (2560 + 1500 of 4000 slots) and may hold NaN
    assert torch.equal(first.view(torch.uint8), second.view(torch.uint8))
    check(q, k, v, starts, k_starts, out=out, lse=lse)
    held = torch.empty_like(out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        _, lse = b2q.prompt_attention(q, k, v, starts, k_starts, out=held, return_lse=True)
    for cut in ([2500, 1500], [12, 3988], [4000, 0]):
        k_starts.copy_(starts_of(cut))
        g.replay()
        check(q, k, v, starts, k_starts, out=held, lse=lse)
    fresh = torch.cuda.Stream()  # no scratch yet
    with pytest.raises(RuntimeError, match="scratch"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=fresh):
            b2q.prompt_attention(q, k, v, starts, k_starts)


@pytest.mark.parametrize("dtype", TYPES)
def test_bad_starts_where_keys_are_in_parts(cuda_lib, dtype):
    """Rows that two sequences claim are nobody's; what lies outside stays, and the stream's scratch is as it was for the next call."""
    q, k, v = make(40, 6000, 2, 1, 64, dtype)
    for rows in ([0, 20, 10, 28], [0, 28, 0, 28], [28, 0, 28, 5]):
        out = torch.full((40, 2, 64), 7.0, device="cuda", dtype=dtype)
        starts = torch.tensor(rows, dtype=torch.int32, device="cuda")
        b2q.prompt_attention(q, k, v, starts, torch.tensor([0, 2000, 4000, 6000], dtype=torch.int32, device="cuda"), out=out)
        with pytest.raises(b2q.B200QError, match="starts"):
            b2q.device_error()
        assert (out[28:] == 7).all()
        check(q, k, v, starts_of([10, 30]), starts_of([2500, 3500]))
