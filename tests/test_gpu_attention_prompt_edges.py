"""prompt_attention where values, scores and weights lie at the ends of their ranges; bounds are s8_ref's unless a test derives its own."""
import math

import pytest
import torch

import my_own_cnn_b200 as b2q
from tests import s8_ref
from tests.lowbit_ref import UNIT, within

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def starts_of(*lens):
    return torch.tensor([0, *lens]).cumsum(0).to(torch.int32).cuda()


def make(tq, tk, hq, hk, d, dtype, seed=0, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, h, d, generator=g, device="cuda") * s).to(dtype) for n, h, s in ((tq, hq, size), (tk, hk, 1), (tk, hk, 1))]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lq,lk,cut", [(50, 300, 64), (50, 300, 70), (50, 300, 130), (140, 700, 500), (28, 7000, 3000)])
def test_keys_masked_by_scores_of_minus_infinity(cuda_lib, dtype, d, lq, lk, cut):
    """The first keys' scores are -inf (a key of -inf in a channel that is 1 in all queries), the others' about -40: softmax of the
    others alone, whatever lies between them and 0."""
    q, k, v = make(lq, lk, 2, 1, d, dtype, d, 0.1)
    q[:, :, :2] = 1
    k[:, :, 0], k[:, :, 1] = 0, -40
    k[:cut, :, 0] = -math.inf
    out, lse = b2q.prompt_attention(q, k, v, starts_of(lq), starts_of(lk), 1.0, return_lse=True)
    want, want_lse, ob, lb = s8_ref.attention(q, k[cut:], v[cut:], starts_of(lq), starts_of(lk - cut), 1.0, dtype)
    within(out, want, ob)
    within(lse, want_lse, lb)


def same_kind(a, b):
    """NaN and infinities in the same places."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a == math.inf, b == math.inf) and torch.equal(a == -math.inf, b == -math.inf)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("low", [-30.0, -200.0])
def test_values_under_weights_that_vanish(cuda_lib, dtype, d, low):
    """A NaN and an infinity among values whose keys' scores lie far below the others' (their weights are zero in fp32 at -200): what the
    row gives does not depend on the parts that its keys are cut into.  160 heads of the same numbers are not cut."""
    q, k, v = make(8, 6000, 2, 1, d, dtype, d)
    q[:, :, 0] = 1
    k[:, :, 0] = 0
    k[:1000, :, 0] = low
    v[10, 0, 5] = math.nan
    v[11, 0, 6] = math.inf
    v[5995, 0, 7] = -math.inf  # at a weight above zero, seen by some rows
    ends = starts_of(8), starts_of(6000)
    out, lse = b2q.prompt_attention(q, k, v, *ends, 1.0, return_lse=True)
    whole, whole_lse = b2q.prompt_attention(q.repeat(1, 80, 1), k.expand(6000, 160, d), v.expand(6000, 160, d), *ends, 1.0, return_lse=True)
    assert out[:, :, 5].isnan().all()
    assert same_kind(out, whole[:, :2]) and lse.isfinite().all()
    assert (out[3:, :, 7] == -math.inf).all() and out[:3, :, 7].isfinite().all()
    # the rest is the softmax of what is left without the three channels
    keep = [c for c in range(d) if c not in (5, 6, 7)]
    want, want_lse, ob, lb = s8_ref.attention(q, k, v.nan_to_num(0, 0, 0), *ends, 1.0, dtype)
    within(out[..., keep], want[..., keep], ob[..., keep])
    within(whole[:, :2][..., keep], want[..., keep], ob[..., keep])
    within(lse, want_lse, lb)


@pytest.mark.parametrize("dtype", TYPES)
def test_scales_at_the_end_of_the_range(cuda_lib, dtype):
    """2.3e38 is the largest that is taken, in size: scores of zero are all alike."""
    q, k, v = make(300, 300, 2, 1, 64, dtype)
    for scale in (2.4e38, -3e38, 1e39, math.inf, math.nan):
        with pytest.raises(RuntimeError, match="scale"):
            b2q.prompt_attention(q, k, v, starts_of(300), scale=scale)
    k.zero_()
    for scale in (2.3e38, -2.3e38):
        out, lse = b2q.prompt_attention(q, k, v, starts_of(300), scale=scale, return_lse=True)
        want, want_lse, ob, lb = s8_ref.attention(q, k, v, starts_of(300), starts_of(300), scale, dtype)
        within(out, want, ob)
        within(lse, want_lse, lb)
    with pytest.raises(RuntimeError, match="256"):
        b2q.prompt_attention(q[..., :0], k[..., :0], v[..., :0], starts_of(300))


def best_ms(call, times=3):
    call()
    best = math.inf
    for _ in range(times):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        call()
        end.record()
        end.synchronize()
        best = min(best, start.elapsed_time(end))
    return best


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lq,inf,nan", [(500, 3, 300), (500, 300, 3), (500, 130, 131), (20, 3, 3990), (20, 3990, 3), (20, 1000, 2000)])
def test_log_sums_of_infinite_scores(cuda_lib, dtype, d, lq, inf, nan):
    """A score of +inf gives the log-sum +inf unless another one is NaN, and a NaN row either way; -inf has no part in it.  Rows of 500
    keys, and the last 20 of 4000 (in parts)."""
    n = 500 if lq == 500 else 4000
    q, k, v = make(lq, n, 4, 1, d, dtype, d)
    k[inf, :, 9] = math.inf
    k[nan, :, 2] = math.nan
    out, lse = b2q.prompt_attention(q, k, v, starts_of(lq), starts_of(n), return_lse=True)
    at = torch.arange(n - lq, n, device="cuda")[:, None]
    bad = (at >= nan).expand(lq, 4)
    up = (at >= inf) & ~bad & (q[..., 9] > 0)
    assert lse[bad].isnan().all() and out[bad].isnan().all()
    assert (lse[up] == math.inf).all() and out[up].isnan().all()
    left = ~bad & ~up
    assert lse[left].isfinite().all() and out[left].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lse", [True, False])
def test_an_infinite_key_costs_no_more(cuda_lib, dtype, lse):
    """Every row sees a score of +inf or -inf."""
    q, k, v = make(2048, 2048, 32, 8, 128, dtype)
    clean = best_ms(lambda: b2q.prompt_attention(q, k, v, starts_of(2048), return_lse=lse))
    k[3, :, 5] = math.inf
    assert best_ms(lambda: b2q.prompt_attention(q, k, v, starts_of(2048), return_lse=lse)) < 10 * clean


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("place", [3, 1024])
def test_a_value_that_is_not_finite_costs_little(cuda_lib, dtype, value, place):
    """All rows from `place` on have one channel that is not finite; a warp finds the reason for all of its rows in one read."""
    q, k, v = make(2048, 2048, 32, 8, 128, dtype)
    call = lambda: b2q.prompt_attention(q, k, v, starts_of(2048))
    clean = best_ms(call)
    v[place, :, 5] = value
    assert best_ms(call) < 10 * clean
    out = call()
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[place:, :, 5] = True
    assert out[~hit].isfinite().all() and not out[hit].isfinite().any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [1, 33, 64, 80, 128, 200, 256])
def test_rows_done_again_key_by_key(cuda_lib, dtype, d):
    """Poison in the middle of tiles: rows before it see none of it, those after see it (NaN, or two infinities) in some channels; what
    is left of them is as without."""
    n, hq, hk = 611, 6, 2
    q, k, v = make(n, n, hq, hk, d, dtype, d)
    starts = starts_of(n)
    want, want_lse, ob, lb = s8_ref.attention(q, k, v, starts, starts, d ** -0.5, dtype)
    for place in (0, 37, 300, 610):
        bad = v.clone()
        bad[place, 0, 0] = math.nan
        bad[place // 2, 1, d // 2] = math.inf
        bad[place, 1, d // 2] = -math.inf
        out, lse = b2q.prompt_attention(q, k, bad, starts, return_lse=True)
        hit = torch.zeros(n, hq, d, dtype=torch.bool)
        hit[place:, :3, 0] = True
        hit[place // 2:, 3:, d // 2] = True
        assert out.cpu()[place:, :3, 0].isnan().all()
        assert (out.cpu()[place // 2:place, 3:, d // 2] == math.inf).all()
        after = out.cpu()[place:, 3:, d // 2]
        assert after.isnan().all() if place // 2 < place else (after == -math.inf).all()
        within(out.cpu()[~hit], want[~hit], ob[~hit])
        within(lse, want_lse, lb)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_infinite_values_in_fp32_cost_no_more(cuda_lib, d):
    """Keys masked by a score of -inf and an infinite value in fp32, whose operands are three terms each: right, and at the speed of finite
    ones."""
    n, cut = 1024, 100
    q, k, v = make(n, n, 16, 4, d, torch.float32, d)
    q[:, :, 0] = 1
    k[:, :, 0] = 0
    rows = slice(cut, n)
    ends = starts_of(n - cut), starts_of(n)
    clean = best_ms(lambda: b2q.prompt_attention(q[rows], k, v, *ends, return_lse=True))
    k[:cut, :, 0] = -math.inf
    v[cut, :, 5] = math.inf
    call = lambda: b2q.prompt_attention(q[rows], k, v, *ends, return_lse=True)
    assert best_ms(call) < 5 * clean
    out, lse = call()
    assert (out[..., 5] == math.inf).all()
    v[cut, :, 5] = 0
    want, want_lse, ob, lb = s8_ref.attention(q[rows], k[rows], v[rows], ends[0], ends[0], d ** -0.5, torch.float32)
    keep = [c for c in range(d) if c != 5]
    within(out[..., keep], want[..., keep], ob[..., keep])
    within(lse, want_lse, lb)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 80, 256])
@pytest.mark.parametrize("lens,b", [((1, 90, 63, 64), 4), ((128, 129, 1), 3), ((300, 0, 77, 500, 31), 5), (tuple(i % 9 for i in range(40)), 40)])
def test_what_lies_behind_a_sequence_changes_no_bit(cuda_lib, dtype, d, lens, b):
    """Rows behind the last sequence, and every other sequence: finite or poison, the rest gives the same bits."""
    n = sum(lens)
    q, k, v = make(n + 50, n + 50, 4, 2, d, dtype, d)
    starts = starts_of(*lens)
    clean, clean_lse = b2q.prompt_attention(q, k, v, starts, return_lse=True)
    at = starts.tolist()
    for value in (math.nan, math.inf, -math.inf):
        p = [x.clone() for x in (q, k, v)]
        for x in p:
            x[n:] = value
            for i in range(1, b, 2):
                x[at[i]:at[i + 1]] = value
        out, lse = b2q.prompt_attention(*p, starts, return_lse=True)
        for i in range(0, b, 2):
            rows = slice(at[i], at[i + 1])
            assert torch.equal(out[rows], clean[rows]) and torch.equal(lse[rows], clean_lse[rows])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lq", [28, 200])
def test_what_lies_behind_earlier_parts_changes_no_bit(cuda_lib, dtype, lq):
    """The same where the keys are in parts (28 rows) and where sequences have more keys than queries."""
    lk = (3000 - 7, 2000)
    q, k, v = make(2 * lq, 5000, 4, 1, 64, dtype)
    ends = starts_of(lq, lq), starts_of(*lk)
    clean, clean_lse = b2q.prompt_attention(q, k, v, *ends, return_lse=True)
    for x in (k, v):
        x[lk[0]:] = math.nan
    out, lse = b2q.prompt_attention(q, k, v, *ends, return_lse=True)
    assert torch.equal(out[:lq], clean[:lq]) and torch.equal(lse[:lq], clean_lse[:lq])
    assert out[lq:].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_poison_behind_a_prompt_costs_no_more(cuda_lib, dtype):
    q, k, v = make(2048, 2048, 32, 8, 128, dtype)
    call = lambda: b2q.prompt_attention(q, k, v, starts_of(2028))
    clean = best_ms(call)
    for x in (q, k, v):
        x[2028:] = math.nan
    assert best_ms(call) < 3 * clean


@pytest.mark.parametrize("d,aligned", [(64, True), (128, True), (64, False), (256, True)])
def test_small_fp16_weights_add_up(cuda_lib, d, aligned):
    """One key far above 20000 others at 2^-24.6 of its weight, whose values alone are not zero: weights of half that precision would be
    subnormal (1 % off, 50 % without a factor).

    Off by: a weight's rounding and the result's 2^-11 each, the exponent's (24.6 * 2^-24, its product with log2(e) the same, the
    exponential 2^-21) 2^-18 in all, sums (n / 4 + 16) 2^-23.  So is the log-sum: additions of 2^-24.6 (n / 4 of them one after another in a
    lane, or sums of 64) to a sum of 1 are each off by up to 2^-24 of it, and its logarithm near 0 by as much."""
    n, heads = 20000, 80  # heads: enough that the keys are not cut into parts
    room = 0 if aligned else 1
    q = torch.zeros(1, heads, d + room, dtype=torch.float16, device="cuda")[..., room:]
    k, v = (torch.zeros(n, heads, d + room, dtype=torch.float16, device="cuda")[..., room:] for _ in range(2))
    q[..., 0] = 1
    k[1:, :, 0] = -17.05
    v[1:] = 1
    out, lse = b2q.prompt_attention(q, k, v, starts_of(1), starts_of(n), 1.0, return_lse=True)
    assert b2q.last_path() == ("tcgen05-prompt-attention" if aligned and d <= 128 else "mma-prompt-attention")
    rest = (n - 1) * math.exp(float(k[1, 0, 0]))
    want = torch.full_like(out, 0, dtype=torch.float64) + rest / (1 + rest)
    within(out, want, want * (2 * 2.0 ** -11 + 2.0 ** -18 + (n / 4 + 16) * 2.0 ** -23))
    assert (lse.double() - math.log1p(rest)).abs().max() < (n / 4 + 16) * 2.0 ** -23 + 2.0 ** -20


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("d,keys", [(64, 131072), (128, 66001), (256, 40000), (64, 8192), (64, 8193)])
def test_sums_of_many_keys_have_no_bias(cuda_lib, dtype, d, keys):
    """Values of one sign over many keys, in one part: an adder that truncates makes all results low, the more the longer.

    The mean of (result - value) / value over 80 heads: roundings to 16 bits average out (2^-9 / sqrt(80 * 64 * 3) = 1.6e-5 for bf16), weights'
    far more so; what is left are the sums of 8192 keys, 512 products of 16 that may lose 2^-23 of the sum each: 6.1e-5."""
    heads = 80
    g = torch.Generator(device="cuda").manual_seed(d)
    q = torch.randn(1, heads, d, generator=g, device="cuda").to(dtype)
    k, v = (torch.empty(keys, heads, d, dtype=dtype, device="cuda") for _ in range(2))
    want, want_lse = torch.empty(heads, d, dtype=torch.float64, device="cuda"), torch.empty(heads, dtype=torch.float64, device="cuda")
    for h in range(heads):
        k[:, h] = torch.randn(keys, d, generator=g, device="cuda").to(dtype)
        size = 1 + torch.rand(d, generator=g, device="cuda")
        v[:, h] = ((0.5 + torch.rand(keys, d, generator=g, device="cuda")) * size).to(dtype)
        a = (k[:, h].double() @ q[0, h].double()) * d ** -0.5
        want_lse[h] = torch.logsumexp(a, 0)
        want[h] = torch.softmax(a, 0) @ v[:, h].double()
    out, lse = b2q.prompt_attention(q, k, v, starts_of(1), starts_of(keys), return_lse=True)
    off = (out[0].double() - want) / want
    assert abs(float(off.mean())) < 4 * 1.6e-5 + 512 * 2.0 ** -23
    assert float(off.abs().max()) < 2 * UNIT[dtype] + 512 * 2.0 ** -23  # the result and, at worst, all weights alike
    assert (lse[0].double() - want_lse).abs().max() < 2.0 ** -17


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("lq", [130, 5])
def test_long_rows_whose_maxima_grow(cuda_lib, dtype, d, lq):
    """More than 8192 keys whose scores grow along the row, shrink along it, or are -inf for the first 9000: what was summed up before
    is taken over at another reference.  Five rows are in parts."""
    keys = 20000
    q, k, v = make(lq, keys, 2, 1, d, dtype, d, 0.3)
    slope = torch.linspace(-30, 30, keys, device="cuda")
    q[..., 0] = 1
    starts, k_starts = starts_of(lq), starts_of(keys)
    for rise in (slope, -slope, -100 - slope.abs()):
        k[:, 0, 0] = rise.to(dtype)
        out, lse = b2q.prompt_attention(q, k, v, starts, k_starts, 1.0, return_lse=True)
        want, want_lse, ob, lb = s8_ref.attention(q, k, v, starts, k_starts, 1.0, dtype)
        within(out, want, ob)
        within(lse, want_lse, lb)
    q[..., 1], k[..., 1] = 1, 0
    k[:9000, :, 1] = -math.inf
    out, lse = b2q.prompt_attention(q, k, v, starts, k_starts, 1.0, return_lse=True)
    k[:9000, :, 1] = 0
    want, want_lse, ob, lb = s8_ref.attention(q, k[9000:], v[9000:], starts, starts_of(keys - 9000), 1.0, dtype)
    within(out, want, ob)
    within(lse, want_lse, lb)


@pytest.mark.parametrize("d", [64, 128, 80, 200])
@pytest.mark.parametrize("lq,lk", [(300, 300), (700, 700), (28, 7000), (130, 9000)])
def test_saturated_fp16_values_stay_finite(cuda_lib, d, lq, lk):
    """Channels whose values are all fp16's largest, or lie just below it: their average is no infinity, though a weight is rounded by
    up to 2^-11 and 65520 rounds to one.  Off by at most that and the result's own rounding."""
    q, k, v = make(lq, lk, 4, 4, d, torch.float16, d, 3.0)
    v[..., 3], v[..., 5] = 65504, -65504
    v[..., 7] = torch.where(v[..., 7] > 0, 65504.0, 65472.0).half()
    v[..., 9] = math.inf
    out = b2q.prompt_attention(q, k, v, starts_of(lq), starts_of(lk))
    for c, sign in ((3, 1), (5, -1), (7, 1)):
        assert out[..., c].isfinite().all() and (sign * out[..., c].double() >= 65472 * (1 - 2 * 2.0 ** -11 - 2.0 ** -13)).all()
    assert (out[..., 9] == math.inf).all()

@pytest.mark.parametrize("dtype", TYPES)
def test_which_kernel_takes_a_call(cuda_lib, dtype):
    """16-bit heads of up to 128 channels that are a multiple of 8, on 16-byte boundaries, at most 128 of them a key head: tcgen05; the rest and
    fp32: mma.sync."""
    starts = starts_of(20, 17)

    def path(q, k, v, **kw):
        b2q.prompt_attention(q, k, v, starts, **kw)
        return b2q.last_path()

    fast = "mma-prompt-attention" if dtype == torch.float32 else "tcgen05-prompt-attention"
    for d in (8, 40, 64, 72, 80, 128):
        assert path(*make(37, 37, 4, 2, d, dtype)) == fast
    for d in (1, 33, 60, 136, 256):
        assert path(*make(37, 37, 4, 2, d, dtype)) == "mma-prompt-attention"
    assert path(*make(37, 37, 128, 1, 64, dtype)) == fast and path(*make(37, 37, 129, 1, 64, dtype)) == "mma-prompt-attention"
    q, k, v = make(37, 37, 4, 2, 72, dtype)
    assert path(q[..., 8:], k[..., 8:], v[..., 8:]) == fast
    assert path(q[..., 1:65], k[..., 1:65], v[..., 1:65]) == "mma-prompt-attention"
    assert path(q, k, v, scale=0.0) == "mma-prompt-attention"
    assert path(q, k[:, :1].expand(37, 2, 72), v) == "mma-prompt-attention"


def test_many_hand_overs_of_sums(cuda_lib):
    """Rows of 40000 keys (four hand-overs) in 160 tiles, on all SMs, again and again: the same bits each time, and no wait runs out."""
    q, k, v = make(4, 160000, 40, 40, 64, torch.bfloat16)
    ends = starts_of(1, 1, 1, 1), starts_of(*[40000] * 4)
    first = b2q.prompt_attention(q, k, v, *ends)
    for _ in range(20):
        assert torch.equal(b2q.prompt_attention(q, k, v, *ends), first)
    b2q.device_error()
