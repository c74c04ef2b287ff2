"""linear_s8 against whole sums in 64 bits: every plan of the work, odd sizes, the ends of the integers' range."""
import math

import pytest
import torch

import my_own_cnn_b200 as b2q
from tests import s8_ref
from tests.lowbit_ref import within

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def rows(m, k, seed, pitch=None, lo=-128, hi=128):
    """Random codes; what lies past k is anything."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pitch = pitch or -(-k // 16) * 16
    codes = torch.randint(lo, hi, (m, pitch), generator=g, device="cuda", dtype=torch.int8)
    scales = torch.rand(m, generator=g, device="cuda") * 0.02 + 1e-3
    return b2q.S8Rows(codes, scales, k)


def check(x, w, bias=None, dtype=torch.float32, y=None):
    if y is None:
        y = b2q.linear_s8(x, w, bias, dtype=dtype)
        assert b2q.last_path() == "linear-s8"
    want, bound = s8_ref.linear(x.codes[..., :x.k].flatten(0, -2), x.scales.flatten(), w.codes[:, :w.k], w.scales, bias, dtype)
    within(y.flatten(0, -2), want, bound)
    return y


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 77, 128, 129, 200, 256, 257, 300, 511])
@pytest.mark.parametrize("n,k", [(1, 1), (130, 100), (256, 256), (1000, 1437)])
def test_small(cuda_lib, m, n, k):
    check(rows(m, k, m), rows(n, k, n))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k,bias", [(1, 4096, 4096, True), (7, 5003, 4091, True), (16, 2048, 8192, False), (48, 768, 768, True),
                                        (512, 4096, 1024, True), (1000, 2000, 3000, True), (2049, 4100, 640, False),
                                        (4096, 4096, 512, True), (5000, 8200, 129, True)])
def test_types_and_sizes(cuda_lib, dtype, m, n, k, bias):
    b = torch.randn(n, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype) if bias else None
    check(rows(m, k, 3), rows(n, k, 4), b, dtype)


@pytest.mark.parametrize("m", [1, 40, 300, 2100])
def test_sums_at_the_ends_of_the_range(cuda_lib, m):
    """-128 * -128 * 131071 is 16383 below 2^31; the other end is as near."""
    k, n = 131071, 270
    for xv, wv in ((-128, -128), (127, -128), (127, 127)):
        x, w = rows(m, k, 0), rows(n, k, 1)
        x.codes.fill_(xv)
        w.codes.fill_(wv)
        check(x, w)


def test_rows_by_rows(cuda_lib):
    """Each token and channel has its own numbers in the right place: one-hot operands."""
    for m, n, k in ((19, 300, 272), (2304, 2560, 200)):
        x, w = rows(m, k, 0), rows(n, k, 1)
        x.codes.zero_()
        x.codes[torch.arange(m), torch.arange(m) % k] = 1
        check(x, w)


def test_not_finite_scales_stay_in_their_rows(cuda_lib):
    for m in (5, 3000):
        x, w = rows(m, 500, 0), rows(700, 500, 1)
        x.scales[3] = math.nan
        w.scales[699] = math.inf
        w.scales[128] = math.nan
        y = b2q.linear_s8(x, w, dtype=torch.float16)
        assert y[3].isnan().all() and y[:, 128].isnan().all()
        keep = torch.ones_like(y, dtype=torch.bool)
        keep[3] = False
        keep[:, 128] = False
        keep[:, 699] = False
        assert y[keep].isfinite().all()


@pytest.mark.parametrize("m", [6, 2500])
def test_outputs_of_the_caller(cuda_lib, m):
    x, w = rows(m, 320, 0), rows(900, 320, 1)
    for dtype in TYPES:
        room = torch.full((m + 2, 1000), 5.0, dtype=dtype, device="cuda")
        for off in (0, 1, 50):
            room.fill_(5.0)
            y = room[1:m + 1, off:off + 900]
            assert b2q.linear_s8(x, w, dtype=dtype, out=y) is y
            check(x, w, None, dtype, y)
            assert (room[0] == 5).all() and (room[m + 1] == 5).all()
            assert (room[:, :off] == 5).all() and (room[:, off + 900:] == 5).all()
    lead = b2q.S8Rows(x.codes.view(2, m // 2, 320), x.scales.view(2, m // 2), 320)
    y = b2q.linear_s8(lead, w)
    assert y.shape == (2, m // 2, 900) and y.dtype == torch.bfloat16
    check(lead, w, None, torch.bfloat16, y)


def test_nothing_to_do_and_refusals(cuda_lib):
    x, w = rows(4, 64, 0), rows(8, 64, 1)
    none = b2q.S8Rows(x.codes[:0], x.scales[:0], 64)
    assert b2q.linear_s8(none, w).shape == (0, 8)
    assert b2q.linear_s8(x, none).shape == (4, 0)
    with pytest.raises(RuntimeError, match="rows of 64"):
        b2q.linear_s8(x, rows(8, 65, 1))
    with pytest.raises(RuntimeError, match="bias"):
        b2q.linear_s8(x, w, torch.zeros(9, device="cuda"), dtype=torch.float32)
    with pytest.raises(TypeError):
        b2q.linear_s8(x, w, torch.zeros(8, device="cuda"), dtype=torch.float16)
    with pytest.raises(TypeError):
        b2q.linear_s8(x, w, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="out"):
        b2q.linear_s8(x, w, out=torch.empty(4, 9, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="131071"):
        b2q.linear_s8(rows(1, 131072, 0), rows(1, 131072, 1))
    with pytest.raises(RuntimeError, match="aligned"):
        b2q.S8Rows(torch.zeros(40, dtype=torch.int8, device="cuda")[8:24].view(1, 16), torch.zeros(1, device="cuda"), 16)


def test_streams_and_graphs(cuda_lib):
    for m in (3, 2300):
        x, w = rows(m, 512, 0), rows(2600, 512, 1)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        y = b2q.linear_s8(x, w, dtype=torch.float32, stream=side)
        side.synchronize()
        check(x, w, y=y)
        out = torch.empty_like(y)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            b2q.linear_s8(x, w, dtype=torch.float32, out=out)
        for seed in (7, 8):
            x.codes.copy_(rows(m, 512, seed).codes)
            g.replay()
            check(x, w, y=out)
