"""8-bit rows: quantize_s8, rms_norm_s8 and what is read back, against their definition in 64 bits."""
import math

import pytest
import torch

import my_own_cnn_b200 as b2q
from tests import s8_ref
from tests.lowbit_ref import UNIT, within

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def make(t, n, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(t, n, generator=g) * scale).to(dtype).cuda()


def check(rows, x, weight=None, residual=None, eps=None, total=None):
    codes, scales, h = s8_ref.rows(x, weight, residual, eps)
    torch.cuda.synchronize()
    assert torch.equal(rows.codes[..., :rows.k].flatten(0, -2).double(), codes)
    nan = scales.isnan()
    assert torch.equal(rows.scales.flatten().isnan(), nan)
    within(rows.scales.flatten()[~nan], scales[~nan], s8_ref.SCALE * scales[~nan])
    if total is not None:
        assert torch.equal(total.isnan(), h.isnan()) and torch.equal(total.nan_to_num(), h.nan_to_num())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,n", [(1, 1), (3, 7), (5, 16), (9, 250), (2, 512), (4, 520), (17, 1024), (3, 2049), (6, 4096), (3, 5003),
                                 (2, 8192), (2, 16384), (1, 16392), (1, 40001), (1, 65536)])
def test_quantized_rows(cuda_lib, dtype, t, n):
    x = make(t, n, dtype, n)
    rows = b2q.quantize_s8(x)
    assert b2q.last_path() == "rows-s8" and rows.shape == (t, n) and rows.codes.shape[-1] == -(-n // 16) * 16
    check(rows, x)
    for to in TYPES:
        y = rows.dequantize(to)
        want = rows.codes[:, :n].double() * rows.scales.double()[:, None]
        within(y, want, (UNIT[to] + 2.0 ** -24) * want.abs() + 2.0 ** -25)  # fp16: smaller ones are subnormal


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,n", [(1, 1), (3, 7), (9, 250), (33, 512), (4, 4096), (3, 5003), (2, 16384), (1, 40001)])
def test_normed_rows(cuda_lib, dtype, t, n):
    x, w, r = make(t, n, dtype, n), make(1, n, dtype, 1)[0], make(t, n, dtype, 2, 3.0)
    check(b2q.rms_norm_s8(x, w, eps=1e-5), x, w, None, 1e-5)
    check(b2q.rms_norm_s8(x, None), x, None, None, 1e-6)
    total = torch.full_like(x, 7)
    rows, got = b2q.rms_norm_s8(x, w, residual=r, residual_out=total)
    assert got is total
    check(rows, x, w, r, 1e-6, total)
    # in place: over the residual, and over x
    kept = r.clone()
    rows, got = b2q.rms_norm_s8(x, w, residual=kept)
    assert got is kept
    check(rows, x, w, r, 1e-6, kept)
    over = x.clone()
    rows, got = b2q.rms_norm_s8(over, w, residual=r, residual_out=over)
    check(rows, x, w, r, 1e-6, over)


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows_and_given_outputs(cuda_lib, dtype):
    wide = make(12, 700, dtype)
    w = make(1, 256, dtype, 4)[0]
    for x in (wide[:, 8:264], wide[:, 3:259], wide[::2, 16:272], wide.t()[:256].t()[:, :256]):
        check(b2q.rms_norm_s8(x, w), x, w, None, 1e-6)
    # one row for all
    x = wide[:1, :256].expand(5, 256)
    check(b2q.quantize_s8(x), x)
    # three dimensions, outputs of the caller
    x = make(6, 256, dtype, 8).view(2, 3, 256)
    out = b2q.S8Rows.empty(x.shape)
    out.codes.fill_(99)
    assert b2q.quantize_s8(x, out=out) is out
    check(out, x.view(6, 256))
    # a sum with a row stride of its own, x and residual in other strides; what lies beside it stays
    room = torch.full((12, 400), 5.0, dtype=dtype, device="cuda")
    a, r = wide[:, 8:264], wide[:, 300:556]
    rows, total = b2q.rms_norm_s8(a, w, residual=r, residual_out=room[:, 16:272])
    check(rows, a, w, r, 1e-6, total)
    assert (room[:, :16] == 5).all() and (room[:, 272:] == 5).all()


@pytest.mark.parametrize("n", [64, 250, 4096, 20000])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_at_the_edges_of_the_range(cuda_lib, dtype, n):
    x = make(14, n, dtype, 3)
    x[0] = 0
    x[1, n // 2] = math.nan
    x[2, n - 1] = math.inf
    x[3, 0] = -math.inf
    x[4] = torch.finfo(dtype).max
    x[5] = -torch.finfo(dtype).max
    x[6, 1:] = 0
    x[7] = torch.finfo(dtype).tiny
    x[8] *= 1e-4
    x[9] = 127.0  # every code at its end
    x[10] = torch.where(torch.arange(n, device="cuda") % 2 == 0, 127.0, 0.5).to(dtype)  # ties
    x[10, 1::4] *= 3
    x[11] = math.nan
    if dtype != torch.float16:
        x[12] *= 2.0 ** 100  # squares past fp32
        x[13] *= 2.0 ** -100
    check(b2q.quantize_s8(x), x)
    w = make(1, n, dtype, 6)[0]
    for eps in (1e-6, 0.0, 2.0 ** -60):
        check(b2q.rms_norm_s8(x, w, eps=eps), x, w, None, eps)
    r = make(14, n, dtype, 9)
    rows, total = b2q.rms_norm_s8(x, w, residual=r, residual_out=torch.empty_like(x))
    check(rows, x, w, r, 1e-6, total)
    y = rows.dequantize(torch.float32)
    assert torch.equal(y.isnan().all(-1), rows.scales.isnan()) and torch.equal(y.isnan().any(-1), rows.scales.isnan())


def test_many_rows_and_no_rows(cuda_lib):
    x = make(40000, 24, torch.bfloat16)
    check(b2q.quantize_s8(x), x)
    none = b2q.quantize_s8(x[:0])
    assert none.shape == (0, 24) and none.dequantize().shape == (0, 24)
    rows, total = b2q.rms_norm_s8(x[:0], None, residual=x[:0])
    assert rows.shape == (0, 24) and total.shape == (0, 24)


def test_refusals(cuda_lib):
    x = make(4, 64, torch.float32)
    with pytest.raises(RuntimeError, match="without a residual"):
        b2q.rms_norm_s8(x, None, residual_out=x)
    with pytest.raises(RuntimeError, match="eps"):
        b2q.rms_norm_s8(x, None, eps=-1e-6)
    with pytest.raises(RuntimeError, match="eps"):
        b2q.rms_norm_s8(x, None, eps=math.nan)
    with pytest.raises(RuntimeError, match="weight"):
        b2q.rms_norm_s8(x, x[0, :63])
    with pytest.raises(TypeError):
        b2q.rms_norm_s8(x, x[0].half())
    with pytest.raises(TypeError):
        b2q.quantize_s8(x.int())
    with pytest.raises(RuntimeError, match="at least 1"):
        b2q.quantize_s8(x[:, :0])
    with pytest.raises(RuntimeError, match="overlap"):
        b2q.rms_norm_s8(x, None, residual=x.clone(), residual_out=x[:1].expand(4, 64))
    with pytest.raises(RuntimeError, match="out"):
        b2q.quantize_s8(x, out=b2q.S8Rows.empty((4, 65)))
    with pytest.raises(RuntimeError, match="CUDA"):
        b2q.quantize_s8(x.cpu())
    with pytest.raises(RuntimeError):
        b2q.S8Rows(torch.zeros(4, 24, dtype=torch.int8, device="cuda"), torch.zeros(4, device="cuda"), 24)


def test_streams_and_graphs(cuda_lib):
    x = make(33, 4096, torch.bfloat16)
    w, r = make(1, 4096, torch.bfloat16, 2)[0], make(33, 4096, torch.bfloat16, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    rows, total = b2q.rms_norm_s8(x, w, residual=r, residual_out=torch.empty_like(x), stream=side)
    y = rows.dequantize(torch.bfloat16, stream=side)
    side.synchronize()
    check(rows, x, w, r, 1e-6, total)
    within(y, rows.codes.double() * rows.scales.double()[:, None], 2.0 ** -7 * y.double().abs())
    out, kept = b2q.S8Rows.empty(x.shape), torch.empty_like(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b2q.rms_norm_s8(x, w, residual=r, residual_out=kept, out=out)
    for seed in (5, 6):
        x.copy_(make(33, 4096, torch.bfloat16, seed))
        g.replay()
        check(out, x, w, r, 1e-6, kept)
