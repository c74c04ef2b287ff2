"""linear_w4 on the GPU against the 64-bit product of the values that the codes stand for."""
import pytest
import torch

import my_own_cnn_b200 as b2q
from lowbit_ref import UNIT, w4_values, within

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def gen(seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def case(n, k, group, symmetric=False, seed=0):
    return b2q.quantize_w4(torch.randn(n, k, generator=gen(seed), device="cuda") * k ** -0.5, group, symmetric)


def check(y, x, w, bias=None):
    v = w4_values(w)
    want = x.double() @ v.t()
    # one chain per 16 columns, the joins after it, and the bias
    bound = 2.0 ** -23 * (w.k / 16 + 64) * (x.double().abs() @ v.abs().t())
    if bias is not None:
        want = want + bias.double()
        bound = bound + 2.0 ** -23 * bias.double().abs()
    within(y, want, bound + 1.01 * UNIT[x.dtype] * want.abs() + (2.0 ** -25 if x.dtype == torch.float16 else 0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 16, 32), (1, 17, 33), (2, 130, 127), (3, 5, 2049), (7, 256, 256),
                                   (8, 128, 512), (9, 513, 1000), (16, 384, 4096), (17, 65, 640), (33, 300, 96),
                                   (1, 1031, 4099), (5, 64, 8192)])
def test_matches_the_product(dtype, group, m, n, k):
    w = case(n, k, group)
    x = torch.randn(m, k, generator=gen(1), device="cuda").to(dtype)
    bias = torch.randn(n, generator=gen(2), device="cuda").to(dtype) if n % 2 else None
    y = b2q.linear_w4(x, w, bias)
    assert y.dtype == dtype and y.shape == (m, n)
    check(y, x, w, bias)
    assert b2q.last_path() == "linear-w4"


@pytest.mark.parametrize("dtype", TYPES)
def test_symmetric_weights_and_large_and_small_rows(dtype):
    w = case(200, 777, 64, symmetric=True)
    assert w.zeros is None
    big = 3e4 if dtype == torch.float16 else 1e30
    x = torch.randn(4, 777, generator=gen(3), device="cuda")
    x = (x.clamp(-2, 2) / 2 * torch.tensor([1.0, big / 100, 1e-3, 1.0], device="cuda")[:, None]).to(dtype)
    x[3] = 0
    y = b2q.linear_w4(x, w)
    check(y, x, w)
    assert (y[3] == 0).all()


def test_every_code_and_zero_point():
    n, k = 64, 64
    codes = (torch.arange(n * k, device="cuda") % 16).view(n, k)
    zeros = torch.arange(n * 2, device="cuda").view(n, 2) % 16
    scales = torch.full((n, 2), 0.5, device="cuda")
    w = b2q.pack_w4(codes, scales, zeros, 32)
    x = torch.eye(k, device="cuda")[:, :k]
    want = (codes.float() - zeros.float().repeat_interleave(32, 1)) * 0.5
    for dtype in TYPES:
        assert torch.equal(b2q.linear_w4(x.to(dtype), w).float(), want.t())
    assert torch.equal(w.dequantize(), want)


def test_rows_with_strides_and_any_alignment():
    w = case(96, 200, 32)
    store = torch.randn(6, 1 + 230, generator=gen(4), device="cuda").bfloat16()
    for x in (store[:, 1:201], store[::2, 3:203], store[:, 0:200], store[:200 // 40].t()[:200].t()):
        check(b2q.linear_w4(x, w), x, w)
    x = store[:, 8:208]
    out = torch.full((6, 120), 7.0, device="cuda", dtype=torch.bfloat16)
    y = b2q.linear_w4(x, w, out=out[:, 5:101])
    check(y, x, w)
    assert (out[:, :5] == 7).all() and (out[:, 101:] == 7).all()
    cols = torch.randn(200, 3, generator=gen(5), device="cuda").t()  # columns apart
    check(b2q.linear_w4(cols, w), cols, w)


def test_broadcast_and_overlapping_rows():
    w = case(70, 96, 32)
    row = torch.randn(200, generator=gen(12), device="cuda")
    for x in (row[:96].expand(5, 96), row.as_strided((9, 96), (7, 1)), row[:96].expand(2, 3, 96)):
        assert torch.equal(b2q.linear_w4(x, w), b2q.linear_w4(x.contiguous(), w))


def test_out_must_be_on_the_device():
    w = case(8, 64, 32)
    with pytest.raises(RuntimeError, match="out must be"):
        b2q.linear_w4(torch.zeros(2, 64, device="cuda"), w, out=torch.zeros(2, 8))


def test_leading_dimensions_and_none():
    w = case(40, 64, 64)
    x = torch.randn(2, 3, 64, generator=gen(6), device="cuda")
    y = b2q.linear_w4(x, w)
    assert y.shape == (2, 3, 40)
    check(y.view(6, 40), x.view(6, 64), w)
    assert b2q.linear_w4(x[:, :0], w).shape == (2, 0, 40)
    empty = b2q.W4Weight(torch.empty(5, 0, dtype=torch.uint8, device="cuda"),
                         torch.empty(0, 5, dtype=torch.bfloat16, device="cuda"), None, 5, 0, 32)
    bias = torch.arange(5.0, device="cuda")
    assert torch.equal(b2q.linear_w4(x.new_empty(2, 0), empty, bias), bias.expand(2, 5))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(1, 40, 180001), (4, 64, 50001), (2, 700, 20000), (1, 9000, 300), (4, 5000, 700),
                                   (6, 5000, 2500), (16, 40, 30000)])
def test_shapes_of_every_split(dtype, m, n, k):
    """One and few rows with K shared out to warps and clusters, and past what they hold; K split two to eight ways."""
    w = case(n, k, 64)
    x = torch.randn(m, k, generator=gen(11), device="cuda").to(dtype)
    check(b2q.linear_w4(x, w), x, w)


def test_columns_past_k_are_not_used():
    """The nibbles that pad a row, and x beyond its k columns, may hold anything."""
    w = case(48, 50, 32)
    x = torch.randn(3, 64, generator=gen(7), device="cuda")
    x[:, 50:] = float("nan")
    want = b2q.linear_w4(x[:, :50].contiguous(), w)
    w.codes[:, 25:] = 0xFF
    assert torch.equal(b2q.linear_w4(x[:, :50], w), want)


def test_repeats_bit_for_bit_and_on_another_stream():
    w = case(1000, 3000, 64)
    x = torch.randn(4, 3000, generator=gen(8), device="cuda").half()
    want = b2q.linear_w4(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    ys = [b2q.linear_w4(x, w, stream=s) for _ in range(3)]
    ys.append(b2q.linear_w4(x, w, stream=s.cuda_stream))
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(y, want) for y in ys)


def test_in_a_graph():
    w = case(300, 500, 32)
    x = torch.randn(2, 500, generator=gen(9), device="cuda")
    b2q.linear_w4(x, w)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = b2q.linear_w4(x, w)
    x.copy_(torch.randn(2, 500, generator=gen(10), device="cuda"))
    g.replay()
    check(y, x, w)


def test_refusals():
    w = case(8, 64, 32)
    x = torch.zeros(2, 64, device="cuda")
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        b2q.linear_w4(x.double(), w)
    with pytest.raises(RuntimeError, match="63 columns"):
        b2q.linear_w4(x[:, :63], w)
    with pytest.raises(TypeError, match="bias"):
        b2q.linear_w4(x, w, torch.zeros(8, device="cuda").half())
    with pytest.raises(RuntimeError, match="bias"):
        b2q.linear_w4(x, w, torch.zeros(9, device="cuda"))
    with pytest.raises(RuntimeError, match="out must be"):
        b2q.linear_w4(x, w, out=torch.zeros(2, 9, device="cuda"))
    with pytest.raises(RuntimeError, match="CUDA device"):
        b2q.linear_w4(x.cpu(), w)
    with pytest.raises(RuntimeError, match="codes must be"):
        b2q.W4Weight(w.codes[:, :16], w.scales, w.zeros, 8, 64, 32)
    with pytest.raises(RuntimeError, match="scales must be"):
        b2q.W4Weight(w.codes, w.scales.float(), w.zeros, 8, 64, 32)
    with pytest.raises(RuntimeError, match="group"):
        b2q.W4Weight(w.codes, w.scales, w.zeros, 8, 64, 48)
