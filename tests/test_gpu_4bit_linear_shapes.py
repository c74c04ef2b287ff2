"""linear_w4 where x has leading dimensions and there is nothing to sum or no row."""
import pytest
import torch

import my_own_cnn_b200 as b2q

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lead", [(), (1,), (0,), (2, 3), (2, 0, 3), (1, 2, 2, 2)])
@pytest.mark.parametrize("k", [0, 1, 64])
def test_leading_dimensions(lead, k):
    w = b2q.W4Weight(torch.zeros(5, -(-k // 32) * 16, dtype=torch.uint8, device="cuda"),
                     torch.ones(-(-k // 32), 5, dtype=torch.bfloat16, device="cuda"), None, 5, k, 32)  # every weight is -8
    bias = torch.arange(5.0, device="cuda")
    x = torch.rand(*lead, k, device="cuda").mul(16).round()
    y = b2q.linear_w4(x, w, bias)
    assert torch.equal(y, (-8 * x.sum(-1, keepdim=True) + bias).expand(*lead, 5))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m", [1, 3, 16])
def test_every_byte_as_a_zero_point(dtype, m):
    """Codes of formats whose zero points pass 15 (stored plus one, or of a wider type), at even and odd columns: a result is one
    product, exact up to its own rounding."""
    n, k = 256, 64
    codes = (torch.arange(n * k, device="cuda") % 16).view(n, k)
    zeros = torch.arange(n, device="cuda").view(n, 1).expand(n, 2).to(torch.uint8)
    w = b2q.pack_w4(codes, torch.full((n, 2), 0.25, device="cuda"), zeros, 32)
    for at in range(0, k, m):
        x = torch.zeros(m, k, device="cuda", dtype=dtype)
        for i in range(m):
            x[i, (at + i) % k] = 1
        want = (x.double() @ w.dequantize().double().t()).to(dtype)
        assert torch.equal(b2q.linear_w4(x, w), want)
