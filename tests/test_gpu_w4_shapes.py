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
