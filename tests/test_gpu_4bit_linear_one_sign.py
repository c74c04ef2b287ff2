"""linear_w4 on activations of one sign, as gates leave them: the sums of code * x and of zero point * x are then many times their
difference."""
import pytest
import torch

import my_own_cnn_b200 as b2q
from lowbit_ref import UNIT, w4_values

pytestmark = pytest.mark.gpu


def normal(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda")


X = {"squared": lambda x: x.relu().square(), "shifted": lambda x: x.abs() + 0.5, "ones": torch.ones_like, "falling": lambda x: -x.abs().exp(),
     "outliers": lambda x: torch.where(x > 2, 100 * x, x.abs())}


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(1, 700, 8192), (1, 40, 16384), (3, 64, 4096), (5, 1024, 8191), (16, 2048, 4096)])
@pytest.mark.parametrize("what", X)
def test_results_are_the_definition_rounded_once(dtype, group, m, n, k, what):
    """The adder truncates each sum over 16 columns at 2^-23 of its size, and what follows rounds to 2^-24.  The terms' signs differ, so
    that a result is about sum |x w| / sqrt(k), and at worst the truncations all point one way: e = 2^-23 sqrt(k) <= 2^-16 (2^-18
    in fp32 calls, whose two terms of x keep each sum's rounding apart).  Beside the definition rounded once, an element differs by
    one unit in the last place (at most 2 u) where it lies within e of a tie: sqrt(2 u e).  The mean over all results is held to e
    and its own chance: no drift to one side."""
    w = b2q.quantize_w4(normal(1, n, k) * k ** -0.5, group)
    x = X[what](normal(2, m, k)).to(dtype)
    y = b2q.linear_w4(x, w).double()
    want = x.double() @ w4_values(w).t()
    once = want.to(dtype).double()
    size = want.norm()
    if dtype == torch.float32:
        assert float((y - want).norm() / size) <= 2.0 ** -18
    else:
        assert float((y - once).norm() / size) <= (2 * UNIT[dtype] * 2.0 ** -16) ** 0.5
        assert abs(float((y - once).mean() / want.square().mean().sqrt())) <= 2.0 ** -16 + 4 * (2 * UNIT[dtype] * 2.0 ** -16) ** 0.5 / (m * n) ** 0.5


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(1, 300, 4096), (4, 64, 2000), (7, 500, 1000), (16, 300, 777)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_finite_stays_in_its_row(dtype, m, n, k, bad):
    w = b2q.quantize_w4(normal(1, n, k), 64)
    x = normal(2, m, k).to(dtype)
    want = b2q.linear_w4(x, w)
    x[m // 2, k // 3] = bad
    y = b2q.linear_w4(x, w)
    others = torch.arange(m, device="cuda") != m // 2
    assert not y[m // 2].isfinite().any() and torch.equal(y[others], want[others])
