"""linear_s8 where its cost model takes each of its plans: (pairs of SMs, tokens of a tile, blocks that share a reduction) and the smallest
odd sizes found that take it with as many SMs and clusters as a B200 has.  The columns that a block adds up are 2 to 128, even, in pieces
of 16 that end inside another block's share."""
import pytest
import torch

import my_own_cnn_b200 as b2q
from tests import s8_ref
from tests.lowbit_ref import within

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
PLANS = [
    (False, 16, 1, 1, 133, 1), (False, 16, 2, 343, 141, 2673), (False, 16, 4, 3, 135, 2229), (False, 16, 8, 1, 131, 4657),
    (False, 32, 1, 1239, 131, 157), (False, 32, 2, 772, 133, 4227), (False, 32, 4, 303, 137, 3483), (False, 32, 8, 199, 131, 9749),
    (False, 48, 1, 2370, 131, 115), (False, 48, 2, 1566, 137, 3963), (False, 48, 4, 752, 131, 4263), (False, 48, 8, 277, 133, 8497),
    (False, 64, 1, 3672, 135, 483), (False, 64, 2, 2196, 137, 5491), (False, 64, 4, 835, 155, 4979), (False, 64, 8, 340, 135, 13063),
    (False, 80, 1, 4751, 131, 1), (False, 80, 2, 2846, 141, 5283), (False, 80, 4, 1264, 133, 4155), (False, 80, 8, 541, 137, 14577),
    (False, 96, 1, 5958, 135, 1363), (False, 96, 2, 3119, 147, 6333), (False, 96, 4, 1281, 131, 7227), (False, 96, 8, 667, 169, 16307),
    (False, 112, 1, 7186, 131, 1), (False, 112, 2, 3621, 135, 6611), (False, 112, 4, 1789, 229, 6213),
    (False, 112, 8, 553, 277, 13953), (False, 128, 1, 5764, 257, 135), (False, 128, 2, 4592, 135, 8781),
    (False, 128, 4, 1803, 143, 8103), (False, 144, 1, 135, 15267, 151), (False, 160, 1, 6312, 259, 1),
    (False, 176, 1, 163, 15473, 139), (False, 192, 1, 8110, 265, 329), (False, 208, 1, 195, 16193, 3), (False, 224, 1, 7151, 391, 15),
    (False, 240, 1, 228, 15449, 1), (False, 256, 1, 6928, 513, 193), (True, 64, 1, 7189, 641, 41), (True, 96, 1, 5296, 1035, 203),
    (True, 128, 1, 7900, 645, 325), (True, 160, 1, 5391, 781, 929), (True, 192, 1, 5986, 399, 4755), (True, 224, 1, 8192, 263, 7425),
    (True, 256, 1, 5588, 523, 4651),
]


@pytest.mark.parametrize("pair,tokens,split,m,n,k", PLANS)
def test_every_plan(cuda_lib, pair, tokens, split, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m)
    x, w = (b2q.S8Rows(torch.randint(-128, 128, (r, -(-k // 16) * 16), generator=g, device="cuda", dtype=torch.int8),
                       torch.rand(r, generator=g, device="cuda") * 0.02 + 1e-3, k) for r in (m, n))
    for dtype, bias in zip(TYPES, (None, torch.randn(n, generator=g, device="cuda").half(), None)):
        y = b2q.linear_s8(x, w, bias, dtype=dtype)
        assert b2q.last_path() == "linear-s8"
        want, bound = s8_ref.linear(x.codes[:, :k], x.scales, w.codes[:, :k], w.scales, bias, dtype)
        within(y, want, bound)
