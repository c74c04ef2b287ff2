"""Numbers at the ends of their ranges that the 8-bit prompt operators refuse, without a GPU."""
import pytest

from my_own_cnn_b200 import _lib
from tests.test_lowbit_host import INVALID, P, block


@pytest.mark.parametrize("scale", [2.4e38, -2.4e38, 3.4e38, float("inf")])
def test_scales_that_pass_fp32_with_the_base(scale):
    """Exponents are of base 2: a score is multiplied by scale * log2(e), which passes fp32 from 2.36e38 on."""
    args = dict(q=P, q_ts=256, q_hs=64, k=P, k_ts=128, k_hs=64, v=P, v_ts=128, v_hs=64, starts=P, k_starts=0, out=P, lse=0, ftype=1, b=1,
                tq=10, tk=10, hq=4, hk=2, d=64, scale=scale)
    L = _lib.lib()
    assert L.b200q_prompt_attention(block(_lib.CPromptAttentionArgs, args.values()), 0) == INVALID
    assert b"scale" in L.b200q_last_error()
