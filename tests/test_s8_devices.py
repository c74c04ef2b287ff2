"""Tensors of one call of the 8-bit prompt operators on different devices are refused before anything is launched (host only: tensors
that say they are on a GPU)."""
import pytest
import torch

import my_own_cnn_b200 as b2q
from tests.test_lowbit_devices import CURRENT, ONE, On, current  # noqa: F401 (a fixture)


def rows(*shape, at=(0, 0)):
    r = b2q.S8Rows(torch.zeros(*shape[:-1], 64, dtype=torch.int8), torch.ones(shape[:-1]), shape[-1])
    r.codes, r.scales = On(r.codes, at[0]), On(r.scales, at[1])
    return r


@pytest.mark.parametrize("message,at", [(ONE, (1, 0, 0, 0)), (ONE, (0, 1, 0, 0)), (ONE, (0, 0, 1, 0)), (ONE, (0, 0, 0, 1)),
                                        (CURRENT, (1, 1, 1, 1))])
def test_norm_and_linear(message, at):
    x, w, b = torch.zeros(2, 64), torch.zeros(64), torch.zeros(8)
    with pytest.raises(RuntimeError, match=message):
        b2q.rms_norm_s8(On(x, at[0]), On(w, at[1]), On(x, at[2]), out=rows(2, 64, at=(at[3],) * 2))
    with pytest.raises(RuntimeError, match=message):
        b2q.rms_norm_s8(On(x, at[0]), On(w, at[1]), On(x, at[2]), residual_out=On(x, at[3]), out=rows(2, 64, at=(at[0],) * 2))
    with pytest.raises(RuntimeError, match=message):
        b2q.linear_s8(rows(2, 64, at=(at[0],) * 2), rows(8, 64, at=(at[1],) * 2), On(b, at[2]), dtype=torch.float32,
                      out=On(torch.zeros(2, 8), at[3]))


@pytest.mark.parametrize("message,at", [(ONE, (1, 0)), (ONE, (0, 1)), (CURRENT, (1, 1))])
def test_quantize_and_read(message, at):
    with pytest.raises(RuntimeError, match=message):
        b2q.quantize_s8(On(torch.zeros(2, 64), at[0]), out=rows(2, 64, at=(at[1],) * 2))
    if message == CURRENT:
        with pytest.raises(RuntimeError, match=message):
            rows(2, 64, at=at).dequantize()


@pytest.mark.parametrize("other", range(7))
def test_attention(other):
    t = [torch.zeros(3, 2, 16)] * 3 + [torch.zeros(2, dtype=torch.int32)] * 2 + [torch.zeros(3, 2, 16)]
    q, k, v, s, ks, out = (On(x, int(i == other or other == 6)) for i, x in enumerate(t))
    with pytest.raises(RuntimeError, match=ONE if other < 6 else CURRENT):
        b2q.prompt_attention(q, k, v, s, ks, out=out)
