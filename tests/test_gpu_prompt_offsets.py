"""8-bit prompt operators on tensors of more than 2^31 elements: the last rows are those of a call on these rows alone."""
import pytest
import torch

import my_own_cnn_b200 as b2q

pytestmark = pytest.mark.gpu
TAIL = 1000


def random(*shape):
    """bf16 from a few random rows: quick to make."""
    base = torch.randn(1009, *shape[1:], generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").bfloat16()
    return base.repeat(-(-shape[0] // 1009), *[1] * (len(shape) - 1))[:shape[0]]


@pytest.mark.parametrize("n", [1024, 1029])
def test_rows(cuda_lib, n):
    x = random(2200000, n)
    assert x.numel() > 2 ** 31
    w = random(n, 1)[:, 0].contiguous()
    rows = b2q.rms_norm_s8(x, w)
    some = b2q.rms_norm_s8(x[-TAIL:], w)
    assert torch.equal(rows.codes[-TAIL:, :n], some.codes[:, :n]) and torch.equal(rows.scales[-TAIL:], some.scales)
    y = rows.dequantize(torch.bfloat16)
    assert torch.equal(y[-TAIL:], some.dequantize(torch.bfloat16)) and torch.equal(y[:TAIL], b2q.rms_norm_s8(x[:TAIL], w).dequantize(torch.bfloat16))


def test_linear(cuda_lib):
    x, w = b2q.quantize_s8(random(70000, 144)), b2q.quantize_s8(random(32000, 144))
    y = b2q.linear_s8(x, w)
    assert y.numel() > 2 ** 31
    some = b2q.S8Rows(x.codes[-TAIL:], x.scales[-TAIL:], 144)
    assert torch.equal(y[-TAIL:], b2q.linear_s8(some, w))


@pytest.mark.parametrize("d,off", [(128, 0), (128, 1)])
def test_attention(cuda_lib, d, off):
    """40000 prompts of 7 tokens, 64 / 16 heads: on tcgen05 and, not aligned, on mma.sync."""
    t = 280000
    x = random(t, 96, d + off)[..., off:]
    starts = torch.arange(0, t + 1, 7, dtype=torch.int32, device="cuda")
    q, k, v = x[:, :64], x[:, 64:80], x[:, 80:]
    out, lse = b2q.prompt_attention(q, k, v, starts, return_lse=True)
    assert out.numel() > 2 ** 31 and b2q.last_path() == ("mma-prompt-attention" if off else "tcgen05-prompt-attention")
    cut = t - 994  # whole prompts
    some, some_lse = b2q.prompt_attention(q[cut:], k[cut:], v[cut:], starts[:143], return_lse=True)
    assert torch.equal(out[cut:], some) and torch.equal(lse[cut:], some_lse)
    b2q.device_error()
