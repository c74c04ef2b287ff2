"""The 8-bit attention block where there is nothing to do, and where its arguments do not go together."""
import pytest
import torch

import my_own_cnn_b200 as b2q
from my_own_cnn_b200.decoder import random_block_s8

pytestmark = pytest.mark.gpu
HIDDEN, H, HK, D, PAGE = 320, 6, 2, 64, 16


def ints(*shape, dtype=torch.int32):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_no_tokens(cuda_lib, dtype):
    block = random_block_s8(HIDDEN, H, HK, D, dtype, positions=16)
    cache = b2q.KV4Cache.empty(4, HK, PAGE, D, 32)
    x, residual = torch.empty(0, HIDDEN, dtype=dtype, device="cuda"), torch.empty(0, HIDDEN, dtype=dtype, device="cuda")
    for starts in (ints(1), ints(4)):  # no prompts, three empty ones
        y, total = block.prompt(x, residual, ints(0), starts, cache, ints(0, dtype=torch.int64))
        assert y.shape == (0, HIDDEN) and total is residual
        assert block.prompt(x, None, ints(0), starts)[0].shape == (0, HIDDEN)
    y, total = block.forward(x, residual, cache, ints(0), ints(0, dtype=torch.int64), ints(0, 2), ints(0))
    assert y.shape == (0, HIDDEN) and total is residual
    b2q.device_error()


def test_a_cache_and_slots_go_together(cuda_lib):
    block = random_block_s8(HIDDEN, H, HK, D, torch.bfloat16, positions=16)
    cache = b2q.KV4Cache.empty(4, HK, PAGE, D, 32)
    x = torch.zeros(3, HIDDEN, dtype=torch.bfloat16, device="cuda")
    starts = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="slots"):
        block.prompt(x, None, ints(3), starts, cache)
    with pytest.raises(RuntimeError, match="slots"):
        block.prompt(x, None, ints(3), starts, slots=ints(3, dtype=torch.int64))
    with pytest.raises(RuntimeError):  # three tokens of two sequences
        block.forward(x, None, cache, ints(3), ints(3, dtype=torch.int64), ints(2, 2), ints(2))
