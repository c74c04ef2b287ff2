"""Prompts whose sequences have earlier tokens in the 4-bit cache: all tokens read back, one sequence after another, as the keys and
values of prompt_attention."""
import pytest
import torch

import my_own_cnn_b200 as b2q
from tests import s8_ref
from tests.lowbit_ref import within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_next_prompts_over_the_cache(cuda_lib, dtype):
    page, hq, hk, d = 16, 8, 2, 64
    before, new = [37, 0, 100], [20, 33, 1]
    per = 16
    cache = b2q.KV4Cache.empty(3 * per, hk, page, d, 32)
    g = torch.Generator(device="cuda").manual_seed(0)
    table = torch.randperm(3 * per, generator=g, device="cuda").view(3, per)

    def slots_of(first, count):
        """Of tokens first[i] .. first[i] + count[i] of each sequence, one sequence after another."""
        at = [(i, p) for i in range(3) for p in range(first[i], first[i] + count[i])]
        seq, pos = torch.tensor(at, device="cuda").t()
        return table[seq, pos // page] * page + pos % page

    def tokens(n, heads):
        return torch.randn(n, heads, d, generator=g, device="cuda").to(dtype)

    b2q.kv4_append(cache, tokens(sum(before), hk), tokens(sum(before), hk), slots_of([0] * 3, before))
    q, k, v = tokens(sum(new), hq), tokens(sum(new), hk), tokens(sum(new), hk)
    b2q.kv4_append(cache, k, v, slots_of(before, new))
    total = [a + b for a, b in zip(before, new)]
    starts, key_starts = (torch.tensor([0] + n, device="cuda").cumsum(0).int() for n in (new, total))
    keys, values = b2q.kv4_read(cache, slots_of([0] * 3, total), dtype)
    out, lse = b2q.prompt_attention(q, keys, values, starts, key_starts, return_lse=True)
    b2q.device_error()
    want, want_lse, ob, lb = s8_ref.attention(q, keys, values, starts, key_starts, d ** -0.5, dtype)
    within(out, want, ob)
    within(lse, want_lse, lb)
    # the last tokens answered by the cache's own attention: the same keys and values, not rounded to dtype (2^-11 or 2^-8 of scores and values)
    last = starts[1:].long() - 1
    lens = torch.tensor(total, dtype=torch.int32, device="cuda")
    one = b2q.kv4_attention(q[last][:, None], cache, table.int(), lens)[:, 0]
    unit = {torch.float32: 2.0 ** -16, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    big = d ** -0.5 * (q[last].float().abs().unflatten(1, (hk, -1)) * keys.float().abs().amax(0)[:, None]).sum(-1).max()
    assert (one.float() - out[last].float()).abs().max() < 2 * float(values.float().abs().max()) * (3 * unit + unit * float(big))
