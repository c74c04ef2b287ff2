"""Tensors of one call on different devices are refused before anything is launched (host only: tensors that say they are on a GPU)."""
import pytest
import torch

import my_own_cnn_b200 as b2q


class On:
    """A CPU tensor that says it lies on CUDA device `at`."""

    def __init__(self, t, at=0):
        self._t, self._at = t, at

    is_cuda = True

    def get_device(self):
        return self._at

    def __getattr__(self, name):
        return getattr(self._t, name)


@pytest.fixture(autouse=True)
def current(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)


def cache(*at):
    codes, params = torch.zeros(2, 1, 16, 32, dtype=torch.uint8), torch.zeros(2, 1, 16, 1, dtype=torch.int32)
    return b2q.KV4Cache(*(On(t, d) for t, d in zip((codes, params, codes, params), at)))


ONE, CURRENT = "one device", "current device"


@pytest.mark.parametrize("at", [(0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 0, 0, 0)])
def test_caches(at):
    with pytest.raises(RuntimeError, match=ONE):
        cache(*at)


@pytest.mark.parametrize("message,at", [(ONE, (1, 0, 0, 0)), (ONE, (0, 1, 0, 0)), (ONE, (0, 0, 1, 0)), (ONE, (0, 0, 0, 1)),
                                        (CURRENT, (1, 1, 1, 1))])
def test_cache_calls(message, at):
    c, k = cache(*[at[0]] * 4), torch.zeros(3, 1, 64)
    slots = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match=message):
        b2q.kv4_append(c, On(k, at[1]), On(k, at[2]), On(slots, at[3]))
    with pytest.raises(RuntimeError, match=message):
        b2q.kv4_attention(On(torch.zeros(1, 1, 1, 64), at[1]), c, On(torch.zeros(1, 2, dtype=torch.int32), at[2]),
                          On(torch.zeros(1, dtype=torch.int32), at[3]))
    if at[0] != at[3] or message == CURRENT:
        with pytest.raises(RuntimeError, match=message):
            b2q.kv4_read(c, On(slots, at[3]))


@pytest.mark.parametrize("message,at", [(ONE, (1, 0, 0, 0)), (ONE, (0, 1, 0, 0)), (ONE, (0, 0, 1, 0)), (ONE, (0, 0, 0, 1)),
                                        (CURRENT, (1, 1, 1, 1))])
def test_linear(message, at):
    w = b2q.quantize_w4(torch.zeros(8, 64), 32)
    w.codes = On(w.codes, at[0])
    with pytest.raises(RuntimeError, match=message):
        b2q.linear_w4(On(torch.zeros(2, 64), at[1]), w, On(torch.zeros(8), at[2]), out=On(torch.zeros(2, 8), at[3]))


@pytest.mark.parametrize("other", range(7))
def test_norms(other):
    t = [torch.zeros(2, 1, 64), torch.zeros(2, 1, 64), torch.zeros(64), torch.zeros(64), torch.zeros(4, 64),
         torch.zeros(2, dtype=torch.int32)]
    message = ONE if other < 6 else CURRENT
    args = [On(x, int(i == other or other == 6)) for i, x in enumerate(t)]
    with pytest.raises(RuntimeError, match=message):
        b2q.qk_norm_rope(*args)
    with pytest.raises(RuntimeError, match=message):
        b2q.qk_norm_rope_bprop(*args[:2], *args)
