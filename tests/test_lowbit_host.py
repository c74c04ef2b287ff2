"""Host side of the decoder operators without a GPU: weight packing, and the C entries' refusals (which come
before anything is asked of a device)."""
import ctypes

import pytest
import torch

import my_own_cnn_b200 as b2q
from my_own_cnn_b200 import _lib

OK, INVALID, UNSUPPORTED = 0, 1, 2


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("symmetric", [False, True])
def test_quantized_weights_are_within_a_step(group, symmetric):
    w = torch.randn(9, 131, generator=torch.Generator().manual_seed(group))
    w[2] = 0
    w[3] = w[3].abs()
    q = b2q.quantize_w4(w, group, symmetric)
    assert q.codes.shape == (9, 80) and q.scales.shape == (-(-131 // group), 9) and (q.zeros is None) == symmetric
    step = q.scales.float()[torch.arange(131) // group].t()
    # half a step, and the scale's rounding (2^-9) over at most 15 steps
    assert ((q.dequantize() - w).abs() <= step * (0.5 + 15 / 512) + 1e-30).all()
    assert (q.dequantize()[2] == 0).all()


def test_packed_weights_come_back():
    g = torch.Generator().manual_seed(0)
    codes = torch.randint(0, 16, (5, 77), generator=g)
    zeros = torch.randint(0, 16, (5, 2), generator=g)
    scales = torch.rand(5, 2, generator=g).bfloat16()
    w = b2q.pack_w4(codes, scales, zeros, 64)
    at = torch.arange(77) // 64
    assert torch.equal(w.dequantize(), (codes - zeros[:, at]).float() * scales.float()[:, at])
    assert int(w.codes[1, 3]) == int(codes[1, 6]) + 16 * int(codes[1, 7])


def test_rotation_table():
    t = b2q.rope_table(4, 6, base=100.0, device="cpu")
    assert t.shape == (4, 6) and torch.equal(t[0], torch.tensor([1.0, 1, 1, 0, 0, 0]))
    want = torch.tensor(3 * 100.0 ** (-2 / 6), dtype=torch.float64)
    assert abs(t[3, 1] - want.cos()) < 1e-7 and abs(t[3, 4] - want.sin()) < 1e-7


def block(layout, values):
    return bytes(layout(*values))


def cache(**over):
    v = dict(k_codes=4096, k_params=4096, v_codes=4096, v_params=4096, pages=1, heads=2, page_size=16, d=64, group=32)
    v.update(over)
    return block(_lib.CKV4Cache, v.values())


P = 1 << 20  # an address that is never used


@pytest.mark.parametrize("layout,size", [(_lib.CLinearW4Args, 88), (_lib.CQKNormArgs, 200), (_lib.CKV4AttentionArgs, 96),
                                         (_lib.CKV4Cache, 56)])
def test_argument_blocks_have_the_header_layout(layout, size):
    """Sizes as a C compiler gives them, and the packed bytes equal to the structure's."""
    values = [(3 * i + 1) if t is not ctypes.c_float else 0.5 for i, (_, t) in enumerate(layout._fields_)]
    assert ctypes.sizeof(layout) == size
    assert _lib.packer(layout).pack(*values) == bytes(layout(*values))


@pytest.mark.parametrize("rc,message,args", [
    (INVALID, b"floating type", (P, 64, P, P, 0, 0, P, 64, 3, 1, 64, 64, 32, 0)),
    (INVALID, b"negative", (P, 64, P, P, 0, 0, P, 64, 0, -1, 64, 64, 32, 0)),
    (INVALID, b"group", (P, 64, P, P, 0, 0, P, 64, 0, 1, 64, 64, 16, 0)),
    (INVALID, b"null", (0, 64, P, P, 0, 0, P, 64, 0, 1, 64, 64, 32, 0)),
    (INVALID, b"null", (P, 64, P, 0, 0, 0, P, 64, 0, 1, 64, 64, 32, 0)),
    (INVALID, b"stride", (P, 63, P, P, 0, 0, P, 64, 0, 2, 64, 64, 32, 0)),
    (INVALID, b"aligned", (P, 64, P + 8, P, 0, 0, P, 64, 0, 1, 64, 64, 32, 0)),
    (UNSUPPORTED, b"too large", (P, 64, P, P, 0, 0, P, 64, 0, 1, 1 << 29, 64, 32, 0)),
    (OK, None, (0, 64, 0, 0, 0, 0, 0, 64, 0, 0, 64, 64, 32, 0)),
])
def test_linear_refusals(rc, message, args):
    L = _lib.lib()
    assert L.b200q_linear_w4(block(_lib.CLinearW4Args, args[:-1]), args[-1]) == rc
    assert message is None or message in L.b200q_last_error()


def norm_args(ft=0, q=P, table=P, positions=8, pos=P, t=1, hq=2, hk=1, d=64, rot=64, grad=P):
    return block(_lib.CQKNormArgs, (q, P, 0, 0, table, pos, P, P, grad, grad, P, P, *[0] * 8, positions, ft, t, hq, hk, d, rot,
                                    0, 1e-6))


@pytest.mark.parametrize("rc,message,kw", [
    (INVALID, b"floating type", dict(ft=-1)), (INVALID, b"head dimensions", dict(d=0)),
    (INVALID, b"even", dict(rot=63)), (INVALID, b"even", dict(rot=66)), (INVALID, b"null", dict(q=0)),
    (INVALID, b"table", dict(pos=0)), (INVALID, b"table", dict(positions=0)),
    (UNSUPPORTED, b"1024", dict(d=1026)), (OK, None, dict(t=0)),
])
def test_norm_refusals(rc, message, kw):
    L = _lib.lib()
    assert L.b200q_qk_norm_rope(norm_args(**kw), 0) == rc
    assert message is None or message in L.b200q_last_error()
    if rc != OK:
        assert L.b200q_qk_norm_rope_bprop(norm_args(**kw), 0) == rc


@pytest.mark.parametrize("rc,message,kw", [
    (UNSUPPORTED, b"64, 128 or 256", dict(d=96)), (UNSUPPORTED, b"32 or 64", dict(group=128)),
    (INVALID, b"cache shape", dict(heads=0)), (INVALID, b"null cache", dict(v_params=0)),
    (INVALID, b"aligned", dict(k_codes=4104)),
])
def test_cache_refusals(rc, message, kw):
    L = _lib.lib()
    for call in (lambda c: L.b200q_kv4_append(c, P, 0, 0, P, 0, 0, P, 0, 1, 0), lambda c: L.b200q_kv4_read(c, P, P, P, 0, 1, 0),
                 lambda c: L.b200q_kv4_attention(c, attention_args(), 0)):
        assert call(cache(**kw)) == rc and message in L.b200q_last_error()


def attention_args(hq=2, b=1, tq=1, lens=P, table=P, max_pages=1, ft=0):
    return block(_lib.CKV4AttentionArgs, (P, 0, 0, 0, table, 1, lens, P, 0, ft, b, tq, hq, max_pages, 1.0))


def test_attention_refusals():
    L = _lib.lib()

    def call(**kw):
        return L.b200q_kv4_attention(cache(), attention_args(**kw), 0)

    assert call(hq=3) == INVALID and b"divide" in L.b200q_last_error()
    assert call(lens=0) == INVALID and call(table=0) == INVALID and call(ft=7) == INVALID and call(tq=-1) == INVALID
    assert call(max_pages=1 << 28) == UNSUPPORTED
    assert call(b=1 << 20, tq=1 << 16, hq=1 << 16) == UNSUPPORTED and b"too large" in L.b200q_last_error()
    assert call(b=0) == OK and call(tq=0) == OK and call(hq=0) == OK
    assert L.b200q_kv4_append(cache(), P, 0, 0, P, 0, 0, 0, 0, 1, 0) == INVALID
    assert L.b200q_kv4_append(cache(), P, 0, 0, P, 0, 0, P, 0, -1, 0) == INVALID
    assert L.b200q_kv4_append(cache(), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0) == OK


def test_weights_on_one_device():
    codes, scales = torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(1, 4, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="one device"):
        b2q.W4Weight(codes, scales.to("meta"), None, 4, 32, 32)
    with pytest.raises(RuntimeError, match="one device"):
        b2q.W4Weight(codes, scales, torch.zeros(1, 4, dtype=torch.uint8, device="meta"), 4, 32, 32)
