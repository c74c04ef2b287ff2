"""Host side of the 8-bit prompt operators without a GPU: argument blocks, 8-bit rows' checks, the C entries' refusals (which come
before anything is asked of a device)."""
import ctypes

import pytest
import torch

import my_own_cnn_b200 as b2q
from my_own_cnn_b200 import _lib
from tests.test_lowbit_host import INVALID, OK, P, UNSUPPORTED, block


@pytest.mark.parametrize("layout,size", [(_lib.CRowsS8Args, 96), (_lib.CReadS8Args, 56), (_lib.CLinearS8Args, 88), (_lib.CPromptAttentionArgs, 136)])
def test_argument_blocks_have_the_header_layout(layout, size):
    values = [(3 * i + 1) if t is not ctypes.c_float else 0.5 for i, (_, t) in enumerate(layout._fields_)]
    assert ctypes.sizeof(layout) == size
    assert _lib.packer(layout).pack(*values) == bytes(layout(*values))


def rows(**over):
    v = dict(x=P, ldx=64, w=0, residual=0, ldr=64, sum=0, lds=64, codes=P, ldc=64, scales=P, ftype=0, t=2, n=64, eps=1e-6)
    v.update(over)
    return block(_lib.CRowsS8Args, v.values())


@pytest.mark.parametrize("rc,message,kw", [
    (INVALID, b"floating type", dict(ftype=3)), (INVALID, b"negative", dict(t=-1)), (INVALID, b"negative", dict(n=-1)),
    (INVALID, b"null", dict(x=0)), (INVALID, b"null", dict(codes=0)), (INVALID, b"null", dict(scales=0)),
    (INVALID, b"stride", dict(ldc=63)), (INVALID, b"no elements", dict(n=0)), (OK, None, dict(t=0)), (OK, None, dict(t=0, n=0)),
])
def test_row_refusals(rc, message, kw):
    L = _lib.lib()
    for call in (L.b200q_quantize_s8, L.b200q_rms_norm_s8):
        assert call(rows(**kw), 0) == rc
        assert message is None or message in L.b200q_last_error()


def test_norm_and_read_refusals():
    L = _lib.lib()
    for eps in (-1e-6, float("nan"), float("inf")):
        assert L.b200q_rms_norm_s8(rows(eps=eps), 0) == INVALID and b"eps" in L.b200q_last_error()
    assert L.b200q_rms_norm_s8(rows(residual=P), 0) == INVALID and b"null" in L.b200q_last_error()
    assert L.b200q_rms_norm_s8(rows(residual=P, sum=P, lds=63), 0) == INVALID and b"stride" in L.b200q_last_error()
    assert L.b200q_quantize_s8(rows(w=P), 0) == INVALID and L.b200q_quantize_s8(rows(residual=P, sum=P), 0) == INVALID
    assert L.b200q_quantize_s8(None, 0) == INVALID

    def read(*v):
        return L.b200q_read_s8(block(_lib.CReadS8Args, v), 0)

    assert read(P, 64, P, P, 64, 5, 1, 64) == INVALID and read(P, 64, P, P, 64, 0, -1, 64) == INVALID
    assert read(P, 64, 0, P, 64, 0, 1, 64) == INVALID and b"null" in L.b200q_last_error()
    assert read(P, 64, P, P, 63, 0, 2, 64) == INVALID and b"stride" in L.b200q_last_error()
    assert L.b200q_read_s8(None, 0) == INVALID and read(0, 0, 0, 0, 0, 0, 0, 64) == OK


@pytest.mark.parametrize("rc,message,kw", [
    (INVALID, b"floating type", dict(ftype=-1)), (INVALID, b"negative", dict(m=-1)), (INVALID, b"negative", dict(k=-1)),
    (INVALID, b"no elements", dict(k=0)), (UNSUPPORTED, b"131071", dict(k=131072, ldx=131072, ldw=131072)),
    (UNSUPPORTED, b"too large", dict(n=1 << 29)), (INVALID, b"null", dict(x=0)), (INVALID, b"null", dict(w_scales=0)),
    (INVALID, b"stride", dict(ldx=48)), (INVALID, b"stride", dict(ldw=48)), (INVALID, b"stride", dict(ldy=63)),
    (INVALID, b"aligned", dict(x=P + 8)), (INVALID, b"aligned", dict(w=P + 4)), (INVALID, b"multiples", dict(ldx=72)),
    (INVALID, b"multiples", dict(ldw=72)), (OK, None, dict(m=0)), (OK, None, dict(n=0)), (OK, None, dict(m=0, k=0)),
])
def test_linear_refusals(rc, message, kw):
    v = dict(x=P, ldx=64, x_scales=P, w=P, ldw=64, w_scales=P, bias=0, y=P, ldy=64, ftype=0, m=2, n=64, k=64)
    v.update(kw)
    L = _lib.lib()
    assert L.b200q_linear_s8(block(_lib.CLinearS8Args, v.values()), 0) == rc
    assert message is None or message in L.b200q_last_error()


@pytest.mark.parametrize("rc,message,kw", [
    (INVALID, b"floating type", dict(ftype=4)), (INVALID, b"negative", dict(tq=-1)), (INVALID, b"negative", dict(b=-1)),
    (UNSUPPORTED, b"256", dict(d=257)), (UNSUPPORTED, b"256", dict(d=0)), (INVALID, b"finite", dict(scale=float("nan"))),
    (INVALID, b"divide", dict(hk=3)), (INVALID, b"divide", dict(hk=0)), (INVALID, b"null", dict(q=0)), (INVALID, b"null", dict(v=0)),
    (INVALID, b"null", dict(starts=0)), (INVALID, b"starts of the keys", dict(tk=11)), (UNSUPPORTED, b"too many", dict(tq=1 << 30, tk=1 << 30)),
    (OK, None, dict(b=0)), (OK, None, dict(tq=0, tk=0)), (OK, None, dict(hq=0)),
])
def test_prompt_attention_refusals(rc, message, kw):
    v = dict(q=P, q_ts=256, q_hs=64, k=P, k_ts=128, k_hs=64, v=P, v_ts=128, v_hs=64, starts=P, k_starts=0, out=P, lse=0, ftype=1, b=1,
             tq=10, tk=10, hq=4, hk=2, d=64, scale=0.125)
    v.update(kw)
    L = _lib.lib()
    assert L.b200q_prompt_attention(block(_lib.CPromptAttentionArgs, v.values()), 0) == rc
    assert message is None or message in L.b200q_last_error()


def test_rows_check_their_tensors():
    codes, scales = torch.zeros(4, 48, dtype=torch.int8), torch.ones(4)
    assert b2q.S8Rows(codes, scales, 33).shape == (4, 33)
    for bad in (lambda: b2q.S8Rows(codes.float(), scales, 33), lambda: b2q.S8Rows(codes, scales, 49), lambda: b2q.S8Rows(codes, scales, 0),
                lambda: b2q.S8Rows(codes[:, :32], scales, 32), lambda: b2q.S8Rows(codes, scales[:3], 33),
                lambda: b2q.S8Rows(codes, scales.half(), 33), lambda: b2q.S8Rows(codes.view(8, 24), torch.ones(8), 24)):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(RuntimeError, match="one device"):
        b2q.S8Rows(codes, scales.to("meta"), 33)
    with pytest.raises(RuntimeError, match="CUDA"):
        b2q.S8Rows(codes, scales, 33).dequantize()
    with pytest.raises(RuntimeError, match="CUDA"):
        b2q.linear_s8(b2q.S8Rows(codes, scales, 33), b2q.S8Rows(codes, scales, 33))
    for call in (lambda x: b2q.quantize_s8(x), lambda x: b2q.rms_norm_s8(x, None),
                 lambda x: b2q.prompt_attention(x, x, x, torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call(torch.ones(2, 2, 16))
