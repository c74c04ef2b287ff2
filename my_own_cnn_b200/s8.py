"""8-bit rows with one scale each, and the linear layers over them: activations with a scale for each token, weights
with one for each channel.

  * ``quantize_s8(x)`` -- float rows as 8-bit rows (activations, or a weight once when a model is loaded);
  * ``rms_norm_s8(x, weight, residual)`` -- the residual's addition, RMS norm and rounding in one pass;
  * ``linear_s8(x, w, bias)`` -- x @ w.T + bias on int8 tensor cores, sums exact, for one token or a long prompt.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .w4 import FTYPES, _device_tensor, _ftype, _launch_stream, _on

_ROWS = _lib.packer(_lib.CRowsS8Args)
_READ = _lib.packer(_lib.CReadS8Args)
_LINEAR = _lib.packer(_lib.CLinearS8Args)


class S8Rows:
    """Rows of k values: codes int8 [..., pitch] (pitch >= k a multiple of 16; what lies past k is not used) and
    scales fp32 [...]; value = code * scale.  A NaN scale makes its row NaN."""

    __slots__ = ("codes", "scales", "k", "_pitch")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, k: int):
        shape = codes.shape
        if codes.dtype != torch.int8 or not shape or shape[-1] < k or shape[-1] % 16 or k < 1 or not codes.is_contiguous():
            raise RuntimeError(f"codes must be contiguous int8 [..., pitch] with a pitch of at least {k} that is a multiple "
                               f"of 16, got {codes.dtype} {list(shape)}")
        if codes.data_ptr() % 16:
            raise RuntimeError("codes must be 16-byte aligned")
        if scales.dtype != torch.float32 or scales.shape != shape[:-1] or not scales.is_contiguous():
            raise RuntimeError(f"scales must be contiguous float32 {list(shape[:-1])}, got {scales.dtype} {list(scales.shape)}")
        if scales.device != codes.device:
            raise RuntimeError("codes and scales must be on one device")
        self.codes, self.scales, self.k, self._pitch = codes, scales, k, shape[-1]

    @staticmethod
    def empty(shape, device="cuda") -> "S8Rows":
        """Uninitialised rows for values of `shape`."""
        lead, k = tuple(shape[:-1]), shape[-1]
        return S8Rows(torch.empty(lead + (-(-k // 16) * 16,), dtype=torch.int8, device=device),
                      torch.empty(lead, dtype=torch.float32, device=device), k)

    @staticmethod
    def _like(x: torch.Tensor) -> "S8Rows":
        """Uninitialised rows for the values of x, beside it: nothing to check."""
        shape = x.shape
        lead, k = shape[:-1], shape[-1]
        r = S8Rows.__new__(S8Rows)
        r.k, r._pitch = k, -(-k // 16) * 16
        if r._pitch == k and x.is_contiguous():
            r.codes = torch.empty_like(x, dtype=torch.int8)
        else:
            r.codes = x.new_empty(lead + (r._pitch,), dtype=torch.int8)
        r.scales = x.new_empty(lead, dtype=torch.float32)
        return r

    @property
    def shape(self) -> torch.Size:
        return self.scales.shape + (self.k,)

    def dequantize(self, dtype: torch.dtype = torch.float32, stream=None) -> torch.Tensor:
        """The values [..., k], rounded once to `dtype`."""
        ft = FTYPES.get(dtype)
        if ft is None:
            raise TypeError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
        if not self.codes.is_cuda:
            raise RuntimeError("tensor arguments must be CUDA device tensors")
        if stream is not None:
            with _on(stream):
                return self._read(dtype, ft, stream)
        return self._read(dtype, ft, None)

    def _read(self, dtype, ft, stream):
        handle = _launch_stream(stream, self.codes)
        scales = self.scales
        y = scales.new_empty(scales.shape + (self.k,), dtype=dtype)
        _lib.check(_lib.lib().b200q_read_s8(_READ.pack(self.codes.data_ptr(), self._pitch, scales.data_ptr(), y.data_ptr(),
                                                       self.k, ft, scales.numel(), self.k), handle))
        return y


def _float_rows(x, n):
    """x [..., n] as (tensor that is read, its row stride)."""
    if x.dim() == 2:
        ld, step = x.stride()
        if step == 1 or n == 1:
            return x, ld
    if x.is_contiguous():
        return x, n
    rows = x.reshape(-1, n)
    if n > 1 and rows.stride(1) != 1:
        rows = rows.contiguous()
    return rows, rows.stride(0)


def _own_rows(x, n, what):
    """The row stride of a tensor that is written."""
    if x.dim() == 2 and (x.stride(1) == 1 or n == 1) and (x.stride(0) >= n or x.shape[0] < 2):
        return x.stride(0)
    if not x.is_contiguous():
        raise RuntimeError(f"{what} must be contiguous, or 2-D with contiguous rows that do not overlap")
    return n


def _out_rows(out, shape, like):
    if out is None:
        return S8Rows._like(like)
    if out.shape != shape or not out.codes.is_cuda:
        raise RuntimeError(f"out must be 8-bit rows of {list(shape)} on the device, got {list(out.shape)}")
    return out


def _check_like(t, x, shape, what):
    if t.dtype != x.dtype or not t.is_cuda:
        _device_tensor(t, x.dtype, what)
    if t.shape != shape:
        raise RuntimeError(f"{what} must be {list(shape)}, got {list(t.shape)}")


def quantize_s8(x: torch.Tensor, out: S8Rows | None = None, stream=None) -> S8Rows:
    """x [..., k] (fp32, fp16 or bf16; rows may be strided) as 8-bit rows: code = rint(x * fl(127 * fl(1 / max|x|))),
    scale = max|x| / 127.  A row with a NaN or an infinity gets the scale NaN, one with nothing above 2^-119 zeros."""
    ft = FTYPES.get(x.dtype)
    if ft is None or not x.is_cuda:
        _ftype(x, "x")
    if not x.dim() or not x.shape[-1]:
        raise RuntimeError(f"x must be [..., k] with k of at least 1, got {list(x.shape)}")
    if stream is not None:
        with _on(stream):
            return _quantize(x, out, ft, stream)
    return _quantize(x, out, ft, None)


def _quantize(x, out, ft, stream):
    n = x.shape[-1]
    out = _out_rows(out, x.shape, x)
    handle = _launch_stream(stream, x, out.codes)
    rows, ldx = _float_rows(x, n)
    scales = out.scales
    _lib.check(_lib.lib().b200q_quantize_s8(_ROWS.pack(rows.data_ptr(), ldx, 0, 0, 0, 0, 0, out.codes.data_ptr(), out._pitch,
                                                       scales.data_ptr(), ft, scales.numel(), n, 0.0), handle))
    return out


def rms_norm_s8(x: torch.Tensor, weight: torch.Tensor | None, residual: torch.Tensor | None = None,
                residual_out: torch.Tensor | None = None, eps: float = 1e-6, out: S8Rows | None = None, stream=None):
    """8-bit rows of h * (mean(h^2) + eps)^-1/2 * weight with h = x + residual, rounded to x's type.

    x [..., n] (fp32, fp16 or bf16; rows may be strided), weight [n] or None, residual like x.  h is written to
    residual_out, which may be x; to the residual itself when that is None.  Returns the rows, with a residual
    (rows, h).  A row with a NaN or an infinity gets the scale NaN; one with nothing above 2^-119 in size after the weight is zeros, also where
    eps is 0."""
    ft = FTYPES.get(x.dtype)
    if ft is None or not x.is_cuda:
        _ftype(x, "x")
    shape = x.shape
    if not shape or not shape[-1]:
        raise RuntimeError(f"x must be [..., n] with n of at least 1, got {list(shape)}")
    if weight is not None:
        if weight.dtype != x.dtype or not weight.is_cuda:
            _device_tensor(weight, x.dtype, "weight")
        if weight.dim() != 1 or weight.shape[0] != shape[-1] or not weight.is_contiguous():
            raise RuntimeError(f"weight must be contiguous [{shape[-1]}]")
    if residual is None:
        if residual_out is not None:
            raise RuntimeError("residual_out without a residual")
    else:
        _check_like(residual, x, shape, "residual")
        if residual_out is not None:
            _check_like(residual_out, x, shape, "residual_out")
    if stream is not None:
        with _on(stream):
            return _norm(x, weight, residual, residual_out, eps, out, ft, shape, stream)
    return _norm(x, weight, residual, residual_out, eps, out, ft, shape, None)


def _norm(x, weight, residual, residual_out, eps, out, ft, shape, stream):
    n = shape[-1]
    out = _out_rows(out, shape, x)
    handle = _launch_stream(stream, x, weight, residual, residual_out, out.codes)
    rows, ldx = _float_rows(x, n)
    scales = out.scales
    if residual is None:
        _lib.check(_lib.lib().b200q_rms_norm_s8(_ROWS.pack(rows.data_ptr(), ldx, 0 if weight is None else weight.data_ptr(), 0, 0,
                                                           0, 0, out.codes.data_ptr(), out._pitch, scales.data_ptr(), ft,
                                                           scales.numel(), n, eps), handle))
        return out
    total = residual if residual_out is None else residual_out
    lds = _own_rows(total, n, "residual" if residual_out is None else "residual_out")
    added, ldr = (total, lds) if residual is total else _float_rows(residual, n)
    _lib.check(_lib.lib().b200q_rms_norm_s8(_ROWS.pack(rows.data_ptr(), ldx, 0 if weight is None else weight.data_ptr(),
                                                       added.data_ptr(), ldr, total.data_ptr(), lds, out.codes.data_ptr(),
                                                       out._pitch, scales.data_ptr(), ft, scales.numel(), n, eps), handle))
    return out, total


def linear_s8(x: S8Rows, w: S8Rows, bias: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16,
              out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """x [..., k] times the weight w [n, k], both 8-bit rows -> [..., n] of `dtype` (fp32, fp16 or bf16); sums
    exact, k up to 131071.  bias: [n] of `dtype`; out shares no memory with the other tensors."""
    ft = FTYPES.get(dtype)
    if ft is None:
        raise TypeError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    if w.scales.dim() != 1 or x.k != w.k:
        raise RuntimeError(f"x has rows of {x.k}, the weight is {list(w.shape)}")
    if not x.codes.is_cuda or not w.codes.is_cuda:
        raise RuntimeError("tensor arguments must be CUDA device tensors")
    n = w.scales.shape[0]
    if bias is not None:
        _device_tensor(bias, dtype, "bias")
        if bias.shape != (n,) or not bias.is_contiguous():
            raise RuntimeError(f"bias must be contiguous [{n}]")
    if stream is not None:
        with _on(stream):
            return _linear(x, w, bias, dtype, out, ft, n, stream)
    return _linear(x, w, bias, dtype, out, ft, n, None)


def _linear(x, w, bias, dtype, out, ft, n, stream):
    handle = _launch_stream(stream, x.codes, w.codes, bias, out)
    scales = x.scales
    shape = scales.shape + (n,)
    ldy = n
    if out is None:
        out = scales.new_empty(shape, dtype=dtype)
    else:
        if out.dtype != dtype or out.shape != shape or not out.is_cuda:
            raise RuntimeError(f"out must be a {dtype} {list(shape)} CUDA tensor")
        ldy = _own_rows(out, n, "out")
    _lib.check(_lib.lib().b200q_linear_s8(_LINEAR.pack(x.codes.data_ptr(), x._pitch, scales.data_ptr(), w.codes.data_ptr(),
                                                       w._pitch, w.scales.data_ptr(), 0 if bias is None else bias.data_ptr(),
                                                       out.data_ptr(), ldy, ft, math.prod(scales.shape), n, x.k), handle))
    return out
