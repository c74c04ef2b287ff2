"""Linear layers with 4-bit weights and group scales, for the few rows of a decode step.

  * ``quantize_w4(w, group)`` -- a float [n, k] matrix as 4-bit codes with one bf16 scale (and zero point)
    per ``group`` weights of a row; done once, when a model is loaded;
  * ``pack_w4`` -- the same from codes, scales and zero points that exist already;
  * ``linear_w4(x, w, bias)`` -- x @ w.T + bias on tensor cores, the weights read once per 16 rows of x.
"""
from __future__ import annotations

import contextlib
import math

import torch

from . import _lib
from .conv import _raw_stream, _stream

_ARGS = _lib.packer(_lib.CLinearW4Args)
FTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
GROUPS = (32, 64, 128)


def _ftype(t: torch.Tensor, what: str) -> int:
    ft = FTYPES.get(t.dtype)
    if ft is None:
        raise TypeError(f"{what} must be float32, float16 or bfloat16, got {t.dtype}")
    if not t.is_cuda:
        raise RuntimeError("tensor arguments must be CUDA device tensors")
    return ft


def _device_tensor(t, dtype, what: str) -> None:
    if t.dtype != dtype:
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    if not t.is_cuda:
        raise RuntimeError("tensor arguments must be CUDA device tensors")


def _launch_stream(stream, *tensors) -> int:
    """The handle of `stream` (the current one when None), to which the current device belongs: all CUDA tensors of the call have
    to be there (each one's own check asks whether it is one)."""
    at = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.get_device() != at and t.is_cuda:
            if any(x is not None and x.is_cuda and x.get_device() != t.get_device() for x in tensors):
                raise RuntimeError("the tensors of a call must be on one device")
            raise RuntimeError(f"the tensors are on CUDA device {t.get_device()}, the current device is {at}")
    return _raw_stream(at) if stream is None and _raw_stream is not None else _stream(stream)


def _on(stream):
    """Context whose allocations and copies belong to `stream` (the current one when None)."""
    if stream is None:
        return contextlib.nullcontext()
    return torch.cuda.stream(stream if hasattr(stream, "cuda_stream") else torch.cuda.ExternalStream(int(stream)))


class W4Weight:
    """A [n, k] weight: codes uint8 [n, 16 * ceil(k / 32)] (low nibble = even column), scales bf16 and
    zeros uint8 (or None: 8 everywhere) [ceil(k / group), n]; w = (code - zero) * scale."""

    __slots__ = ("codes", "scales", "zeros", "n", "k", "group")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None, n: int, k: int,
                 group: int):
        if group not in GROUPS:
            raise RuntimeError(f"weight group must be 32, 64 or 128, got {group}")
        by_group = (-(-k // group), n)
        if codes.dtype != torch.uint8 or codes.shape != (n, -(-k // 32) * 16) or not codes.is_contiguous():
            raise RuntimeError(f"codes must be contiguous uint8 [{n}, {-(-k // 32) * 16}], got {codes.dtype} "
                               f"{list(codes.shape)}")
        if scales.dtype != torch.bfloat16 or scales.shape != by_group or not scales.is_contiguous():
            raise RuntimeError(f"scales must be contiguous bfloat16 {list(by_group)}, got {scales.dtype} "
                               f"{list(scales.shape)}")
        if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != by_group or not zeros.is_contiguous()):
            raise RuntimeError(f"zeros must be contiguous uint8 {list(by_group)}, got {zeros.dtype} "
                               f"{list(zeros.shape)}")
        if scales.device != codes.device or (zeros is not None and zeros.device != codes.device):
            raise RuntimeError("codes, scales and zeros must be on one device")
        self.codes, self.scales, self.zeros = codes, scales, zeros
        self.n, self.k, self.group = n, k, group

    def dequantize(self) -> torch.Tensor:
        """The fp32 [n, k] matrix that the codes stand for."""
        c = torch.stack([self.codes & 15, self.codes >> 4], -1).flatten(-2)[:, :self.k].float()
        at = torch.arange(self.k, device=c.device) // self.group
        z = 8.0 if self.zeros is None else self.zeros.float()[at].t()
        return (c - z) * self.scales.float()[at].t()


def pack_w4(codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None, group: int = 64) -> W4Weight:
    """codes: [n, k] integers 0..15; scales and zeros: [n, ceil(k / group)]."""
    n, k = codes.shape
    full = torch.zeros((n, -(-k // 32) * 32), dtype=torch.uint8, device=codes.device)
    full[:, :k] = codes.to(torch.uint8)
    packed = (full[:, 0::2] | (full[:, 1::2] << 4)).contiguous()
    return W4Weight(packed, scales.t().to(torch.bfloat16).contiguous(),
                    None if zeros is None else zeros.t().to(torch.uint8).contiguous(), n, k, group)


def quantize_w4(w: torch.Tensor, group: int = 64, symmetric: bool = False) -> W4Weight:
    """Rounds a finite float [n, k] matrix to 4 bits.  Asymmetric: each group's range, widened to hold 0,
    over codes 0..15; symmetric: codes 1..15 around 8.  Codes are chosen for the scale as stored (bf16)."""
    if group not in GROUPS:
        raise RuntimeError(f"weight group must be 32, 64 or 128, got {group}")
    n, k = w.shape
    g = torch.zeros((n, -(-k // group) * group), dtype=torch.float32, device=w.device)
    g[:, :k] = w
    g = g.unflatten(1, (-1, group))
    lo, hi = g.amin(-1).clamp(max=0), g.amax(-1).clamp(min=0)
    s = torch.maximum(hi, -lo) / 7 if symmetric else (hi - lo) / 15
    s = s.bfloat16().float()
    s = torch.where(s < torch.finfo(torch.float32).tiny, torch.zeros_like(s), s)
    inv = torch.where(s > 0, 1 / s, torch.zeros_like(s))
    z = torch.full_like(s, 8) if symmetric else (-lo * inv).round().clamp(0, 15)
    codes = ((g * inv[..., None]).round() + z[..., None]).clamp(1 if symmetric else 0, 15)
    return pack_w4(codes.flatten(1)[:, :k], s, None if symmetric else z, group)


def linear_w4(x: torch.Tensor, w: W4Weight, bias: torch.Tensor | None = None, out: torch.Tensor | None = None,
              stream=None) -> torch.Tensor:
    """x [..., k] (fp32, fp16 or bf16; rows may be strided) -> [..., n] of the same type; fp32 sums.
    bias: [n] of x's type; out shares no memory with x."""
    ft = FTYPES.get(x.dtype)
    if ft is None or not x.is_cuda:
        _ftype(x, "x")
    n, k, shape = w.n, w.k, x.shape
    if not shape or shape[-1] != k:
        raise RuntimeError(f"x has {shape[-1] if shape else 0} columns, the weight {k}")
    if not w.codes.is_cuda:
        raise RuntimeError("tensor arguments must be CUDA device tensors")
    if bias is not None:
        _device_tensor(bias, x.dtype, "bias")
        if bias.shape != (n,) or not bias.is_contiguous():
            raise RuntimeError(f"bias must be contiguous [{n}]")
    if stream is not None:
        with _on(stream):
            return _linear(x, w, bias, out, ft, n, k, stream)
    return _linear(x, w, bias, out, ft, n, k, None)


def _linear(x, w, bias, out, ft, n, k, stream):
    handle = _launch_stream(stream, x, w.codes, bias, out)
    rows = x if x.dim() == 2 else x.reshape(math.prod(x.shape[:-1]), k)
    ldx, step = rows.stride()
    m = rows.shape[0]
    if step != 1 or (ldx < k and m > 1):  # columns apart, or rows that overlap (a broadcast)
        rows = rows.contiguous()
        ldx = k
    y, ldy = out, n
    if out is None:
        out = y = x.new_empty((m, n) if rows is x else x.shape[:-1] + (n,))
    else:
        if out.dtype != x.dtype or out.shape != x.shape[:-1] + (n,) or not out.is_cuda:
            raise RuntimeError(f"out must be a {x.dtype} {list(x.shape[:-1] + (n,))} CUDA tensor")
        if out.dim() == 2 and (out.stride(1) == 1 or n == 1):
            ldy = out.stride(0)
        elif not out.is_contiguous():
            raise RuntimeError("out must be contiguous, or 2-D with contiguous rows")
    zeros = w.zeros
    _lib.check(_lib.lib().b200q_linear_w4(_ARGS.pack(rows.data_ptr(), ldx, w.codes.data_ptr(), w.scales.data_ptr(),
                                                     0 if zeros is None else zeros.data_ptr(),
                                                     0 if bias is None else bias.data_ptr(), y.data_ptr(), ldy, ft, m,
                                                     n, k, w.group), handle))
    return out
