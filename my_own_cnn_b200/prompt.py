"""Causal attention over whole prompts, packed one after another: queries, keys and values as they leave the projection, before
(or beside) their way into a cache."""
from __future__ import annotations

import math

import torch

from . import _lib
from .w4 import FTYPES, _device_tensor, _ftype, _launch_stream, _on

_ARGS = _lib.packer(_lib.CPromptAttentionArgs)


def _check_starts(starts, what, b=None):
    _device_tensor(starts, torch.int32, what)
    if starts.dim() != 1 or not starts.is_contiguous() or not starts.shape[0] or (b is not None and starts.shape[0] != b + 1):
        raise RuntimeError(f"{what} must be contiguous [{'sequences + 1' if b is None else b + 1}], got {list(starts.shape)}")


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor,
                     k_starts: torch.Tensor | None = None, scale: float | None = None, out: torch.Tensor | None = None,
                     return_lse: bool = False, stream=None):
    """q [tq, hq, d], k and v [tk, hk, d] (fp32, fp16 or bf16; views with contiguous channels will do, d up to 256).

    starts int32 [sequences + 1] on the device: sequence i has the rows starts[i] .. starts[i + 1]; k_starts the same for its
    keys, where a sequence has more (an earlier part) or fewer of them than queries.  A sequence's last query is in line with its
    last key: query j of lq sees the first lk - lq + j + 1 keys; where that is none the output is 0 (lse -inf).  Query head
    h reads head h // (hq / hk).  Rows outside every sequence are left as they are in `out`.  A sequence whose
    starts decrease or pass the tensors is left out and reported by device_error().  scale: 1 / sqrt(d) when None; its product
    with log2(e) has to be finite in fp32.
    Returns out [tq, hq, d], and lse fp32 [tq, hq] (log of the sum of exp(scale * q.k)) when return_lse.  out shares no memory
    with the other tensors; starts stay as they are until the call has run.  Sums, statistics and log-sums are fp32; fp16 and bf16 calls round the
    softmax weights to that type before they meet the values.

    Where few rows see many keys (too few tiles of rows for half of the SMs, 512 keys and more a sequence on average) the keys are
    cut into parts that meet in the stream's scratch: make one such call on the stream before capturing a graph on it."""
    ft = FTYPES.get(q.dtype)
    if ft is None or not q.is_cuda:
        _ftype(q, "q")
    shape, ks = q.shape, k.shape
    if len(shape) != 3 or len(ks) != 3 or v.shape != ks or ks[2] != shape[2]:
        raise RuntimeError(f"q must be [rows, heads, channels], k and v [rows, key heads, channels], got {list(shape)}, {list(ks)} "
                           f"and {list(v.shape)}")
    for t, what in ((k, "k"), (v, "v")):
        if t.dtype != q.dtype or not t.is_cuda:
            _device_tensor(t, q.dtype, what)
    _check_starts(starts, "starts")
    if k_starts is not None:
        _check_starts(k_starts, "k_starts", starts.shape[0] - 1)
    if stream is not None:
        with _on(stream):
            return _attention(q, k, v, starts, k_starts, scale, out, return_lse, ft, shape, stream)
    return _attention(q, k, v, starts, k_starts, scale, out, return_lse, ft, shape, None)


def _attention(q, k, v, starts, k_starts, scale, out, return_lse, ft, shape, stream):
    handle = _launch_stream(stream, q, k, v, starts, k_starts, out)
    tq, hq, d = shape
    if q.stride(2) != 1:
        q = q.contiguous()
    if k.stride(2) != 1 or v.stride(2) != 1:
        k, v = k.contiguous(), v.contiguous()
    if out is None:
        out = starts.new_empty(shape, dtype=q.dtype)
    elif out.dtype != q.dtype or out.shape != shape or not out.is_contiguous() or not out.is_cuda:
        raise RuntimeError(f"out must be a contiguous {q.dtype} {list(shape)} CUDA tensor")
    lse = starts.new_empty((tq, hq), dtype=torch.float32) if return_lse else None
    (qt, qh, _), (kt, kh, _), (vt, vh, _) = q.stride(), k.stride(), v.stride()
    if scale is None:
        scale = d ** -0.5 if d else 1.0
    elif abs(scale) > 3e38:  # not an fp32: as what it would round to
        scale = math.inf
    _lib.check(_lib.lib().b200q_prompt_attention(
        _ARGS.pack(q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, starts.data_ptr(),
                   0 if k_starts is None else k_starts.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0, ft,
                   starts.shape[0] - 1, tq, k.shape[0], hq, k.shape[1], d, scale), handle))
    return (out, lse) if return_lse else out
