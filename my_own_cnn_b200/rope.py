"""RMS norm of each query and key head with the position rotation in the same pass, and its gradient.

  * ``rope_table(positions, rot)`` -- the cosines and sines, fp32 [positions, rot];
  * ``qk_norm_rope(q, k, q_weight, k_weight, table, positions)`` -> (q, k) normalised and rotated;
  * ``qk_norm_rope_bprop(dq, dk, q, k, ...)`` -> gradients of q, k, q_weight and k_weight.
"""
from __future__ import annotations

import torch

from . import _lib
from .w4 import FTYPES, _device_tensor, _ftype, _launch_stream, _on


_ARGS = _lib.packer(_lib.CQKNormArgs)


def rope_table(positions: int, rot: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """cos, then sin, of position * base^(-2 i / rot), i < rot / 2 (angles in 64 bits, stored as fp32)."""
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    a = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * f
    return torch.cat([a.cos(), a.sin()], -1).float()


def _checked(q, k, q_weight, k_weight, table, positions):
    dtype = q.dtype
    ft = FTYPES.get(dtype)
    if ft is None or not q.is_cuda:
        _ftype(q, "q")
    if k.dtype != dtype or not k.is_cuda:
        _device_tensor(k, dtype, "k")
    qs, ks = q.shape, k.shape
    if len(qs) != 3 or len(ks) != 3 or qs[0] != ks[0] or qs[2] != ks[2]:
        raise RuntimeError(f"q and k must be [tokens, heads, channels] of the same tokens and channels, got "
                           f"{list(qs)} and {list(ks)}")
    t, hq, d = qs
    for w, what in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None and (w.dtype != dtype or not w.is_cuda or w.shape != (d,) or not w.is_contiguous()):
            _device_tensor(w, dtype, what)
            raise RuntimeError(f"{what} must be contiguous [{d}]")
    rot = rows = 0
    if table is not None:
        if table.dtype != torch.float32 or not table.is_cuda:
            _device_tensor(table, torch.float32, "table")
        if table.dim() != 2 or not table.is_contiguous():
            raise RuntimeError("table must be a contiguous [positions, rotated channels] tensor")
        rows, rot = table.shape
        if positions is None:
            raise RuntimeError("a rotation needs positions")
        if positions.dtype != torch.int32 or not positions.is_cuda:
            _device_tensor(positions, torch.int32, "positions")
        if positions.shape != (t,) or not positions.is_contiguous():
            raise RuntimeError(f"positions must be contiguous [{t}]")
    return ft, t, hq, ks[1], d, rot, rows


def _p(t) -> int:
    return 0 if t is None else t.data_ptr()


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                 table: torch.Tensor | None, positions: torch.Tensor | None, eps: float = 1e-6,
                 interleaved: bool = False, q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None,
                 stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """q [t, hq, d], k [t, hk, d]: views into a fused projection will do (contiguous channels).  Weights [d]
    of q's type or None; table None: no rotation; positions int32 [t].  q_out / k_out may be q / k."""
    ft, t, hq, hk, d, rot, rows = _checked(q, k, q_weight, k_weight, table, positions)
    if stream is None:
        return _norm(q, k, q_weight, k_weight, table, positions, eps, interleaved, q_out, k_out, ft, t, hq, hk, d, rot,
                     rows, None)
    with _on(stream):
        return _norm(q, k, q_weight, k_weight, table, positions, eps, interleaved, q_out, k_out, ft, t, hq, hk, d, rot,
                     rows, stream)


def _norm(q, k, q_weight, k_weight, table, positions, eps, interleaved, q_out, k_out, ft, t, hq, hk, d, rot, rows,
          stream):
    handle = _launch_stream(stream, q, k, q_weight, k_weight, table, positions, q_out, k_out)
    (qt, qh, qc), (kt, kh, kc) = q.stride(), k.stride()
    if qc != 1:
        q = q.contiguous()
        qt, qh, _ = q.stride()
    if kc != 1:
        k = k.contiguous()
        kt, kh, _ = k.stride()
    if q_out is None:
        q_out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((t, hq, d))
        ot, oh = hq * d, d
    else:
        ot, oh = _out_strides(q_out, q, "q_out")
    if k_out is None:
        k_out = torch.empty_like(k) if k.is_contiguous() else k.new_empty((t, hk, d))
        pt, ph = hk * d, d
    else:
        pt, ph = _out_strides(k_out, k, "k_out")
    _lib.check(_lib.lib().b200q_qk_norm_rope(_ARGS.pack(q.data_ptr(), k.data_ptr(), _p(q_weight), _p(k_weight), _p(table),
                                                        _p(positions), q_out.data_ptr(), k_out.data_ptr(), 0, 0, 0, 0,
                                                        qt, qh, kt, kh, ot, oh, pt, ph, rows, ft, t, hq, hk, d, rot,
                                                        interleaved, eps), handle))
    return q_out, k_out


def _out_strides(out, x, what):
    if out.dtype != x.dtype or out.shape != x.shape or out.stride(2) != 1 or not out.is_cuda:
        raise RuntimeError(f"{what} must be a {x.dtype} {list(x.shape)} CUDA tensor with contiguous channels")
    return out.stride(0), out.stride(1)


def qk_norm_rope_bprop(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                       q_weight: torch.Tensor | None, k_weight: torch.Tensor | None, table: torch.Tensor | None,
                       positions: torch.Tensor | None, eps: float = 1e-6, interleaved: bool = False, stream=None):
    """dq, dk: gradients of qk_norm_rope's outputs.  Returns the gradients of q, k, q_weight and k_weight
    (None for a weight that is None); the weights' are summed over tokens and heads in fp32 in a fixed order."""
    ft, t, hq, hk, d, rot, rows = _checked(q, k, q_weight, k_weight, table, positions)
    if dq.shape != q.shape or dk.shape != k.shape:
        raise RuntimeError("dq and dk must have the shapes of q and k")
    _device_tensor(dq, q.dtype, "dq")
    _device_tensor(dk, q.dtype, "dk")
    with _on(stream):
        handle = _launch_stream(stream, q, k, dq, dk, q_weight, k_weight, table, positions)
        if q.stride(2) != 1:
            q = q.contiguous()
        if k.stride(2) != 1:
            k = k.contiguous()
        dq, dk = dq.contiguous(), dk.contiguous()
        gq, gk = q.new_empty(dq.shape), k.new_empty(dk.shape)
        gqw = None if q_weight is None else q.new_empty((d,))
        gkw = None if k_weight is None else q.new_empty((d,))
        _lib.check(_lib.lib().b200q_qk_norm_rope_bprop(
            _ARGS.pack(q.data_ptr(), k.data_ptr(), _p(q_weight), _p(k_weight), _p(table), _p(positions), gq.data_ptr(),
                       gk.data_ptr(), dq.data_ptr(), dk.data_ptr(), _p(gqw), _p(gkw), q.stride(0), q.stride(1),
                       k.stride(0), k.stride(1), 0, 0, 0, 0, rows, ft, t, hq, hk, d, rot, interleaved, eps),
            handle))
    return gq, gk, gqw, gkw
