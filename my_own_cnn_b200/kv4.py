"""Paged key / value cache held in 4 bits, and the attention of new tokens over it.

  * ``KV4Cache.empty(pages, heads, page_size, head_dim, group)`` -- the cache;
  * ``kv4_append(cache, k, v, slots)`` -- quantizes keys and values into slots (page * page_size + place);
  * ``kv4_read(cache, slots, dtype)`` -- the values that slots hold;
  * ``kv4_attention(q, cache, block_table, lens)`` -- softmax(scale * q k^T) v over each sequence's pages.
"""
from __future__ import annotations

import torch

from . import _lib
from .w4 import FTYPES, _device_tensor, _ftype, _launch_stream, _on


_CACHE = _lib.packer(_lib.CKV4Cache)
_ARGS = _lib.packer(_lib.CKV4AttentionArgs)


class KV4Cache:
    """codes uint8 [pages, heads, page_size, d / 2] (low nibble = even channel) and params int32
    [pages, heads, page_size, d / group] (bf16 scale bits, zero point in bits 16-23), for keys and values;
    value = (code - zero) * scale."""

    __slots__ = ("k_codes", "k_params", "v_codes", "v_params", "pages", "heads", "page_size", "head_dim", "group",
                 "_c")

    def __init__(self, k_codes: torch.Tensor, k_params: torch.Tensor, v_codes: torch.Tensor, v_params: torch.Tensor):
        shape, pshape = k_codes.shape, k_params.shape
        if len(shape) != 4 or len(pshape) != 4 or pshape[:3] != shape[:3] or pshape[3] == 0:
            raise RuntimeError(f"cache codes [pages, heads, page_size, d / 2] and params [pages, heads, page_size, "
                               f"d / group] expected, got {list(shape)} and {list(pshape)}")
        if v_codes.shape != shape or v_params.shape != pshape:
            raise RuntimeError("keys and values must have the same cache shapes")
        if k_codes.dtype != torch.uint8 or v_codes.dtype != torch.uint8:
            raise TypeError("cache codes must be uint8")
        if k_params.dtype != torch.int32 or v_params.dtype != torch.int32:
            raise TypeError("cache params must be int32")
        at = k_codes.get_device()
        for x in (k_codes, k_params, v_codes, v_params):
            if not x.is_contiguous():
                raise RuntimeError("cache tensors must be contiguous")
            if not x.is_cuda:
                raise RuntimeError("tensor arguments must be CUDA device tensors")
            if x.get_device() != at:
                raise RuntimeError("the tensors of a cache must be on one device")
        self.k_codes, self.k_params, self.v_codes, self.v_params = k_codes, k_params, v_codes, v_params
        self.pages, self.heads, self.page_size, half = shape
        self.head_dim = 2 * half
        self.group = self.head_dim // pshape[3]
        self._c = _CACHE.pack(k_codes.data_ptr(), k_params.data_ptr(), v_codes.data_ptr(), v_params.data_ptr(),
                              self.pages, self.heads, self.page_size, self.head_dim, self.group)

    @staticmethod
    def empty(pages: int, heads: int, page_size: int, head_dim: int, group: int = 64, device="cuda") -> "KV4Cache":
        """An uninitialised cache: places that no kv4_append has written hold any bits."""
        if head_dim not in (64, 128, 256) or group not in (32, 64):
            raise RuntimeError(f"4-bit caches have heads of 64, 128 or 256 channels in groups of 32 or 64, got "
                               f"{head_dim} and {group}")
        def codes():
            return torch.empty((pages, heads, page_size, head_dim // 2), dtype=torch.uint8, device=device)

        def params():
            return torch.empty((pages, heads, page_size, head_dim // group), dtype=torch.int32, device=device)

        return KV4Cache(codes(), params(), codes(), params())


def _check_slots(slots, t=None):
    if slots.dtype != torch.int64 or not slots.is_cuda:
        _device_tensor(slots, torch.int64, "slots")
    if slots.dim() != 1 or not slots.is_contiguous() or (t is not None and slots.shape[0] != t):
        raise RuntimeError(f"slots must be contiguous [{'tokens' if t is None else t}]")


def kv4_append(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, stream=None) -> None:
    """k, v [t, heads, d] (views with contiguous channels will do) into slots int64 [t]; negative slots are
    skipped, and no slot may be named twice.  A group of channels with a NaN or an infinity in it is stored as NaN."""
    ft = FTYPES.get(k.dtype)
    if ft is None or not k.is_cuda:
        _ftype(k, "k")
    if v.dtype != k.dtype or not v.is_cuda:
        _device_tensor(v, k.dtype, "v")
    shape = k.shape
    if len(shape) != 3 or v.shape != shape or shape[1] != cache.heads or shape[2] != cache.head_dim:
        raise RuntimeError(f"k and v must be [tokens, {cache.heads}, {cache.head_dim}], got {list(shape)} and "
                           f"{list(v.shape)}")
    _check_slots(slots, shape[0])
    if stream is not None:
        with _on(stream):
            return _append(cache, k, v, slots, ft, stream)
    return _append(cache, k, v, slots, ft, None)


def _append(cache, k, v, slots, ft, stream):
    handle = _launch_stream(stream, k, v, slots, cache.k_codes)
    (kt, kh, kc), (vt, vh, vc) = k.stride(), v.stride()
    if kc != 1 or vc != 1:
        k, v = k.contiguous(), v.contiguous()
        (kt, kh, _), (vt, vh, _) = k.stride(), v.stride()
    _lib.check(_lib.lib().b200q_kv4_append(cache._c, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, slots.data_ptr(), ft,
                                           k.shape[0], handle))


def kv4_read(cache: KV4Cache, slots: torch.Tensor, dtype: torch.dtype = torch.float32,
             stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [t, heads, d] of `dtype`: the values held in slots int64 [t]; zeros where a slot is negative."""
    ft = FTYPES.get(dtype)
    if ft is None:
        raise TypeError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    _check_slots(slots)
    if stream is not None:
        with _on(stream):
            return _read(cache, slots, dtype, ft, stream)
    return _read(cache, slots, dtype, ft, None)


def _read(cache, slots, dtype, ft, stream):
    handle = _launch_stream(stream, slots, cache.k_codes)
    t = slots.shape[0]
    k = slots.new_empty((t, cache.heads, cache.head_dim), dtype=dtype)
    v = torch.empty_like(k)
    _lib.check(_lib.lib().b200q_kv4_read(cache._c, slots.data_ptr(), k.data_ptr(), v.data_ptr(), ft, t, handle))
    return k, v


def kv4_attention(q: torch.Tensor, cache: KV4Cache, block_table: torch.Tensor, lens: torch.Tensor,
                  scale: float | None = None, out: torch.Tensor | None = None, return_lse: bool = False, stream=None):
    """q [b, tq, hq, d]: the last tq tokens of each sequence, whose keys and values the cache already holds;
    lens int32 [b] counts all tokens, block_table int32 [b, max_pages] names each sequence's pages.  Token i sees
    the first lens - tq + i + 1 places; where that is none the output is 0 (lse -inf).  Query head h reads cache
    head h // (hq / heads).  Table and lengths stay as they are until the call has run.  scale: 1 / sqrt(d) when None.  Returns out [b, tq, hq, d], and lse fp32 [b, tq, hq]
    (log of the sum of exp(scale * q.k)) when return_lse."""
    ft = FTYPES.get(q.dtype)
    if ft is None or not q.is_cuda:
        _ftype(q, "q")
    shape = q.shape
    if len(shape) != 4 or shape[3] != cache.head_dim:
        raise RuntimeError(f"q must be [sequences, tokens, heads, {cache.head_dim}], got {list(shape)}")
    b = shape[0]
    if block_table.dtype != torch.int32 or not block_table.is_cuda:
        _device_tensor(block_table, torch.int32, "block_table")
    if lens.dtype != torch.int32 or not lens.is_cuda:
        _device_tensor(lens, torch.int32, "lens")
    table = block_table.shape
    if len(table) != 2 or table[0] != b or (table[1] > 1 and block_table.stride(1) != 1):
        raise RuntimeError(f"block_table must be [{b}, pages] with contiguous rows, got {list(table)}")
    if lens.shape != (b,) or not lens.is_contiguous():
        raise RuntimeError(f"lens must be contiguous [{b}]")
    if stream is not None:
        with _on(stream):
            return _attention(q, cache, block_table, lens, scale, out, return_lse, ft, shape, table[1], stream)
    return _attention(q, cache, block_table, lens, scale, out, return_lse, ft, shape, table[1], None)


def _attention(q, cache, block_table, lens, scale, out, return_lse, ft, shape, max_pages, stream):
    handle = _launch_stream(stream, q, cache.k_codes, block_table, lens, out)
    b, tq, hq, d = shape
    qb, qt, qh, qc = q.stride()
    if qc != 1:
        q = q.contiguous()
        qb, qt, qh, _ = q.stride()
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
    elif out.dtype != q.dtype or out.shape != shape or not out.is_contiguous() or not out.is_cuda:
        raise RuntimeError(f"out must be a contiguous {q.dtype} {list(shape)} CUDA tensor")
    lse = lens.new_empty((b, tq, hq), dtype=torch.float32) if return_lse else None
    _lib.check(_lib.lib().b200q_kv4_attention(cache._c, _ARGS.pack(q.data_ptr(), qb, qt, qh, block_table.data_ptr(),
                                                                   block_table.stride(0), lens.data_ptr(),
                                                                   out.data_ptr(), lse.data_ptr() if return_lse else 0,
                                                                   ft, b, tq, hq, max_pages,
                                                                   d ** -0.5 if scale is None else scale), handle))
    return (out, lse) if return_lse else out
