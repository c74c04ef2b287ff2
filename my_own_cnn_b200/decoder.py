"""Attention blocks of a decoder: 4-bit weights for tokens (W4Attention), 8-bit weights for prompts and tokens (S8Attention), both
over a 4-bit cache.

``W4Attention.forward`` runs the block for the new tokens of a batch of sequences: projection (linear_w4),
norms and rotation in place (qk_norm_rope), keys and values into the paged cache (kv4_append), attention over
the cache (kv4_attention), output projection (linear_w4).  Five kernels, no copy in between: queries, keys
and values stay views into the projection's output.
examples/decode_w4.py answers tokens with a random block, captured in a CUDA graph.

``S8Attention`` also adds the residual and norms its input.  ``prompt`` takes whole prompts, packed one after another, and leaves
their keys and values in the cache; ``forward`` goes on from there token by token.  examples/prompt_s8.py does both.
"""
from __future__ import annotations

import torch

from .kv4 import KV4Cache, kv4_append, kv4_attention
from .prompt import prompt_attention
from .rope import qk_norm_rope, rope_table
from .s8 import S8Rows, linear_s8, quantize_s8, rms_norm_s8
from .w4 import W4Weight, linear_w4, quantize_w4


class W4Attention:
    """wqkv: [(heads + 2 * kv_heads) * head_dim, hidden] (queries, keys, values); wo: [hidden, heads * head_dim];
    q_norm, k_norm: [head_dim] of the activations' type, or None; table: rope_table's, or None."""

    def __init__(self, wqkv: W4Weight, wo: W4Weight, q_norm: torch.Tensor | None, k_norm: torch.Tensor | None,
                 table: torch.Tensor | None, heads: int, kv_heads: int, head_dim: int, eps: float = 1e-6,
                 interleaved: bool = False):
        if wqkv.n != (heads + 2 * kv_heads) * head_dim or wo.k != heads * head_dim:
            raise RuntimeError(f"projections of {wqkv.n} and from {wo.k} channels do not fit {heads} + 2 * {kv_heads} heads "
                               f"of {head_dim}")
        self.wqkv, self.wo, self.q_norm, self.k_norm, self.table = wqkv, wo, q_norm, k_norm, table
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.eps, self.interleaved = eps, interleaved

    def forward(self, x: torch.Tensor, cache: KV4Cache, positions: torch.Tensor, slots: torch.Tensor,
                block_table: torch.Tensor, lens: torch.Tensor, stream=None) -> torch.Tensor:
        """x [b, tq, hidden]: the next tq tokens of each sequence; positions int32 and slots int64 [b * tq] place them;
        lens int32 [b] counts each sequence's tokens with the new ones.  Returns [b, tq, wo.n]."""
        b, tq, _ = x.shape
        h, hk, d = self.heads, self.kv_heads, self.head_dim
        qkv = linear_w4(x, self.wqkv, stream=stream).view(b * tq, h + 2 * hk, d)
        q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
        qk_norm_rope(q, k, self.q_norm, self.k_norm, self.table, positions, self.eps, self.interleaved, q_out=q, k_out=k,
                     stream=stream)
        kv4_append(cache, k, v, slots, stream=stream)
        out = kv4_attention(q.unflatten(0, (b, tq)), cache, block_table, lens, stream=stream)
        return linear_w4(out.view(b * tq, h * d), self.wo, stream=stream).view(b, tq, self.wo.n)


def random_block(hidden: int, heads: int, kv_heads: int, head_dim: int, dtype: torch.dtype, positions: int = 8192,
                 group: int = 64, device="cuda", seed: int = 0) -> W4Attention:
    g = torch.Generator(device=device)
    g.manual_seed(seed)

    def weight(n, k):
        return quantize_w4(torch.randn(n, k, generator=g, device=device) * k ** -0.5, group)

    norms = [(1 + 0.1 * torch.randn(head_dim, generator=g, device=device)).to(dtype) for _ in range(2)]
    return W4Attention(weight((heads + 2 * kv_heads) * head_dim, hidden), weight(hidden, heads * head_dim), *norms,
                       rope_table(positions, head_dim, device=device), heads, kv_heads, head_dim)


class S8Attention:
    """norm: [hidden] of the activations' type; wqkv: 8-bit rows [(heads + 2 * kv_heads) * head_dim, hidden] (queries, keys,
    values); wo: [hidden, heads * head_dim]; q_norm, k_norm: [head_dim], or None; table: rope_table's, or None."""

    def __init__(self, norm: torch.Tensor, wqkv: S8Rows, wo: S8Rows, q_norm: torch.Tensor | None, k_norm: torch.Tensor | None,
                 table: torch.Tensor | None, heads: int, kv_heads: int, head_dim: int, eps: float = 1e-6,
                 interleaved: bool = False):
        if wqkv.shape != ((heads + 2 * kv_heads) * head_dim, norm.shape[0]) or wo.k != heads * head_dim:
            raise RuntimeError(f"projections {list(wqkv.shape)} and from {wo.k} channels do not fit {heads} + 2 * {kv_heads} heads "
                               f"of {head_dim} and {norm.shape[0]} hidden channels")
        self.norm, self.wqkv, self.wo, self.q_norm, self.k_norm, self.table = norm, wqkv, wo, q_norm, k_norm, table
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.eps, self.interleaved = eps, interleaved

    def _project(self, x, residual, cache, positions, slots, stream):
        """Queries, keys and values of x [t, hidden], keys and values in the cache; and the residual."""
        h, hk, d = self.heads, self.kv_heads, self.head_dim
        if residual is None:
            rows, residual = rms_norm_s8(x, self.norm, eps=self.eps, stream=stream), x
        else:
            rows, residual = rms_norm_s8(x, self.norm, residual=residual, eps=self.eps, stream=stream)
        qkv = linear_s8(rows, self.wqkv, dtype=x.dtype, stream=stream).view(x.shape[0], h + 2 * hk, d)
        q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
        qk_norm_rope(q, k, self.q_norm, self.k_norm, self.table, positions, self.eps, self.interleaved, q_out=q, k_out=k,
                     stream=stream)
        if cache is not None:
            kv4_append(cache, k, v, slots, stream=stream)
        return q, k, v, residual

    def _output(self, attention, t, dtype, stream):
        rows = quantize_s8(attention.view(t, self.heads * self.head_dim), stream=stream)
        return linear_s8(rows, self.wo, dtype=dtype, stream=stream)

    def prompt(self, x: torch.Tensor, residual: torch.Tensor | None, positions: torch.Tensor, starts: torch.Tensor,
               cache: KV4Cache | None = None, slots: torch.Tensor | None = None, stream=None) -> tuple[torch.Tensor, torch.Tensor]:
        """x [t, hidden]: prompts packed one after another, sequence i in rows starts[i] .. starts[i + 1] (int32 on the device);
        positions int32 [t]; slots int64 [t] place keys and values in the cache (None: they are not kept).  Returns the block's
        output [t, hidden] (anything in rows outside every prompt) and the residual (x + residual, in place of the residual; x when
        there is none)."""
        if (cache is None) != (slots is None):
            raise RuntimeError("a cache and slots go together")
        q, k, v, residual = self._project(x, residual, cache, positions, slots, stream)
        return self._output(prompt_attention(q, k, v, starts, stream=stream), x.shape[0], x.dtype, stream), residual

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None, cache: KV4Cache, positions: torch.Tensor, slots: torch.Tensor,
                block_table: torch.Tensor, lens: torch.Tensor, stream=None) -> tuple[torch.Tensor, torch.Tensor]:
        """x [b * tq, hidden]: the next tq tokens of each of the b sequences; lens int32 [b] counts each one's tokens with the new ones."""
        q, _, _, residual = self._project(x, residual, cache, positions, slots, stream)
        b = lens.shape[0]
        out = kv4_attention(q.unflatten(0, (b, x.shape[0] // max(b, 1))), cache, block_table, lens, stream=stream)
        return self._output(out, x.shape[0], x.dtype, stream), residual


def random_block_s8(hidden: int, heads: int, kv_heads: int, head_dim: int, dtype: torch.dtype, positions: int = 8192,
                    device="cuda", seed: int = 0) -> S8Attention:
    g = torch.Generator(device=device)
    g.manual_seed(seed)

    def weight(n, k):
        return quantize_s8(torch.randn(n, k, generator=g, device=device) * k ** -0.5)

    norms = [(1 + 0.1 * torch.randn(n, generator=g, device=device)).to(dtype) for n in (hidden, head_dim, head_dim)]
    return S8Attention(norms[0], weight((heads + 2 * kv_heads) * head_dim, hidden), weight(hidden, heads * head_dim), *norms[1:],
                       rope_table(positions, head_dim, device=device), heads, kv_heads, head_dim)
