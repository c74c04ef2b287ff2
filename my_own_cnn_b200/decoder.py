"""One attention block of a decoder with everything that it keeps held in 4 bits.

``W4Attention.forward`` runs the block for the new tokens of a batch of sequences: projection (linear_w4),
norms and rotation in place (qk_norm_rope), keys and values into the paged cache (kv4_append), attention over
the cache (kv4_attention), output projection (linear_w4).  Five kernels, no copy in between: queries, keys
and values stay views into the projection's output.
examples/decode_w4.py answers tokens with a random block, captured in a CUDA graph.
"""
from __future__ import annotations

import torch

from .kv4 import KV4Cache, kv4_append, kv4_attention
from .rope import qk_norm_rope, rope_table
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
