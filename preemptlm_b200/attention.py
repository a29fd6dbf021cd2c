"""A decoder layer around the expert block: norm, paged attention, norm, experts.

The operators between two expert layers, run together as a serving step runs
them.  Every projection is 8-bit with block scales; the rows that enter one are
brought to 8 bits by the kernel before it (the norm, or ``ops.quantize_fp8``).
No host read anywhere, so a step can be captured as a CUDA graph.  A block with
a gate on its output or projections in another format puts the single calls
together itself.  No counterpart in the reference (its attention blocks are
mlx_lm's).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import ops
from .kv_cache import PagedKVCache
from .quant import quantize_fp8_weight


def rope_table(max_pos: int, rot: int, theta: float, device: str | torch.device = "cuda") -> torch.Tensor:
    """Cosines, then sines, of position * theta ** (-2 i / rot), i < rot / 2:
    fp32 [max_pos, rot], the angles formed in 64 bits."""
    i = torch.arange(0, rot, 2, device=device, dtype=torch.float64)
    angle = torch.arange(max_pos, device=device, dtype=torch.float64)[:, None] * theta ** (-i / rot)[None]
    return torch.cat((angle.cos(), angle.sin()), dim=1).float()


@dataclass
class PagedAttention:
    """Pre-norm attention of one layer over its paged cache.

    norm: bf16 [H].  qkv: 8-bit weight and scales of [(q_heads + 2 kv_heads) *
    D, H] (queries, keys, values).  out: of [H, q_heads * D].  q_norm / k_norm:
    bf16 [D] or None.  rope: ``rope_table`` or None."""

    norm: torch.Tensor
    qkv: tuple[torch.Tensor, torch.Tensor]
    out: tuple[torch.Tensor, torch.Tensor]
    cache: PagedKVCache
    q_heads: int
    rope: torch.Tensor | None = None
    q_norm: torch.Tensor | None = None
    k_norm: torch.Tensor | None = None
    eps: float = 1e-6

    @classmethod
    def from_weights(cls, norm, qkv, out, cache, q_heads, **kw) -> "PagedAttention":
        """With bf16 projection weights, brought to 8 bits here."""
        return cls(norm, quantize_fp8_weight(qkv), quantize_fp8_weight(out), cache, q_heads, **kw)

    def __call__(self, x: torch.Tensor, residual: torch.Tensor | None, page_table: torch.Tensor,
                 positions: torch.Tensor, rows: torch.Tensor | None = None):
        """One step of T tokens.  x [T, H] bf16 is added to the residual
        stream; token t is the positions[t]-th of page_table row rows[t] (row
        t if None; several tokens of a row in one call see each other's keys
        up to their own place).  A negative position marks a padding token,
        whose row may be anything.  A token whose row lies outside the table,
        or whose position outside ``rope``, attends nothing;
        ``ops.device_status`` reports it.  Returns (the attention's output [T,
        H], the new residual [T, H])."""
        T, D, kv = x.shape[0], self.cache.head_dim, self.cache.kv_heads
        y8, scales, residual = ops.add_rms_norm_fp8(x, self.norm, residual=residual, eps=self.eps)
        qkv = ops.fp8_linear(y8, scales, *self.qkv).view(T, self.q_heads + 2 * kv, D)
        q, k, v = qkv.split([self.q_heads, kv, kv], dim=1)
        q = ops.append_kv(self.cache, q, k, v, page_table, positions, self.rope, rows=rows, q_weight=self.q_norm,
                          k_weight=self.k_norm, eps=self.eps)
        o = ops.paged_attention(self.cache, q, page_table, positions + 1, rows=rows,
                                max_length=None if self.rope is None else self.rope.shape[0])
        o8, scales = ops.quantize_fp8(o.view(T, self.q_heads * D))
        return ops.fp8_linear(o8, scales, *self.out), residual


@dataclass
class DecoderLayer:
    """Attention, then an expert block on the normed residual stream.  moe: a
    ``Qwen3_xMoEWrapper`` (or any module of its call)."""

    attention: PagedAttention
    post_norm: torch.Tensor
    moe: object

    def __call__(self, x: torch.Tensor, residual: torch.Tensor | None, page_table: torch.Tensor,
                 positions: torch.Tensor, rows: torch.Tensor | None = None):
        """(the experts' output [T, H], the residual stream [T, H]): the next
        layer's x and residual."""
        a, residual = self.attention(x, residual, page_table, positions, rows)
        y, residual = ops.add_rms_norm(a, self.post_norm, residual=residual, eps=self.attention.eps)
        return self.moe(y.unsqueeze(0)).squeeze(0), residual
