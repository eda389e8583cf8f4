"""W4A16 attention block on B200: QKV projection, norms and rotation, a 4-bit paged cache, attention, output projection.

The neighbour of :class:`xqt_b200.ops.mlp.W4A16SwiGLUMLP` in a decoder layer.  Query, key and value projections are one horizontally fused W4A16
linear, as that block fuses gate and up; what lies between the projections is :func:`qk_norm_rope`, :func:`kv4_append` and
:func:`kv4_attention`.  One GPU: a rank of a larger group holds the block of its own heads.
"""

from __future__ import annotations

import torch

from ..contracts import PackedWeight
from ..errors import XQTBackendError
from .kv4 import HEAD_DIMS, allocate_kv4_cache, kv4_append, kv4_attention
from .mlp import _concat_rows, _Linear
from .rotary import qk_norm_rope


class W4A16Attention:
    """``o(attention(rope(norm(q x)), rope(norm(k x)), v x))`` over a cache that keeps keys and values in 4 bits.

    ``q`` is a canonical ``[q_heads * head_dim, hidden]`` weight, ``k`` and ``v`` ``[kv_heads * head_dim, hidden]``, ``o`` ``[hidden, q_heads * head_dim]``.
    ``frequencies``, ``axes``, ``interleaved``, ``q_norm`` / ``k_norm`` (weights of the head norms) and ``eps`` as :func:`qk_norm_rope` takes them; ``window``
    and ``scale`` as :func:`kv4_attention` does."""

    def __init__(self, q: PackedWeight, k: PackedWeight, v: PackedWeight, o: PackedWeight, *, kv_heads: int, head_dim: int, frequencies: torch.Tensor,
                 device: torch.device, dtype: torch.dtype = torch.bfloat16, axes: torch.Tensor | None = None, interleaved: bool = False,
                 q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-6, window: int | None = None,
                 scale: float | None = None) -> None:
        rows, hidden = q.metadata.logical_shape
        if head_dim not in HEAD_DIMS or kv_heads < 1 or rows % (kv_heads * head_dim) or rows == 0:
            raise XQTBackendError(f"W4A16Attention: a head dimension of {HEAD_DIMS}, and query heads that are a multiple of the key heads")
        for weight, shape in ((k, (kv_heads * head_dim, hidden)), (v, (kv_heads * head_dim, hidden)), (o, (hidden, rows))):
            if tuple(weight.metadata.logical_shape) != shape:
                raise XQTBackendError(f"W4A16Attention: a weight of {tuple(weight.metadata.logical_shape)} where {shape} is needed")
        self.q_heads, self.kv_heads, self.head_dim, self.hidden, self.dtype, self.device = rows // head_dim, kv_heads, head_dim, hidden, dtype, device
        self.qkv = _Linear(_concat_rows(_concat_rows(q, k), v), device, dtype)
        self.o = _Linear(o, device, dtype)

        def here(t: torch.Tensor | None) -> torch.Tensor | None:
            return None if t is None else t.to(device).contiguous()

        self.frequencies, self.axes, self.q_norm, self.k_norm = here(frequencies), here(axes), here(q_norm), here(k_norm)
        self.interleaved, self.eps, self.window, self.scale = interleaved, eps, window, scale

    def allocate_cache(self, pages: int, page_size: int = 64) -> tuple[torch.Tensor, torch.Tensor]:
        """``(codes, params)`` of a cache of this layer."""

        return allocate_kv4_cache(pages, self.kv_heads, self.head_dim, page_size=page_size, dtype=self.dtype, device=self.device)

    def __call__(self, x: torch.Tensor, positions: torch.Tensor, cache: tuple[torch.Tensor, torch.Tensor], slots: torch.Tensor, block_table: torch.Tensor,
                 seq_lens: torch.Tensor, query_starts: torch.Tensor | None = None) -> torch.Tensor:
        """``x`` ``[tokens, hidden]``: the new tokens of all sequences, ``slots`` where the cache keeps them, the rest as :func:`kv4_attention` takes it
        (``seq_lens`` with the new tokens)."""

        if x.ndim != 2 or x.shape[1] != self.hidden or x.dtype != self.dtype:
            raise XQTBackendError("W4A16Attention expects [tokens, hidden] in the block's type")
        tokens = x.shape[0]
        if tokens == 0:
            return torch.empty((0, self.hidden), dtype=self.dtype, device=x.device)
        heads = self.qkv(x).view(tokens, self.q_heads + 2 * self.kv_heads, self.head_dim)
        q, k = qk_norm_rope(heads[:, :self.q_heads], heads[:, self.q_heads:self.q_heads + self.kv_heads], positions, self.frequencies, axes=self.axes,
                            q_weight=self.q_norm, k_weight=self.k_norm, eps=self.eps, interleaved=self.interleaved)
        kv4_append(k, heads[:, self.q_heads + self.kv_heads:], *cache, slots)
        out = kv4_attention(q, *cache, block_table, seq_lens, query_starts=query_starts, window=self.window, scale=self.scale)
        return self.o(out.view(tokens, self.q_heads * self.head_dim))


__all__ = ["W4A16Attention"]
