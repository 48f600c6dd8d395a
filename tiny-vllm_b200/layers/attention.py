"""The attention layer of a decoder (reference: ``nanovllm/layers/attention.py:43-89``, same constructor, cache
attributes and call)."""
from __future__ import annotations

import torch
from torch import nn

from ..attention import decode_attention, prefill_attention, store_kv
from ..utils.context import get_context


class Attention(nn.Module):
    """Grouped-head attention of one decoder layer (of one rank's heads, with tensor parallelism).

    ``k_cache`` and ``v_cache`` are empty until the runner assigns this layer's part of the cache,
    ``[pages, page size, num_kv_heads, head_dim]`` each; a call then stores its keys and values first, by the
    context's ``slot_mapping``.  In a prefill step sequences are packed; where the context has ``block_tables``
    the keys and values come from the cache (a cached prefix in front of the prompt), else from the call.  In a
    decode step each token attends over its sequence's pages.
    """

    def __init__(self, num_heads: int, head_dim: int, scale: float, num_kv_heads: int):
        super().__init__()
        self.num_heads = num_heads
        self.head_dim = head_dim
        self.scale = scale
        self.num_kv_heads = num_kv_heads
        self.k_cache = self.v_cache = torch.tensor([])

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        """``q``: ``[tokens, num_heads, head_dim]``, ``k`` and ``v``: ``[tokens, num_kv_heads, head_dim]``, or the
        same with heads and dim in one dimension; returns ``q``'s shape."""
        context = get_context()
        shape = q.shape
        q = q.view(-1, self.num_heads, self.head_dim)
        k = k.view(-1, self.num_kv_heads, self.head_dim)
        v = v.view(-1, self.num_kv_heads, self.head_dim)
        if self.k_cache.numel() and context.slot_mapping is not None:
            store_kv(k, v, self.k_cache, self.v_cache, context.slot_mapping)
        if context.is_prefill:
            if context.block_tables is not None:
                k, v = self.k_cache, self.v_cache
            o = prefill_attention(q, k, v, context.cu_seqlens_q, context.cu_seqlens_k, context.max_seqlen_q,
                                  context.max_seqlen_k, scale=self.scale, block_tables=context.block_tables)
        else:
            o = decode_attention(q, self.k_cache, self.v_cache, context.context_lens, context.block_tables,
                                 scale=self.scale)
        return o.view(shape)
