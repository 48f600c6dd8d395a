"""What the attention layers of a step have to know, set by the runner before the model is called (reference:
``nanovllm/utils/context.py:5-27``, same names)."""
from __future__ import annotations

from dataclasses import dataclass

import torch


@dataclass
class Context:
    is_prefill: bool = False
    cu_seqlens_q: torch.Tensor | None = None     # int32 [sequences + 1]
    cu_seqlens_k: torch.Tensor | None = None
    max_seqlen_q: int = 0
    max_seqlen_k: int = 0
    slot_mapping: torch.Tensor | None = None     # int32 [tokens], -1: not stored
    context_lens: torch.Tensor | None = None     # int32 [sequences]
    block_tables: torch.Tensor | None = None     # int32 [sequences, pages]


_CONTEXT = Context()


def get_context() -> Context:
    return _CONTEXT


def set_context(is_prefill: bool, cu_seqlens_q=None, cu_seqlens_k=None, max_seqlen_q: int = 0, max_seqlen_k: int = 0,
                slot_mapping=None, context_lens=None, block_tables=None) -> None:
    global _CONTEXT
    _CONTEXT = Context(is_prefill, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, slot_mapping, context_lens,
                       block_tables)


def reset_context() -> None:
    global _CONTEXT
    _CONTEXT = Context()
