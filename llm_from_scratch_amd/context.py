"""Attention-metadata side channel, as utils/context.py:5-27 of the reference.

The model runner sets it before a forward pass; the paged attention layer
reads it (slot_mapping for store_kvcache; context_lens and block_tables for
the decode kernel; cu_seqlens for prefill).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch


@dataclass
class Context:
    is_prefill: bool = False
    cu_seqlens_q: Optional[torch.Tensor] = None
    cu_seqlens_k: Optional[torch.Tensor] = None
    max_seqlen_q: int = 0
    max_seqlen_k: int = 0
    slot_mapping: Optional[torch.Tensor] = None
    context_lens: Optional[torch.Tensor] = None
    block_tables: Optional[torch.Tensor] = None
    total_seqlen_k: Optional[int] = None  # of a prefill behind cached blocks: its keys in all
    cu_groups: Optional[torch.Tensor] = None  # of a decode over shared prefixes
    shared_blocks: Optional[torch.Tensor] = None


_CONTEXT = Context()


def get_context() -> Context:
    return _CONTEXT


def set_context(is_prefill, cu_seqlens_q=None, cu_seqlens_k=None, max_seqlen_q=0, max_seqlen_k=0,
                slot_mapping=None, context_lens=None, block_tables=None, total_seqlen_k=None, cu_groups=None,
                shared_blocks=None) -> None:
    global _CONTEXT
    _CONTEXT = Context(is_prefill, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k,
                       slot_mapping, context_lens, block_tables, total_seqlen_k, cu_groups, shared_blocks)


def reset_context() -> None:
    global _CONTEXT
    _CONTEXT = Context()
