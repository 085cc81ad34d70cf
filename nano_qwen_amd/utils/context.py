"""Per-step attention metadata side channel.

Field-for-field restatement of the reference's ``Context``
(utils/context.py:5-28): the model runner fills it before each forward and
``Attention.forward`` reads it.  ``state_indices`` is carried for parity
(the reference uses it only for its linear-attention layers).  A step that
verifies trees of drafted tokens (no counterpart in the reference) has a
``TreeContext``: the fields of a prefill over paged K/V, and the trees' mask.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch


@dataclass(slots=True)
class Context:
    is_prefill: bool = False
    cu_seqlens_q: torch.Tensor | None = None
    cu_seqlens_k: torch.Tensor | None = None
    max_seqlen_q: int = 0
    max_seqlen_k: int = 0
    slot_mapping: torch.Tensor | None = None
    context_lens: torch.Tensor | None = None
    block_tables: torch.Tensor | None = None
    state_indices: torch.Tensor | None = None


@dataclass(slots=True)
class TreeContext(Context):
    tree_mask: torch.Tensor | None = None


_CONTEXT = Context()


def get_context() -> Context:
    return _CONTEXT


def set_context(is_prefill, cu_seqlens_q=None, cu_seqlens_k=None, max_seqlen_q=0, max_seqlen_k=0,
                slot_mapping=None, context_lens=None, block_tables=None, state_indices=None):
    global _CONTEXT
    _CONTEXT = Context(is_prefill, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k,
                       slot_mapping, context_lens, block_tables, state_indices)


def set_tree_context(cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, slot_mapping, block_tables, tree_mask):
    global _CONTEXT
    _CONTEXT = TreeContext(True, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, slot_mapping, None,
                           block_tables, None, tree_mask)


def reset_context():
    global _CONTEXT
    _CONTEXT = Context()
