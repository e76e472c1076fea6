"""Attention over the paged cache on MI355X where sequences begin with the same pages: a long prompt that a batch has in common is read
once for all of its rows."""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from . import moba_efficient as E
from .paged import PagedKVCache, _addressable, _check_no_gradients, _check_rows, _check_table, _plain, _table, _taken, paged_attention


def _check_query(cache, query):
    _check_rows(cache, "query", query)
    tokens, heads = query.shape[:2]
    if tokens >= 1 << 24 or tokens * heads >= 1 << 31:
        raise ValueError("at most 2^24 - 1 tokens, and fewer than 2^31 rows")
    if not heads or heads % cache.k_pages.shape[1]:
        raise ValueError("the number of query heads must be a multiple of the number of key/value heads")


def paged_prefix_attention(query: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, lengths: torch.Tensor,
                           cu_new: torch.Tensor, cu_groups: torch.Tensor, shared: torch.Tensor,
                           scaling: Optional[float] = None) -> torch.Tensor:
    """``paged_attention`` of a batch in which sequences begin with the same pages.

    Args:
        query, cache, page_table, lengths, cu_new, scaling: as for ``paged_attention``; the table's rows name the common pages too,
            and the lengths count their tokens
        cu_groups: [groups + 1] int32, ascending: sequences ``cu_groups[g]`` .. ``cu_groups[g + 1] - 1`` begin alike; those in front of
            the first and behind the last group share nothing
        shared: [groups] int32, how many leading tokens the table's rows of a group name the same pages for.  The keys of these,
            up to a multiple of 64, are read through the group's first row, once for the new tokens of all of its sequences.
    Returns:
        what ``paged_attention`` does (with the sums in another order): every new token sees its sequence's tokens up to itself,
        also where ``shared`` says more than a sequence has.  Rows that see nothing are zeros.

    Precision is that of ``paged_attention`` for few rows where a group (for what it shares), or a sequence (for the rest), has up to
    256 rows, new tokens times heads on a key/value head; 128 with 16-bit pages and heads of 128.  Otherwise it is that for many, for
    the shared keys of a large group also where its sequences have few rows each.  The index tensors stay on the device: a captured call
    follows them.  The workspace holds every row's parts in 32 bits, two or three of them with many tokens.  No gradients.
    """
    out = _lib.host().paged_prefix_attention(cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales, query, page_table, lengths, cu_new,
                                             cu_groups, shared, scaling)
    if out is not NotImplemented:
        return out
    # tensors that have to be copied first, none at all, or wrong ones
    _check_no_gradients(cache, query)
    _check_query(cache, query)
    _check_table(cache, page_table, lengths, cu_new, query.device)
    for name, t in (("cu_groups", cu_groups), ("shared", shared)):
        if t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32")
        if t.dim() != 1:
            raise ValueError("cu_groups must be [groups + 1], shared [groups]")
        if t.device != query.device:
            raise ValueError("all tensors must be on one device")
    if cu_groups.shape[0] != shared.shape[0] + 1:
        raise ValueError("cu_groups must be [groups + 1], shared [groups]")
    if not query.is_cuda:
        raise RuntimeError("paged_prefix_attention needs tensors on an AMD GPU (there is no CPU path)")
    if not query.shape[0] or not page_table.shape[0] or not shared.shape[0]:
        return paged_attention(query, cache, page_table, lengths, cu_new, scaling)
    query = query if _addressable(query) else E._aligned(query)
    tensors = (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales, query, _table(page_table), lengths.contiguous(),
               cu_new.contiguous(), cu_groups.contiguous(), shared.contiguous())
    return _taken(_lib.host().paged_prefix_attention(*map(_plain, tensors), scaling), "paged_prefix_attention")
