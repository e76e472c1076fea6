"""Mixture of block attention for new tokens over the paged cache on MI355X: the sums of the pages' keys, the choice of blocks by them,
and the attention over the chosen blocks.  (The reference attends all keys once a prompt is in the cache, moba/wrapper.py:76-82; its
operator for whole prompts chooses by the means of the blocks' keys, moba/moba_efficient.py:326-371.)"""

from __future__ import annotations

from types import SimpleNamespace
from typing import Optional

import torch

from . import _lib
from . import moba_efficient as E
from .norm_rope import _has_tangent
from .paged import HEAD_DIMS, MAX_TOKENS, PAGE_SIZES, PagedKVCache, _addressable, _check_no_gradients, _check_table, _plain, _table, _taken
from .paged_prefix import _check_query

MAX_TOPK = 64
MAX_BLOCKS = 16384          # of a sequence, that paged_select_blocks chooses from
MAX_BLOCK_SIZE = 1 << 24


def paged_key_sums(cache: PagedKVCache, sums: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, cu_new: torch.Tensor,
                   rows: int) -> None:
    """The sums of the keys that pages hold, of those pages that have received new tokens.

    Args:
        cache, page_table, lengths, cu_new: as ``paged_append`` has had them
        sums: [num_pages, kv_heads, head_dim] float32, to be kept with the cache: ``sums[page, head]`` becomes the sum, in 32 bits,
            of the keys of the tokens that the page holds up to its sequence's last.  Other pages' sums are left as they are.
        rows: the packed rows that cu_new counts in (its last number or more, for which time is spent); at most 2^30 - 1

    At most some million sequences times key/value heads.
    """
    if _lib.host().paged_key_sums(cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales, sums, page_table, lengths, cu_new,
                                  rows) is not NotImplemented:
        return
    _check_no_gradients(cache, sums)
    k = cache.k_pages
    if sums.dtype != torch.float32:
        raise TypeError("the sums must be float32")
    if sums.shape != (*k.shape[:2], k.shape[3]) or not sums.is_contiguous() or sums.data_ptr() % 16:
        raise ValueError("the sums must be [num_pages, kv_heads, head_dim], contiguous and 16-byte aligned")
    _check_table(cache, page_table, lengths, cu_new, sums.device)
    if not 0 <= rows <= MAX_TOKENS:
        raise ValueError(f"rows must be 0 to {MAX_TOKENS}")
    if not k.is_cuda:
        raise RuntimeError("paged_key_sums needs tensors on an AMD GPU (there is no CPU path)")
    if rows and page_table.shape[0]:
        tensors = (k, cache.v_pages, cache.k_scales, cache.v_scales, sums, _table(page_table), lengths.contiguous(), cu_new.contiguous())
        _taken(_lib.host().paged_key_sums(*map(_plain, tensors), rows), "paged_key_sums")


def _check_blocks(block_size, page_size, topk):
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}")
    if not 0 < block_size <= MAX_BLOCK_SIZE or block_size % page_size:
        raise ValueError(f"block_size must be a multiple of page_size, at most {MAX_BLOCK_SIZE}")
    if not 0 < topk <= MAX_TOPK:
        raise ValueError(f"1 to {MAX_TOPK} blocks for each row")


def paged_select_blocks(query: torch.Tensor, sums: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, cu_new: torch.Tensor,
                        page_size: int, block_size: int, topk: int) -> torch.Tensor:
    """The blocks that every new token and head attends: its own, and those before it whose keys' mean has the largest product with
    the query.

    Args:
        query: [tokens, heads, head_dim] bf16 or fp16, the new tokens of all sequences one after the other; heads a multiple of the
            sums'
        sums: [num_pages, kv_heads, head_dim] float32, of ``paged_key_sums``
        page_table, lengths, cu_new: as for ``paged_attention``
        page_size, block_size: tokens of a page and of a block; block_size a multiple of page_size (``moba_chunk_size``)
        topk: blocks of a row, its own among them (``moba_topk``), 1 to 64
    Returns:
        [tokens, heads, topk] int32: numbers of blocks in the sequence, ascending; -1 behind the last where there are fewer, and
        throughout where a row belongs to no sequence.

    The products are with the sums of a block's pages, in 64 bits (all blocks before a token's own are whole), and do not depend on what
    else is in the batch; of equal ones the lowest block counts as larger, NaN as minus infinity.  A page that the table names wrongly
    adds nothing.  Tables of at most 16384 blocks; at most 2^24 - 1 tokens, fewer than 2^31 tokens times heads, and some million sequences
    times key/value heads.  The workspace holds the scores, up to 512 MiB (one token's at least).
    (``moba_attn_varlen`` rounds the blocks' means to the keys' type first, which can decide between blocks of nearly equal
    products otherwise.)  No gradients.
    """
    out = _lib.host().paged_select_blocks(query, sums, page_table, lengths, cu_new, page_size, block_size, topk)
    if out is not NotImplemented:
        return out
    if torch.is_grad_enabled() and (query.requires_grad or sums.requires_grad):
        raise RuntimeError("the choice of blocks has no gradients: call it under torch.no_grad()")
    if _has_tangent(query, sums):
        raise RuntimeError("the choice of blocks has no forward-mode derivatives: tensors with a tangent are refused")
    if query.dtype not in (torch.bfloat16, torch.float16) or sums.dtype != torch.float32:
        raise TypeError("query must be bfloat16 or float16, and sums float32")
    if sums.dim() != 3 or sums.shape[2] not in HEAD_DIMS or not sums.shape[0] or not 0 < sums.shape[1] <= 65535:
        raise ValueError(f"sums must be [num_pages, kv_heads, head_dim], head_dim one of {HEAD_DIMS}")
    if query.dim() != 3 or query.shape[2] != sums.shape[2] or not query.shape[1] or query.shape[1] % sums.shape[1]:
        raise ValueError("query must be [tokens, heads, head_dim] with the sums' head_dim and a multiple of their heads")
    if query.shape[0] >= 1 << 24 or query.shape[0] * query.shape[1] >= 1 << 31:
        raise ValueError("at most 2^24 - 1 tokens, and fewer than 2^31 rows")
    _check_table(SimpleNamespace(k_pages=sums), page_table, lengths, cu_new, query.device)
    _check_blocks(block_size, page_size, topk)
    if page_table.shape[1] > MAX_BLOCKS * (block_size // page_size):
        raise ValueError(f"at most {MAX_BLOCKS} blocks in a row of the table")
    if not query.is_cuda:
        raise RuntimeError("paged_select_blocks needs tensors on an AMD GPU (there is no CPU path)")
    if not query.shape[0] or not page_table.shape[0]:
        return torch.full((*query.shape[:2], topk), -1, dtype=torch.int32, device=query.device)
    query = query if _addressable(query) else E._aligned(query)
    sums = sums if sums.is_contiguous() and sums.data_ptr() % 16 == 0 else E._aligned(sums)
    tensors = (query, sums, _table(page_table), lengths.contiguous(), cu_new.contiguous())
    return _taken(_lib.host().paged_select_blocks(*map(_plain, tensors), page_size, block_size, topk), "paged_select_blocks")


def paged_block_attention(query: torch.Tensor, cache: PagedKVCache, blocks: torch.Tensor, page_table: torch.Tensor,
                          lengths: torch.Tensor, cu_new: torch.Tensor, block_size: int, scaling: Optional[float] = None) -> torch.Tensor:
    """Attention of new tokens over some blocks of the cache, each token and head its own: mixture of block attention for generation.

    Args:
        query, cache, page_table, lengths, cu_new, scaling: as for ``paged_attention``
        blocks: [tokens, heads, n] int32, n at most 64, as ``paged_select_blocks`` gives them: numbers of blocks of ``block_size`` tokens in
            the token's sequence, in any order.  An entry that is no block of the sequence up to the token's own is none, one that
            is there twice counts once.  A token's own block is attended only if it is among them.
        block_size: a multiple of the page size, at most 2^24
    Returns:
        [tokens, heads, head_dim] in query's dtype: softmax attention over the tokens of the blocks up to the row's own.  Rows
        that see nothing are zeros, as in ``paged_attention``.  No gradients.

    Up to 32 rows (new tokens times heads on a key/value head) of a sequence read the union of their blocks once.  Made for one or some
    new tokens of each sequence; a long piece of a prompt is cut into groups of 32 rows, each of which reads its own union.  How much the
    rows' blocks have in common decides: 64 and 2048 tokens behind 131072 (twelve blocks of 4096, 32 heads on 8, 8 bits) take 0.10 and 2.8 ms
    where all of a key/value head's rows have the same blocks and 0.27 and 9.0 ms where each has its own at random; ``paged_attention``
    over all keys 0.16 and 3.9, the less for pieces of prompts from some ten tokens on unless their rows choose much alike or the
    history is many times what they choose.
    Scores, softmax statistics and sums are 32 bits, a probability the sum of two 16-bit elements, as in ``paged_attention`` for few
    rows.  The workspace holds parts of the rows in 32 bits and, where 32 rows may choose more than 1024 of a table's blocks, the lists of these,
    up to 512 MiB.  At most 2^24 - 1 tokens, fewer than 2^31 tokens times heads, and some million sequences times key/value heads.
    """
    out = _lib.host().paged_block_attention(cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales, query, page_table, lengths, cu_new,
                                            blocks, block_size, scaling)
    if out is not NotImplemented:
        return out
    _check_no_gradients(cache, query)
    _check_query(cache, query)
    if blocks.dtype != torch.int32:
        raise TypeError("blocks must be int32")
    if blocks.dim() != 3 or blocks.shape[:2] != query.shape[:2]:
        raise ValueError("blocks must be [tokens, heads, n]")
    if blocks.device != query.device:
        raise ValueError("all tensors must be on one device")
    _check_blocks(block_size, cache.k_pages.shape[2], blocks.shape[2])
    _check_table(cache, page_table, lengths, cu_new, query.device)
    if not query.is_cuda:
        raise RuntimeError("paged_block_attention needs tensors on an AMD GPU (there is no CPU path)")
    if not query.shape[0] or not page_table.shape[0]:
        return torch.zeros(query.shape, dtype=query.dtype, device=query.device)
    query = query if _addressable(query) else E._aligned(query)
    tensors = (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales, query, _table(page_table), lengths.contiguous(),
               cu_new.contiguous(), blocks.contiguous())
    return _taken(_lib.host().paged_block_attention(*map(_plain, tensors), block_size, scaling), "paged_block_attention")
