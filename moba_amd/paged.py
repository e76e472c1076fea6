"""A paged key/value cache on MI355X, with 16-bit elements or 8-bit ones and a scale for every page and head, and the operators on
it: ``paged_append`` writes the keys and values of new tokens, rotated by position on the way, and ``paged_attention`` attends
them.  Sequences of any lengths and any numbers of new tokens are served together.  (The reference keeps transformers' contiguous
cache, one length for the whole batch, moba/wrapper.py:76-82.)"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from . import moba_efficient as E
from .norm_rope import _check_inv_freq, _has_tangent, _readable, _strides_of

E4M3 = torch.float8_e4m3fn
PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128)
MAX_KV_HEADS = 256
MAX_TOKENS = (1 << 30) - 1   # packed rows of a call; paged_append's launch and paged_attention take fewer, see there


@dataclass(frozen=True, eq=False)
class PagedKVCache:
    """The pages of one layer.

    k_pages, v_pages: [num_pages, kv_heads, page_size, head_dim], bf16, fp16 or e4m3 (``torch.float8_e4m3fn``); page_size
        16, 32, 64, 128 or 256, head_dim 64 or 128
    k_scales, v_scales: [num_pages, kv_heads] float32, for e4m3 only: an element stands for its value times the scale of its
        page and head.  Those that ``paged_append`` sets are powers of two; of a page that holds tokens it keeps one of any value
        that is large enough for the new ones as well.

    Which pages belong to which sequence is the caller's affair (the ``page_table`` of the calls).  Pages may be shared by
    sequences that only read them; a page that receives tokens in a call must be named once in the whole table.
    """

    k_pages: torch.Tensor
    v_pages: torch.Tensor
    k_scales: Optional[torch.Tensor] = None
    v_scales: Optional[torch.Tensor] = None

    def __post_init__(self):
        k = self.k_pages
        if k.dtype not in (torch.bfloat16, torch.float16, E4M3) or self.v_pages.dtype != k.dtype:
            raise TypeError("the pages must be bfloat16, float16 or float8_e4m3fn, keys and values alike")
        if k.dim() != 4 or self.v_pages.shape != k.shape:
            raise ValueError("k_pages and v_pages must be [num_pages, kv_heads, page_size, head_dim]")
        if k.shape[2] not in PAGE_SIZES or k.shape[3] not in HEAD_DIMS:
            raise ValueError(f"page_size must be one of {PAGE_SIZES} and head_dim one of {HEAD_DIMS}")
        if not (0 < k.shape[0] < 1 << 31 and 0 < k.shape[1] <= MAX_KV_HEADS):
            raise ValueError(f"there must be pages, and 1 to {MAX_KV_HEADS} key/value heads")
        scales = [s for s in (self.k_scales, self.v_scales) if s is not None]
        if len(scales) != (2 if k.dtype == E4M3 else 0):
            raise ValueError("e4m3 pages need k_scales and v_scales, others take none")
        if any(s.dtype != torch.float32 for s in scales):
            raise TypeError("the scales must be float32")
        if any(s.shape != k.shape[:2] for s in scales):
            raise ValueError("the scales must be [num_pages, kv_heads]")
        held = [k, self.v_pages, *scales]
        if any(t.device != k.device for t in held):
            raise ValueError("all tensors of a cache must be on one device")
        if any(not t.is_contiguous() or t.data_ptr() % 16 for t in held):
            raise ValueError("the tensors of a cache must be contiguous and 16-byte aligned")

    @classmethod
    def empty(cls, num_pages: int, kv_heads: int, head_dim: int = 128, page_size: int = 64, dtype: torch.dtype = E4M3,
              device="cuda") -> "PagedKVCache":
        """A cache of zeros."""
        shape = (num_pages, kv_heads, page_size, head_dim)
        pages = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(2)]
        if dtype != E4M3:
            return cls(*pages)
        return cls(*pages, *(torch.ones(shape[:2], dtype=torch.float32, device=device) for _ in range(2)))

    @property
    def quantized(self) -> bool:
        return self.k_scales is not None


def _check_table(cache, page_table, lengths, cu_new, device):
    for name, t, dims in (("page_table", page_table, 2), ("lengths", lengths, 1), ("cu_new", cu_new, 1)):
        if t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32")
        if t.dim() != dims:
            raise ValueError("page_table must be [sequences, pages], lengths [sequences], cu_new [sequences + 1]")
        if t.device != device:
            raise ValueError("all tensors must be on one device")
    b = page_table.shape[0]
    if lengths.shape[0] != b or cu_new.shape[0] != b + 1 or (b and not page_table.shape[1]):
        raise ValueError("page_table must be [sequences, pages], lengths [sequences], cu_new [sequences + 1]")
    if cache.k_pages.device != device:
        raise ValueError("all tensors must be on one device")


def _table(page_table):
    """The page table with contiguous rows."""
    return page_table if page_table.stride(1) == 1 or page_table.shape[1] <= 1 else page_table.contiguous()


def _check_rows(cache, name, x, heads=None):
    if x.dtype not in (torch.bfloat16, torch.float16) or not (cache.quantized or x.dtype == cache.k_pages.dtype):
        raise TypeError(f"{name} must be bfloat16 or float16, and of the pages' dtype unless that is float8_e4m3fn")
    if x.dim() != 3 or x.shape[2] != cache.k_pages.shape[3] or (heads is not None and x.shape[1] != heads):
        raise ValueError(f"{name} must be [tokens, heads, head_dim] with the cache's head_dim (and, keys and values, its heads)")
    if x.shape[0] > MAX_TOKENS:
        raise ValueError(f"at most {MAX_TOKENS} tokens")


def _check_no_gradients(cache, *tensors):
    tensors = [t for t in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales, *tensors) if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("the operators on the paged cache have no gradients: call them under torch.no_grad()")
    if _has_tangent(*tensors):
        raise RuntimeError("the operators on the paged cache have no forward-mode derivatives: tensors with a tangent are refused")


def paged_append(cache: PagedKVCache, key: torch.Tensor, value: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                 cu_new: torch.Tensor, inv_freq: Optional[torch.Tensor] = None, query: Optional[torch.Tensor] = None,
                 interleaved: bool = False) -> Optional[torch.Tensor]:
    """The keys and values of new tokens go into the cache; keys, and queries if given, are rotated by their positions first.

    Args:
        key, value: [tokens, kv_heads, head_dim] bf16 or fp16, the new tokens of all sequences one after the other
        page_table: [sequences, pages] int32, the pages of every sequence in the order of their tokens (entries behind its
            last page are not read)
        lengths: [sequences] int32, tokens of every sequence, the new ones included: the last new token of sequence b has
            position ``lengths[b] - 1``
        cu_new: [sequences + 1] int32, 0 and the running sum of the numbers of new tokens; a sequence may have none.  Rows of
            key and value behind ``cu_new[-1]`` are not read.
        inv_freq, interleaved: the rotation, as for ``qk_norm_rope``; without inv_freq nothing is rotated
        query: [tokens, heads, head_dim] of key's dtype, or None
    Returns:
        the rotated queries (rows that belong to no sequence: zeros), or None without ``query``.  No gradients: tensors that
        require one, the cache's and inv_freq among them, are refused outside ``torch.no_grad()``, those with a forward-mode
        tangent everywhere.

    The three index tensors stay on the device, and a captured call follows their contents.  A token whose position has no
    page (beyond the table's row, or an entry that is no page) is not written.  Elements of 8-bit pages are rounded from
    the rotated 32-bit values; the scale of a page and head is the smallest power of two that takes its largest
    magnitude into e4m3's range, and where new tokens raise the scale of a page, what it holds is rounded again.  An
    infinite value is held as the largest number an 8-bit page has.  Fewer than 2^30 tokens, and tokens / page_size +
    2 * sequences (with ``query`` tokens / 16 more) below 2^23.
    """
    out = _lib.host().paged_append(cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales, key, value, page_table, lengths,
                                   cu_new, inv_freq, query, interleaved)
    if out is not NotImplemented:
        return out
    # tensors that have to be copied first, none at all, or wrong ones
    hkv, d = cache.k_pages.shape[1], cache.k_pages.shape[3]
    _check_no_gradients(cache, key, value, query, inv_freq)
    for name, x in (("key", key), ("value", value)):
        _check_rows(cache, name, x, hkv)
    if value.shape != key.shape or value.dtype != key.dtype:
        raise ValueError("key and value must have one shape and dtype")
    if query is not None:
        _check_rows(cache, "query", query)
        if query.dtype != key.dtype or query.shape[0] != key.shape[0] or not 0 < query.shape[1] <= 65536:
            raise ValueError("query must have key's dtype and tokens")
    _check_table(cache, page_table, lengths, cu_new, key.device)
    if inv_freq is not None:
        _check_inv_freq(inv_freq, d)
    if any(t is not None and t.device != key.device for t in (value, query, inv_freq)):
        raise ValueError("all tensors must be on one device")
    if not key.is_cuda:
        raise RuntimeError("paged_append needs tensors on an AMD GPU (there is no CPU path)")
    tokens, b = key.shape[0], page_table.shape[0]
    out = None if query is None else torch.empty(query.shape, dtype=query.dtype, device=query.device)
    if not tokens:
        return out
    if not b:
        return out if out is None else out.zero_()
    key, value, query = _readable(key), _readable(value), None if query is None else _readable(query)
    page_table, lengths, cu_new = _table(page_table), lengths.contiguous(), cu_new.contiguous()
    inv_freq = None if inv_freq is None else inv_freq.contiguous()
    strides = (ctypes.c_int64 * 7)(*(_strides_of(query) if query is not None else (0, 0)), *_strides_of(key), *_strides_of(value),
                                   page_table.stride(0))
    with torch.cuda.device(key.device):
        _lib.check(_lib.load().moba_paged_append(
            E._ptr(key), E._ptr(value), E._ptr(query), E._ptr(out), E._ptr(cache.k_pages), E._ptr(cache.v_pages),
            E._ptr(cache.k_scales), E._ptr(cache.v_scales), E._ptr(page_table), E._ptr(lengths), E._ptr(cu_new),
            E._ptr(inv_freq), tokens, b, 0 if query is None else query.shape[1], hkv, d,
            0 if inv_freq is None else 2 * inv_freq.numel(), cache.k_pages.shape[2], cache.k_pages.shape[0],
            page_table.shape[1], strides, int(cache.quantized), int(interleaved), E._dtype_code(key),
            E._stream(key.device)), "moba_paged_append")
    # (autograd learns that they have changed, as after any operator that writes; an inference tensor keeps no such number)
    changed = (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)
    torch.autograd.graph.increment_version([t for t in changed if t is not None and not t.is_inference()])
    return out


def paged_attention(query: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, lengths: torch.Tensor, cu_new: torch.Tensor,
                    scaling: Optional[float] = None, max_new: Optional[int] = None) -> torch.Tensor:
    """Attention of new tokens over the cache that holds them: full causal attention, as in ``decode_attention``.

    Args:
        query: [tokens, heads, head_dim] bf16 or fp16, the new tokens of all sequences one after the other; heads a multiple
            of the cache's.  With 8-bit pages it may be either type.
        page_table, lengths, cu_new: as for ``paged_append``: row ``cu_new[b + 1] - 1`` of query is token ``lengths[b] - 1`` of
            sequence b, and every row sees its sequence's tokens up to itself
        scaling: softmax scale, ``head_dim ** -0.5`` by default
        max_new: the most new tokens that a sequence has, if that is known: a hint that spares the search for sequences
            with many.  Results do not depend on it; with one that is too small, sequences that have more than it says are slow,
            and in the precision of few rows
    Returns:
        [tokens, heads, head_dim] in query's dtype.  Rows that see no token (those of no sequence, of a sequence without
        pages), or whose scores are all minus infinity, are zeros; a page that the table names wrongly (no page of the pool) holds
        no tokens.  No gradients: a query or a cache that requires one is refused outside ``torch.no_grad()``, one with a
        forward-mode tangent everywhere.

    Scores, softmax statistics and sums are 32 bits.  A probability meets the values as the sum of two 16-bit elements (of the
    values' products: query's type with 16-bit pages, bf16 with 8-bit ones) where a sequence has few rows, new tokens times heads on a
    key/value head: up to 32, with 8-bit pages 64.  With more rows it is one element, rounded (fp16 queries on 8-bit pages: two of
    bf16), and values of 8-bit pages whose scale is no power of two are rounded to bf16.  At most 2^24 - 1 tokens, fewer than 2^31
    tokens times heads, and some million sequences times key/value heads.
    """
    out = _lib.host().paged_attention(cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales, query, page_table, lengths,
                                      cu_new, scaling, max_new)
    if out is not NotImplemented:
        return out
    # tensors that have to be copied first, none at all, or wrong ones
    _check_no_gradients(cache, query)
    _check_rows(cache, "query", query)
    hkv, d = cache.k_pages.shape[1], cache.k_pages.shape[3]
    tokens, heads = query.shape[:2]
    if tokens >= 1 << 24 or tokens * heads >= 1 << 31:
        raise ValueError("at most 2^24 - 1 tokens, and fewer than 2^31 rows")
    if not heads or heads % hkv:
        raise ValueError("the number of query heads must be a multiple of the number of key/value heads")
    if max_new is not None and max_new < 0:
        raise ValueError("max_new must not be negative")
    _check_table(cache, page_table, lengths, cu_new, query.device)
    if not query.is_cuda:
        raise RuntimeError("paged_attention needs tensors on an AMD GPU (there is no CPU path)")
    b = page_table.shape[0]
    out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    if not tokens or not b:
        return out.zero_()
    lib = _lib.load()
    if not _addressable(query):
        query = E._aligned(query)
    page_table, lengths, cu_new = _table(page_table), lengths.contiguous(), cu_new.contiguous()
    strides = (ctypes.c_int64 * 3)(*E._row_strides(query), page_table.stride(0))
    hint = -1 if max_new is None else min(max_new, tokens)
    with torch.cuda.device(query.device):
        space = torch.empty(lib.moba_paged_attention_workspace_bytes(tokens, b, heads, hkv, d, int(cache.quantized), hint),
                            dtype=torch.uint8, device=query.device)
        _lib.check(lib.moba_paged_attention(
            E._ptr(query), E._ptr(out), E._ptr(cache.k_pages), E._ptr(cache.v_pages), E._ptr(cache.k_scales),
            E._ptr(cache.v_scales), E._ptr(page_table), E._ptr(lengths), E._ptr(cu_new), E._ptr(space), tokens, b, heads, hkv,
            d, cache.k_pages.shape[2], cache.k_pages.shape[0], page_table.shape[1], hint, strides, int(cache.quantized),
            float(scaling) if scaling is not None else d ** -0.5, E._dtype_code(query), E._stream(query.device)),
            "moba_paged_attention")
    return out


def _addressable(query):
    ts, hs = E._row_strides(query)
    return query.stride(2) == 1 and ts % 8 == 0 and hs % 8 == 0 and query.data_ptr() % 16 == 0
