"""Pages for new tokens from a pool and back, on MI355X: the page table, the lengths and the places of the new tokens that the paged
cache's operators and ``qk_norm_rope`` take, from the sequences' lengths on the device.  (The reference's cache is transformers'
contiguous one, moba/wrapper.py:76-82.)"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Tuple

import torch

from . import _lib
from .paged import PAGE_SIZES, _plain, _table, _taken

MAX_SEQUENCES = 8192   # of a call
MAX_ROWS = (1 << 30) - 1
MAX_ENTRIES = (1 << 31) - 1   # of a page table, or a pool


@dataclass(frozen=True, eq=False)
class PagePool:
    """The pages that nobody holds, as a stack.

    free_pages: [num_pages] int32, as many as the cache has; the first ``free_count`` of them are free, the last of these is given
        out first
    free_count: [1] int32
    page_size: tokens of a page, the cache's
    """

    free_pages: torch.Tensor
    free_count: torch.Tensor
    page_size: int

    def __post_init__(self):
        for name, t in (("free_pages", self.free_pages), ("free_count", self.free_count)):
            if t.dtype != torch.int32:
                raise TypeError(f"{name} must be int32")
            if t.dim() != 1 or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous, of one dimension")
        if not self.free_pages.numel() or self.free_count.numel() != 1:
            raise ValueError("there must be pages, and one free_count")
        if self.free_pages.numel() > MAX_ENTRIES:
            raise ValueError("fewer than 2^31 pages")
        if self.free_count.device != self.free_pages.device:
            raise ValueError("all tensors of a pool must be on one device")
        if self.page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}")

    @classmethod
    def full(cls, num_pages: int, page_size: int = 64, device="cuda") -> "PagePool":
        """A pool in which all pages are free; page 0 is given out first."""
        if num_pages <= 0:
            raise ValueError("there must be pages")
        pages = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=device)
        return cls(pages, torch.full((1,), num_pages, dtype=torch.int32, device=device), page_size)


def _check(pool, page_table, lengths, name, asked):
    device = pool.free_pages.device
    for what, t, dims in (("page_table", page_table, 2), ("lengths", lengths, 1), (name, asked, 1)):
        if t.dtype != torch.int32:
            raise TypeError(f"{what} must be int32")
        if t.dim() != dims:
            raise ValueError(f"page_table must be [sequences, pages], lengths and {name} [sequences]")
        if t.device != device:
            raise ValueError("all tensors must be on one device")
    b = lengths.shape[0]
    if page_table.shape[0] != b or asked.shape[0] != b or (b and not page_table.shape[1]):
        raise ValueError(f"page_table must be [sequences, pages], lengths and {name} [sequences]")
    if b > MAX_SEQUENCES:
        raise ValueError(f"at most {MAX_SEQUENCES} sequences")
    if page_table.numel() > MAX_ENTRIES:
        raise ValueError("page_table must have fewer than 2^31 entries")
    # (they are written)
    if not lengths.is_contiguous() or _table(page_table) is not page_table or (b > 1 and page_table.stride(0) < page_table.shape[1]):
        raise ValueError("lengths and the rows of page_table must be contiguous and apart from each other")


def paged_reserve(pool: PagePool, page_table: torch.Tensor, lengths: torch.Tensor, new_tokens: torch.Tensor,
                  rows: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Pages for the next tokens of every sequence, and where each of these tokens belongs.

    Args:
        pool: its ``free_count`` goes down
        page_table: [sequences, pages] int32, the pages of every sequence in the order of their tokens; the new ones are written
            behind those that hold its ``lengths[b]`` tokens
        lengths: [sequences] int32, the tokens that every sequence has; goes up by the new ones
        new_tokens: [sequences] int32, how many more are wanted (negative: none)
        rows: packed rows that there are for the new tokens of all sequences
    Returns:
        (cu_new, owners, positions, slots).  cu_new [sequences + 1] int32: 0 and the running sum of the tokens that were given, which
        are the packed rows ``cu_new[b]`` .. ``cu_new[b + 1] - 1``.  Of each of the ``rows``: the sequence, the position in it
        (int32, both), and the slot in the cache, ``page * page_size`` + place in the page (int64); -1, 0 and -1 behind the
        last, and slot -1 where the table names no page of the pool.

    A sequence gets all that it wants or nothing (its row of the table, its length and the pool stay as they are, and it has no
    rows): nothing if its tokens do not fit its row of the table; if they, with those that the others before it want (those that do
    not fit aside), are more than ``rows``; or if it needs more pages and they, with those that the others before it need, are more
    than the pool has.  The index tensors stay on the device: a captured call follows them.  Calls that share a pool or a table have to
    run one after the other (one stream, or streams that wait for each other).  At most 8192 sequences, and fewer than 2^31 entries of the
    table.
    """
    out = _lib.host().paged_reserve(pool.free_pages, pool.free_count, page_table, lengths, new_tokens, rows, pool.page_size)
    if out is not NotImplemented:
        return out
    _check(pool, page_table, lengths, "new_tokens", new_tokens)
    if not 0 <= rows <= MAX_ROWS:
        raise ValueError(f"rows must be 0 to {MAX_ROWS}")
    if not lengths.is_cuda:
        raise RuntimeError("paged_reserve needs tensors on an AMD GPU (there is no CPU path)")
    if not lengths.shape[0]:
        none = torch.full((rows,), -1, dtype=torch.int32, device=lengths.device)
        return torch.zeros(1, dtype=torch.int32, device=lengths.device), none, torch.zeros_like(none), none.long()
    tensors = (pool.free_pages, pool.free_count, page_table, lengths, new_tokens.contiguous())
    return _taken(_lib.host().paged_reserve(*map(_plain, tensors), rows, pool.page_size), "paged_reserve")


def paged_release(pool: PagePool, page_table: torch.Tensor, lengths: torch.Tensor, keep: torch.Tensor) -> None:
    """Sequences are cut to their first tokens, and the pages behind these go back to the pool.

    Args:
        pool: its ``free_count`` goes up
        page_table: [sequences, pages] int32; the entries of the pages that go become -1
        lengths: [sequences] int32, the tokens that every sequence has; becomes ``keep`` where that is less
        keep: [sequences] int32: 0 (or less) for a sequence that has ended, fewer than it has after drafted tokens were rejected

    Undoes ``paged_reserve``: the pages go back so that they come out again in the order in which they came.  Entries that name no
    page of the pool do not go back.  A page that several sequences share would go back with each of them: keep the tokens that
    are shared, and release their pages once, with the sequence that they belong to.  Limits are those of ``paged_reserve``.
    """
    if _lib.host().paged_release(pool.free_pages, pool.free_count, page_table, lengths, keep, pool.page_size) is not NotImplemented:
        return
    _check(pool, page_table, lengths, "keep", keep)
    if not lengths.is_cuda:
        raise RuntimeError("paged_release needs tensors on an AMD GPU (there is no CPU path)")
    if lengths.shape[0]:
        tensors = (pool.free_pages, pool.free_count, page_table, lengths, keep.contiguous())
        _taken(_lib.host().paged_release(*map(_plain, tensors), pool.page_size), "paged_release")
