"""Pages and step tables from request lengths, made on the device (HIP).

The reference gives every request a fixed range of pages and makes a step's index arrays on the host
(aspire/models/sparse_draft_runner.py:240-250, aspire/backends/host_plan.py). Here requests share a pool whose pages they take and
give back as their lengths change, and the arrays of a step come from lengths that are already on the GPU (after a
verification, say), without a wait for the host, in two launches that a graph can hold:

* ``PagePool.resize(lengths)``: every request holds the pages of its length;
* ``StepTables.build(block_table, cached, new_tokens, parents)``: running counts of tokens and pages, the page list, last
  page lengths, and for each new token its position, its slot in the cache and, in a drafted tree, the bits of its
  ancestors. They are what ``mylib::update_kv_padded``, ``RotaryEmbedding.append`` (``positions``), ``tree_attention`` and
  ``compact_accepted`` (``slots``) take.
"""

from __future__ import annotations

import struct

import torch

from aspire_amd import _lib

MAX_REQUESTS = 4096
MAX_TREE_WORDS = 64

_RESIZE = struct.Struct("6P4i")          # aspire_page_resize_args
_TABLES = struct.Struct("PqPPP8i8P")     # aspire_step_tables_args


def _counts(t: torch.Tensor, length: int | None, index: int, what: str, name: str) -> torch.Tensor:
    """An int32 vector on device ``index``, in one piece."""
    if t.dtype is torch.int32 and t.get_device() == index and t.dim() == 1 and t.is_contiguous() \
            and (length is None or t.shape[0] == length):
        return t
    _lib.require_cuda(t, what=what)
    if t.dim() != 1 or t.dtype not in (torch.int32, torch.int64) or t.get_device() != index or (length is not None and t.shape[0] != length):
        raise ValueError(f"{what}: {name} must be int32 [{'requests' if length is None else length}] on cuda:{index}")
    return _lib.indices(t)


class PagePool:
    """``num_pages`` pages shared by up to ``max_requests`` requests (at most 4,096) of at most ``max_pages`` pages each.

    ``block_table [max_requests, max_pages]`` holds each request's pages (-1 behind its ``held`` ones), ``free`` the pages of
    no request as a stack of ``free_count`` entries, ``shortage`` what the last ``resize`` could not give. All are int32 device
    tensors."""

    def __init__(self, num_pages: int, page_size: int, max_requests: int, max_pages: int, device="cuda"):
        if num_pages < 1 or page_size < 1 or max_pages < 1 or not 1 <= max_requests <= MAX_REQUESTS:
            raise ValueError(f"PagePool: sizes must be positive, max_requests at most {MAX_REQUESTS}")
        if max_requests * max_pages >= 1 << 31 or num_pages >= 1 << 31:
            raise ValueError("PagePool: max_requests * max_pages and num_pages must be below 2^31")
        self.num_pages, self.page_size, self.max_requests, self.max_pages = num_pages, page_size, max_requests, max_pages
        i32 = dict(dtype=torch.int32, device=device)
        self.block_table = torch.full((max_requests, max_pages), -1, **i32)
        self.held = torch.zeros(max_requests, **i32)
        self.free = torch.arange(num_pages - 1, -1, -1, **i32)  # page 0 is taken first
        self.free_count = torch.full((1,), num_pages, **i32)
        self.shortage = torch.zeros(max_requests, **i32)
        self.device, self._index = self.held.device, self.held.get_device()

    def resize(self, lengths: torch.Tensor) -> torch.Tensor:
        """Give request ``b`` the pages of ``lengths[b]`` tokens, ``lengths`` int32 ``[max_requests]``: 0 gives all of its pages
        back, a negative length leaves it as it is. Requests first give back what they hold above that (their last pages), then
        take what they lack in row order. From the first one on that lacks more pages than are left, or more than
        ``max_pages``, none takes any: ``shortage`` (returned) has what each of them lacks, 0 for the others."""
        what = "PagePool.resize"
        if self._index < 0:
            _lib.require_cuda(self.held, what=what)
        lengths = _counts(lengths, self.max_requests, self._index, what, "lengths")
        args = _RESIZE.pack(self.block_table.data_ptr(), self.held.data_ptr(), self.free.data_ptr(), self.free_count.data_ptr(),
                            self.shortage.data_ptr(), lengths.data_ptr(), self.max_requests, self.max_pages, self.num_pages,
                            self.page_size)
        _lib.launch(_lib.lib().aspire_page_resize, self._index, what, args)
        return self.shortage


class StepTables:
    """A step's device arrays at fixed addresses, for up to ``max_rows`` requests with ``max_tokens`` new tokens and
    ``max_entries`` pages in all; ``tree_words`` 64-bit words of ancestors a token (0: no masks).

    ``qo_indptr``, ``kv_indptr`` int32 ``[max_rows + 1]``; ``kv_indices`` int32 ``[max_entries]``; ``last_page_len`` int32
    ``[max_rows]``; ``positions`` int32, ``slots`` int64 ``[max_tokens]``; ``masks`` int64 ``[max_tokens, tree_words]`` (None
    without); ``totals`` int64 ``[3]``: the tokens and pages that were asked for, and the first row that was left out."""

    def __init__(self, max_rows: int, max_tokens: int, max_entries: int, page_size: int, device="cuda", tree_words: int = 0):
        if not 0 <= max_rows <= MAX_REQUESTS or not 0 <= tree_words <= MAX_TREE_WORDS or page_size < 1 \
                or not 0 <= max_tokens <= 1 << 30 or not 0 <= max_entries <= 1 << 30:
            raise ValueError(f"StepTables: at most {MAX_REQUESTS} rows, {MAX_TREE_WORDS} tree words, 2^30 tokens and entries, "
                             "a positive page size")
        self.max_rows, self.max_tokens, self.max_entries = max_rows, max_tokens, max_entries
        self.page_size, self.tree_words = page_size, tree_words
        i32, i64 = dict(dtype=torch.int32, device=device), dict(dtype=torch.int64, device=device)
        self.qo_indptr, self.kv_indptr = torch.zeros(max_rows + 1, **i32), torch.zeros(max_rows + 1, **i32)
        self.kv_indices = torch.full((max_entries,), -1, **i32)
        self.last_page_len = torch.zeros(max_rows, **i32)
        self.positions, self.slots = torch.full((max_tokens,), -1, **i32), torch.full((max_tokens,), -1, **i64)
        self.masks = torch.zeros(max_tokens, tree_words, **i64) if tree_words else None
        self.totals = torch.zeros(3, **i64)
        self.device, self._index = self.totals.device, self.totals.get_device()
        # the tensors, not their addresses: a copy of the object has its own
        self._outputs = (self.qo_indptr, self.kv_indptr, self.kv_indices, self.last_page_len, self.positions, self.slots, self.masks, self.totals)

    def build(self, block_table: torch.Tensor, cached: torch.Tensor, new_tokens: torch.Tensor,
              parents: torch.Tensor | None = None) -> "StepTables":
        """Row ``b`` of ``block_table`` ``[>= rows, width]`` int32 holds the pages of ``cached[b]`` tokens and of ``new_tokens[b]``
        new ones behind them (int32 ``[rows]``). ``parents`` int32 ``[max_tokens]`` (None: every row is a chain) gives, for each
        new token of a tree, the index in its row of the token that it continues, -1 for a root: positions are then
        ``cached + depth``. Tokens behind the last row get position and slot -1 and no bits; a page that the table does not have
        is -1. Rows without new tokens list no pages. From the first row on that does not fit (``max_tokens``,
        ``max_entries``, or more than ``64 * tree_words`` tokens, with ``parents`` and no masks more than 4,096) no row has
        tokens or pages."""
        what = "StepTables.build"
        index = self._index
        if index < 0:
            _lib.require_cuda(self.totals, what=what)
        cached = _counts(cached, None, index, what, "cached")
        rows = cached.shape[0]
        new_tokens = _counts(new_tokens, rows, index, what, "new_tokens")
        if rows > self.max_rows:
            raise ValueError(f"{what}: {rows} rows, but the tables hold {self.max_rows}")
        shape, strides = block_table.shape, block_table.stride()
        if len(shape) != 2 or block_table.dtype is not torch.int32 or shape[0] < rows or block_table.get_device() != index \
                or (shape[1] > 1 and strides[1] != 1):
            _lib.require_cuda(block_table, what=what)
            raise ValueError(f"{what}: block_table must be int32 [at least {rows}, pages] on {self.device} with contiguous rows")
        at = 0
        if parents is not None:
            parents = _counts(parents, None, index, what, "parents")
            if parents.shape[0] < self.max_tokens:
                raise ValueError(f"{what}: parents needs {self.max_tokens} entries")
            at = parents.data_ptr()
        args = _TABLES.pack(block_table.data_ptr(), strides[0], cached.data_ptr(), new_tokens.data_ptr(), at, rows, shape[1],
                            self.max_rows, self.max_tokens, self.max_entries, self.page_size, self.tree_words, 0,
                            *[0 if t is None else t.data_ptr() for t in self._outputs])
        _lib.launch(_lib.lib().aspire_step_tables, index, what, args)
        return self


__all__ = ["MAX_REQUESTS", "MAX_TREE_WORDS", "PagePool", "StepTables"]
