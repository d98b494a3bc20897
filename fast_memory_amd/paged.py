"""Local keys and values in pages: the cache a server keeps its recent tokens in, for many sequences, and the attention
of new tokens over it.  The reference's local attention (memory.py:302-304) reads dense tensors of one forward and
keeps nothing; what leaves this cache at the front (:meth:`PagedCache.drop`) is what a :class:`Memory` takes over."""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib, ops
from .ops import ScoreTerms

REFUSALS = {1: "the pool has fewer free pages than the call needs",
            2: "a row would outgrow its table of pages",
            3: "cu is not ascending from 0 to at most T, or a fork names a row that holds tokens, itself, a row outside "
               "the cache or a row that is forked into"}


class PagedCache:
    """Keys and values of ``n_rows`` sequences in pages of ``page_size`` tokens (a power of two), out of a pool of
    ``n_pages`` pages ``k_pages, v_pages [n_pages, n_heads, page_size, d]``.  ``max_tokens``: the most a row may hold
    (the whole pool without it); :meth:`attend` takes rows of up to 2^24.

    All bookkeeping is one int32 tensor, ``book``, on the device; ``length [n_rows]``, ``refs [n_pages]`` (rows that
    hold a page, 0 = free) and ``table [n_rows, width]`` are views of it.  No call reads anything back, so all of them
    record into a graph; a request that cannot be met (:data:`REFUSALS`) changes nothing and is counted, and
    :meth:`check`, called wherever waiting costs nothing, raises.  The calls of one cache follow each other on one
    stream, or are ordered by events.  ``snapshot`` / ``restore`` take the bookkeeping back (speculative tokens that
    were not accepted), but not the count of refused calls; a page that a call after the snapshot freed, or moved, may
    hold other rows by then.
    """

    def __init__(self, n_rows: int, n_pages: int, page_size: int, n_heads: int, d: int,
                 dtype: torch.dtype = torch.bfloat16, device="cuda", max_tokens: Optional[int] = None):
        if int(page_size) < 1:
            raise ValueError(f"PagedCache: page_size={page_size}")
        width = n_pages if max_tokens is None else -(-int(max_tokens) // int(page_size))
        words = _lib.load().fm_cache_book_ints(int(n_pages), int(n_rows), int(width))
        if words == 0:
            raise ValueError(f"PagedCache: n_rows={n_rows} n_pages={n_pages} max_tokens={max_tokens}")
        book = torch.zeros(words, dtype=torch.int32, device=device)
        shape = (int(n_pages), int(n_heads), int(page_size), int(d))
        self._init(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device), book, n_rows)
        self.table.fill_(-1)

    @classmethod
    def over(cls, k_pages: torch.Tensor, v_pages: torch.Tensor, book: torch.Tensor, n_rows: int) -> "PagedCache":
        """A cache over tensors the caller has already (a pool that is shared, a restored checkpoint)."""
        self = cls.__new__(cls)
        self._init(k_pages, v_pages, book, n_rows)
        return self

    def _init(self, k_pages, v_pages, book, n_rows):
        ops._dev(k_pages, v_pages, book)
        ops._same_device(k_pages, v_pages, book)
        n_pages, H, P, d = k_pages.shape
        R, meta = int(n_rows), _lib.FM_CACHE_META_INTS
        ops._dt(k_pages)
        if k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype or book.dtype != torch.int32 or book.dim() != 1:
            raise ValueError("PagedCache: k_pages and v_pages are alike and book is a flat int32 tensor")
        if P < 1 or P & (P - 1) or P > _lib.FM_CACHE_MAX_PAGE:
            raise ValueError(f"PagedCache: page size {P} is no power of two up to {_lib.FM_CACHE_MAX_PAGE}")
        words = book.numel() - meta - R - n_pages
        if R < 1 or words < R or words % R:
            raise ValueError(f"PagedCache: {book.numel()} words of bookkeeping do not fit {R} rows and {n_pages} pages")
        self.k_pages, self.v_pages, self.book = k_pages, v_pages, book
        self.n_rows, self.n_pages, self.n_heads, self.page_size, self.d = R, n_pages, H, P, d
        self.width = words // R
        self.length = book[meta:meta + R]
        self.refs = book[meta + R:meta + R + n_pages]
        self.table = book[meta + R + n_pages:].view(R, self.width)
        self._ws_bytes = int(_lib.load().fm_cache_workspace(n_pages, R))

    # ------------------------------------------------------------------ rows come, are forked, and leave
    def append(self, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor) -> None:
        """Row r receives tokens ``cu[r] .. cu[r+1]`` of ``k, v [T, n_heads, d]`` at its end; ``cu [n_rows+1]`` int32.
        The cache holds values: no gradient reaches ``k`` or ``v`` through it."""
        ops.cache_append_(self, k, v, cu)

    def fork(self, src: torch.Tensor) -> None:
        """Row r, which is empty, becomes a copy of row ``src[r]`` (``src [n_rows]`` int32, negative: left alone): whole
        pages are shared, a last partial page is copied."""
        ops.cache_fork_(self, src)

    def drop(self, pages: torch.Tensor) -> None:
        """The first ``pages[r]`` whole pages of row r leave it (``pages [n_rows]`` int32; at least as many as it has:
        the row is empty); pages that no row holds any more are free."""
        ops.cache_drop_(self, pages)

    def free(self, rows: torch.Tensor) -> None:
        """Rows where ``rows [n_rows]`` is true give up all they hold."""
        if rows.shape != (self.n_rows,):
            raise ValueError(f"PagedCache.free: a truth value for each of {self.n_rows} rows")
        ops.cache_drop_(self, rows.to(torch.bool).to(torch.int32) * (1 << 30))

    def compact(self) -> None:
        """The used pages move to the front of the pool (as few as that takes); its tail is free afterwards."""
        ops.cache_compact_(self)

    def snapshot(self) -> torch.Tensor:
        return self.book.clone()

    def restore(self, book: torch.Tensor) -> None:
        if book.shape != self.book.shape:
            raise ValueError(f"PagedCache.restore: {tuple(book.shape)} is no snapshot of this cache ({tuple(self.book.shape)})")
        self.book[2:].copy_(book[2:])  # (what check() counts stays: a refused call stays refused)

    def check(self) -> None:
        """Raises when a call since the last check was refused (synchronises)."""
        refused, why = self.book[:2].tolist()
        if refused:
            self.book[:2].zero_()
            raise RuntimeError(f"PagedCache: {refused} call(s) refused; the first because {REFUSALS.get(why, why)}")

    # ------------------------------------------------------------------ attention
    def attend(self, q: torch.Tensor, cu: torch.Tensor, sm_scale: float, terms: Optional[ScoreTerms] = None,
               max_new: int = 0):
        """The attention of the new tokens ``q [T, n_query_heads, d]``, tokens ``cu[r] .. cu[r+1]`` being the last ones
        of row r (:meth:`append` them first), over their rows: ``(out [T, n_query_heads, d], lse [T, n_query_heads]
        fp32)``, to be merged with a memory's by ``merge``.  Query head ``h*G + g`` reads KV head h.  ``terms``: cap,
        slopes, and ``prefix [n_rows]`` (the first keys of a row that all its new tokens see); a row is a document of
        its own.  ``max_new``: the largest number of new tokens of a row where the caller knows it (it only shapes the
        launch).  There is no backward: a ``q`` that asks for gradients is refused."""
        return ops.paged_attn_fwd(q, self, cu, sm_scale, terms, max_new)
