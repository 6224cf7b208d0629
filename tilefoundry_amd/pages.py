"""The pages of a cache: who has which, shared, copied before a write, freed and compacted.

``Pages`` keeps a page table and how many of its entries name each page, over pools such as the
engines' key and value caches (a page holds 16 positions).  All of it stays on the device:

    cache = Pages([k_pool, v_pool], rows=32, max_pages=256)
    cache.take(lengths, 1)                       # pages for the next position of every row
    lengths = cache.fork(parents, lengths)       # rows continue other rows, sharing their pages
    cache.free(finished)                         # rows give their pages back
    lengths = cache.keep(lengths, path, counts)  # accepted drafted positions move together
    live = cache.compact()                       # pages in use get the lowest numbers

Forked rows share pages; ``take`` copies a shared page before a row writes into it, so call it for
every position before the position is written.  ``lengths`` (int32 ``[rows]``, positions in use)
belong to the caller, who appends.  The exact definitions are declared in
``include/tf_search.h``.

Every call runs on the current stream of the pools' device and can be captured into a HIP
graph.  The calls on one ``Pages`` change one state: keep them, and what reads the pools, in one
stream's order.  No gradients.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import lib, ptr
from .mx4 import INT32, _settle, check_apart, check_device, check_input, launch

PAGE = _lib.PAGE_SIZE
MAX_ROWS = _lib.PAGES_MAX_ROWS
BOOL = (torch.bool, torch.uint8)


class Pages:
    """See the module docstring.

    *pools*: tensors ``[pages, heads, 16, dim]``, or ``[layers, pages, heads, 16, dim]``,
    contiguous, rows of a multiple of 16 bytes, all of one number of pages, no two in the same
    memory; they are kept.
    *table* int32 ``[rows, max_pages]`` (-1: no page) and *refs* int32 ``[pages]`` are used in place if given;
    without *table* it starts empty, without *refs* the table's entries are counted."""

    def __init__(self, pools, *, rows: int | None = None, max_pages: int | None = None,
                 table: torch.Tensor | None = None, refs: torch.Tensor | None = None):
        self.pools = list(pools)
        if not self.pools:
            raise ValueError("Pages: no pools")
        parts = []
        for t in self.pools:
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"Pages: expected tensors, got {type(t).__name__}")
            check_input(t, "Pages", (t.dtype,))
            if t.dim() not in (4, 5) or t.shape[-2] != PAGE or not t.is_contiguous():
                raise ValueError(f"Pages: contiguous pools [pages, heads, {PAGE}, dim], with or "
                                 f"without layers before, got {tuple(t.shape)}")
            parts += list(t) if t.dim() == 5 else [t]
        if not parts:
            raise ValueError("Pages: pools without layers")
        check_apart(self.pools, "Pages")
        self.device, self.num_pages = parts[0].device, parts[0].shape[0]
        check_device(self.device, *parts)
        entries = []
        for t in parts:
            row = t.shape[3] * t.element_size()
            if t.shape[0] != self.num_pages or t.numel() == 0:
                raise ValueError(f"Pages: pools of one number of pages, got {tuple(t.shape)} and "
                                 f"{self.num_pages} pages")
            if row % 16 or row >= 1 << 27 or t.data_ptr() % 16 or t.shape[1] > 65535:
                raise ValueError(f"Pages: rows of a multiple of 16 bytes, got {t.shape[3]} of "
                                 f"{t.dtype}")
            entries.append(_lib.TfdPool(ptr(t), t.shape[1] * PAGE * row, t.shape[1], row))
        if self.num_pages > 1 << 28 or len(entries) > 65535:
            raise ValueError(f"Pages: {self.num_pages} pages of {len(entries)} pools are too many")
        if table is None:
            if rows is None or max_pages is None:
                raise ValueError("Pages: rows and max_pages, or a table")
            if not 1 <= rows <= MAX_ROWS or not 1 <= max_pages <= 1 << 20:
                raise ValueError(f"Pages: 1 to {MAX_ROWS} rows of 1 to 2^20 pages, got {rows} of "
                                 f"{max_pages}")
            table = torch.full((rows, max_pages), -1, dtype=torch.int32, device=self.device)
        check_input(table, "table", INT32)
        if table.dim() != 2 or not table.is_contiguous() or \
                not 1 <= table.shape[0] <= MAX_ROWS or not 1 <= table.shape[1] <= 1 << 20 or \
                (rows is not None and rows != table.shape[0]) or \
                (max_pages is not None and max_pages != table.shape[1]):
            raise ValueError(f"Pages: a contiguous table of 1 to {MAX_ROWS} rows of 1 to 2^20 "
                             f"pages, got {tuple(table.shape)}")
        check_device(self.device, table)
        if refs is None:
            used = table.flatten().long()
            used = used[(used >= 0) & (used < self.num_pages)]
            refs = torch.zeros(self.num_pages, dtype=torch.int32, device=self.device)
            refs.scatter_add_(0, used, torch.ones_like(used, dtype=torch.int32))
        check_input(refs, "refs", INT32)
        if refs.shape != (self.num_pages,) or not refs.is_contiguous():
            raise ValueError(f"Pages: refs must be [{self.num_pages}], got {tuple(refs.shape)}")
        check_device(self.device, refs)
        self.table, self.refs = table, refs
        self.rows, self.max_pages = table.shape
        self._scratch = torch.zeros(_lib.pages_scratch(self.rows, self.max_pages, self.num_pages),
                                    dtype=torch.int32, device=self.device)
        raw = bytearray(bytes((_lib.TfdPool * len(entries))(*entries)))
        self._entries = torch.frombuffer(raw, dtype=torch.uint8).to(self.device)
        self.err = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.index = self.err.get_device()
        self._args = _lib.TfdPages(
            ptr(self._entries), len(entries), max(e.page_bytes for e in entries),
            ptr(table), ptr(refs), self.rows, self.max_pages, self.num_pages, ptr(self._scratch),
            ptr(self.err))
        self._at = ctypes.addressof(self._args)
        _settle(self.device)

    def _ints(self, x, what: str, shape):
        check_input(x, what, INT32)
        if x.shape != shape:
            raise ValueError(f"{what} must be {list(shape)}, got {tuple(x.shape)}")
        if x.get_device() != self.index:
            raise ValueError(f"Pages: {what} on {x.device}, pools on {self.device}")
        return x.contiguous()

    def fork(self, parents: torch.Tensor, lengths: torch.Tensor) -> torch.Tensor:
        """Row r becomes what row ``parents[r]`` was, sharing its pages; -> the new lengths.
        -1 empties a row; a row that is its own parent keeps its entries, reserved ones too.
        What no row has any more is free.  A parent outside the rows leaves its row as it is
        (``check_errors``)."""
        parents = self._ints(parents, "parents", (self.rows,))
        lengths = self._ints(lengths, "lengths", (self.rows,))
        out = torch.empty_like(lengths)
        launch(self.index, lib().tfd_pages_fork, self._at, ptr(parents), 0, ptr(lengths),
               ptr(out))
        return out

    def free(self, which: torch.Tensor) -> None:
        """The rows with which[r] (bool ``[rows]``) give their pages back."""
        check_input(which, "which", BOOL)
        if which.shape != (self.rows,):
            raise ValueError(f"which must be [{self.rows}], got {tuple(which.shape)}")
        if which.get_device() != self.index:
            raise ValueError(f"Pages: which on {which.device}, pools on {self.device}")
        which = which.contiguous()
        launch(self.index, lib().tfd_pages_fork, self._at, 0, ptr(which), 0, 0)

    def take(self, lengths: torch.Tensor, n) -> None:
        """Pages of their own for positions ``lengths[r] .. lengths[r] + n - 1`` of every row; n: a
        number, or int32 ``[rows]``.  New pages are the free ones of lowest number, in the order of
        rows and positions; a shared page's positions below ``lengths[r]`` are copied along.
        Rows for which no page is left get -1 (``check_errors``)."""
        lengths = self._ints(lengths, "lengths", (self.rows,))
        counts, one = None, 0
        if isinstance(n, torch.Tensor):
            counts = self._ints(n, "n", (self.rows,))
        else:
            one = int(n)
            if one != n or not 0 <= one < 1 << 31:
                raise ValueError(f"n must be a number of positions, got {n}")
        launch(self.index, lib().tfd_pages_take, self._at, ptr(lengths), ptr(counts), one)

    def copy(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Page ``dst[i]`` of every pool becomes page ``src[i]`` (int32 ``[n]``).  No page may be in
        both lists or twice in *dst*; a pair with a number outside the pools is left out
        (``check_errors``).  Table and references stay as they are."""
        check_input(src, "src", INT32)
        if src.dim() != 1:
            raise ValueError(f"src must be [n], got {tuple(src.shape)}")
        src, dst = self._ints(src, "src", src.shape), self._ints(dst, "dst", src.shape)
        launch(self.index, lib().tfd_pages_copy, self._at, ptr(src), ptr(dst), src.numel())

    def keep(self, lengths: torch.Tensor, path: torch.Tensor, counts: torch.Tensor
             ) -> torch.Tensor:
        """Positions ``lengths[r] + path[r, i]`` move to ``lengths[r] + i`` for i < ``counts[r]``,
        in every pool; -> ``lengths + counts``.  path (int32 ``[rows, nodes]``) rises along a row;
        a row where it does not keeps its positions and length (``check_errors``)."""
        check_input(path, "path", INT32)
        if path.dim() != 2 or path.shape[0] != self.rows or path.shape[1] < 1:
            raise ValueError(f"path must be [{self.rows}, nodes], got {tuple(path.shape)}")
        path = self._ints(path, "path", path.shape)
        lengths = self._ints(lengths, "lengths", (self.rows,))
        counts = self._ints(counts, "counts", (self.rows,))
        out = torch.empty_like(lengths)
        launch(self.index, lib().tfd_pages_keep, self._at, ptr(lengths), ptr(path), ptr(counts),
               path.shape[1], ptr(out))
        return out

    def compact(self) -> torch.Tensor:
        """The pages in use move to the numbers 0 .. live - 1 (those behind, in rising order, to
        the free ones before, in rising order) -> live, int32 on the device."""
        live = self.refs.new_empty(())
        launch(self.index, lib().tfd_pages_compact, self._at, ptr(live))
        return live

    def check_errors(self) -> None:
        """Raises if a call since the last check met something out of range or found no page
        (waits for the device)."""
        torch.cuda.synchronize(self.device)
        e = int(self.err.item())
        if e:
            self.err.zero_()
            torch.cuda.synchronize(self.device)
            names = [n for bit, n in (
                (_lib.ERR_POS_RANGE, "a position outside the table"),
                (_lib.ERR_PAGE_RANGE, "a page outside the pools"),
                (_lib.ERR_ROW_RANGE, "a parent, path or count outside its range"),
                (_lib.ERR_NO_PAGES, "no free page")) if e & bit]
            raise RuntimeError(f"Pages: {', '.join(names)}")
