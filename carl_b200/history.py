"""Paged history: records of ragged sequences in pages that forked sequences share.

An env overwrites its output buffers with every step; a history keeps what they
held.  A row is one sequence (an agent's episode, a beam's lineage), a record any
fixed shape (an observation row, an action).  Episodes end at different times and
lineages share their past, so records lie in pages of `page_len` that a table
assigns to rows; a page is shared until a row writes to it::

    history = PagedHistory.empty(n_rows, row_pages, n_pages, page_len, (obs_dim,))
    torch.cuda.current_stream().wait_stream(torch.cuda.ExternalStream(env.stream))
    history.append(env.get_obs().view(n_rows, obs_dim))     # one record per row
    history.free(done)                                      # rows of ended episodes
    history = history.fork(parents)                         # rows become their parents
    history.compact()                                       # live pages to the front
    records, counts = history.read(steps)                   # the last records, dense

An env writes its outputs on its own stream, hence the wait before they are read.

Everything runs on torch's current stream of the pages' device, without a host
synchronisation, and can be captured into CUDA graphs; two calls on one history (or
on a history and its fork) must be ordered by the caller if they run on different
streams.  Errors are as in ``carl_b200.carl``.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import capi


@functools.lru_cache
def _workspaces(n_rows: int, row_pages: int, n_pages: int, page_len: int) -> tuple[int, int]:
    """Workspace bytes of an append and a compaction."""
    sizes = ctypes.c_int64(), ctypes.c_int64()
    # The addresses are not looked at beyond being there.
    capi.check(capi.load().carlb_history_workspace(capi.History(16, 16, 16, 16, 1, n_rows, row_pages, n_pages, page_len, 0),
                                                   *sizes))
    return max(16, sizes[0].value), max(16, sizes[1].value)


class PagedHistory:
    """Pages, table, lengths and reference counts of a paged history.

    pages    any dtype [n_pages, page_len, *record], contiguous
    table    int32 [n_rows, row_pages]: record i of row r lies in page
             table[r, i // page_len]; entries behind the last page in use are -1
    lengths  int32 [n_rows]
    refs     int32 [n_pages]: how many table entries name the page; 0 = free

    The constructor wraps tensors that already hold a history; `empty` makes a new one.
    `dropped` (int32 [1]) counts the records that `append` found no place for; forks go on
    with it.  A constructor that is given none makes it with the first append, or fork, or
    look: one of these before a capture keeps it out of the graph.
    """

    def __init__(self, pages: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor,
                 dropped: torch.Tensor | None = None):
        books = (("table", table), ("lengths", lengths), ("refs", refs))
        if dropped is not None:
            books += ("dropped", dropped),
        if not isinstance(pages, torch.Tensor):
            raise TypeError("pages must be a tensor")
        for name, t in books:
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a tensor")
            if t.dtype is not torch.int32:
                raise TypeError(f"{name} must have dtype int32")
        device, shape, rows = pages.device, pages.shape, table.shape
        if not pages.is_cuda:
            raise ValueError("pages must be on a CUDA device")
        if not pages.is_contiguous():
            raise ValueError("pages must be contiguous")
        for name, t in books:
            if t.device != device:
                raise ValueError(f"{name} must be on {device}")
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
        if pages.requires_grad:
            raise ValueError("pages must not require a gradient")
        if len(shape) < 2 or 0 in shape[1:]:
            raise ValueError("pages must have shape [n_pages, page_len, *record] without empty dimensions")
        if len(rows) != 2 or rows[1] < 1 or lengths.shape != rows[:1] or refs.shape != shape[:1]:
            raise ValueError("table must be [n_rows, row_pages], lengths [n_rows] and refs [n_pages]")
        if dropped is not None and dropped.numel() != 1:
            raise ValueError("dropped must have one element")
        if rows[1] * shape[1] > 0x7fffffff or max(shape[0], rows[0]) > 0x7fffffff:
            raise ValueError("too many rows, pages or records of a row")
        record_bytes = pages.element_size()
        for n in shape[2:]:
            record_bytes *= n
        self._pages, self._books, self._dropped, self._device = pages, (table, lengths, refs), dropped, device
        at, t, n, r = pages.data_ptr(), table.data_ptr(), lengths.data_ptr(), refs.data_ptr()
        self._view = capi.History(at, t, n, r, record_bytes, rows[0], rows[1], shape[0], shape[1], device.index)
        self._own = ((at, at + record_bytes * shape[0] * shape[1]), (t, t + 4 * rows[0] * rows[1]), (n, n + 4 * rows[0]),
                     (r, r + 4 * shape[0]))  # what the operators write to

    @classmethod
    def empty(cls, n_rows: int, row_pages: int, n_pages: int, page_len: int, record_shape: tuple = (),
              dtype: torch.dtype = torch.float32, device: torch.device | str | int | None = None) -> PagedHistory:
        """A history without records: every row empty, every page free."""
        if min(n_rows, n_pages) < 0 or min(row_pages, page_len) < 1:
            raise ValueError("n_rows and n_pages must be non-negative, row_pages and page_len positive")
        if device is None:
            device = torch.device("cuda", torch.cuda.current_device())
        return cls(torch.zeros((n_pages, page_len, *record_shape), dtype=dtype, device=device),
                   torch.full((n_rows, row_pages), -1, dtype=torch.int32, device=device),
                   torch.zeros(n_rows, dtype=torch.int32, device=device),
                   torch.zeros(n_pages, dtype=torch.int32, device=device),
                   torch.zeros(1, dtype=torch.int32, device=device))

    @property
    def pages(self) -> torch.Tensor:
        return self._pages

    def _book(self, which: int) -> torch.Tensor:
        # A fork keeps its books in one tensor and parts them when they are looked at.
        if not isinstance(self._books, tuple):
            v = self._view
            entries = v.n_rows * v.row_pages
            table, lengths, refs, _ = self._books.split((entries, v.n_rows, v.n_pages, 1))
            self._books = table.view(v.n_rows, v.row_pages), lengths, refs
        return self._books[which]

    @property
    def table(self) -> torch.Tensor:
        return self._book(0)

    @property
    def lengths(self) -> torch.Tensor:
        return self._book(1)

    @property
    def refs(self) -> torch.Tensor:
        return self._book(2)

    @property
    def record_shape(self) -> tuple[int, ...]:
        return tuple(self._pages.shape[2:])

    @property
    def n_rows(self) -> int:
        return self._view.n_rows

    @property
    def n_pages(self) -> int:
        return self._view.n_pages

    @property
    def page_len(self) -> int:
        return self._view.page_len

    @property
    def dropped(self) -> torch.Tensor:
        if self._dropped is None:
            self._dropped = torch.zeros(1, dtype=torch.int32, device=self._device)
        return self._dropped

    def _written(self, *tensors: torch.Tensor) -> None:
        # The kernels write by address; a backward pass that has saved a tensor must not use it.
        books = self._books if isinstance(self._books, tuple) else (self._books,)
        torch.autograd.graph.increment_version((*books, *tensors))

    def _stream(self) -> int:
        return torch._C._cuda_getCurrentRawStream(self._view.device)

    def _mask(self, mask, name: str) -> torch.Tensor:
        if not isinstance(mask, torch.Tensor) or mask.dtype != torch.bool:
            raise TypeError(f"{name} must be a bool tensor")
        if mask.device != self._device:
            raise ValueError(f"{name} must be on {self._device}")
        if mask.shape != (self._view.n_rows,):
            raise ValueError(f"{name} must have shape [n_rows]")
        return mask if mask.is_contiguous() else mask.contiguous()

    def _indices(self, indices, name: str) -> torch.Tensor:
        if not isinstance(indices, torch.Tensor) or indices.dtype != torch.int64:
            raise TypeError(f"{name} must be an int64 tensor")
        if indices.device != self._device:
            raise ValueError(f"{name} must be on {self._device}")
        if indices.numel() > 0x7fffffff:
            raise ValueError(f"too many {name}")
        return indices if indices.is_contiguous() else indices.contiguous()

    def fork(self, parents: torch.Tensor, out: PagedHistory | None = None) -> PagedHistory:
        """The history whose row r continues row parents[r] of this one.

        parents  int64 of any shape, flattened to rows; a value outside [0, n_rows)
                 gives an empty row

        Pages are shared, not copied; pages that no row of the result names are free
        in it.  The result replaces this history, which is void once the result is
        appended to or compacted.  `out` takes the result instead of a new history: one
        over the same pages with a table, lengths and refs of its own (two histories
        used in turn, for instance by captured graphs); it takes over this one's `dropped`."""
        p = self._indices(parents, "parents")
        v, n, counter, dropped = self._view, p.numel(), None, None
        if out is None:
            entries = n * v.row_pages
            book = torch.empty(entries + n + v.n_pages + 1, dtype=torch.int32, device=self._device)
            out = PagedHistory.__new__(PagedHistory)
            out._pages, out._books, out._dropped, out._device = self._pages, book, self._dropped, self._device
            at = book.data_ptr()
            lengths = at + 4 * entries
            refs = lengths + 4 * n
            out._view = capi.History(v.pages, at, lengths, refs, v.record_bytes, n, v.row_pages, v.n_pages, v.page_len, v.device)
            out._own = self._own[0], (at, refs + 4 * v.n_pages + 4)  # the pages; the books and a counter
            if out._dropped is None:
                out._dropped, counter = book[-1:], refs + 4 * v.n_pages
        elif (out._view.pages != v.pages or out._pages.shape != self._pages.shape or out._pages.dtype != self._pages.dtype
              or (out._view.n_rows, out._view.row_pages) != (n, v.row_pages)):
            raise ValueError("out must be over the same pages, with a row for every parent")
        else:
            dropped = self.dropped
        capi.check(capi.load().carlb_history_fork(v, out._view, p.data_ptr(), counter, self._stream()))
        if dropped is not None:
            out._dropped = dropped
            out._written()
        return out

    def append(self, records: torch.Tensor, mask: torch.Tensor | None = None) -> None:
        """Appends records[r] to every row r, or to those with mask[r].

        A row at a page's end takes a free page.  A row whose last page is shared takes
        a free page and copies that page's records first; where all rows that share the
        page append, the longest of them (the first of those) writes on in it instead.
        Free pages go lowest first to the rows in order.  A row that finds no free page,
        or has no table entry left, stays as it was and is counted in `dropped`."""
        if not isinstance(records, torch.Tensor) or records.dtype != self._pages.dtype:
            raise TypeError("records must be a tensor of the pages' dtype")
        if records.device != self._device:
            raise ValueError(f"records must be on {self._device}")
        shape, v = records.shape, self._view
        n = v.n_rows
        if len(shape) == 0 or shape[0] != n or shape[1:] != self._pages.shape[2:]:
            raise ValueError("records must have shape [n_rows, *record]")
        m = None if mask is None else self._mask(mask, "mask")
        if n == 0:
            return
        if not records.is_contiguous() and not records[0].is_contiguous():
            records = records.detach().contiguous()
        at, step, counter = records.data_ptr(), records.stride(0) * records.element_size(), self.dropped.data_ptr()
        end = at + (n - 1) * step + v.record_bytes
        for low, high in self._own:
            if at < high and low < end:
                break
        else:
            low, high = counter, counter + 4
        if at < high and low < end:
            records = records.clone()  # the history's own memory, which is written to
            at, step = records.data_ptr(), records.stride(0) * records.element_size()
        lib = capi.load()
        size = _workspaces(n, v.row_pages, v.n_pages, v.page_len)[0]
        work = torch.empty(size, dtype=torch.uint8, device=self._device)
        capi.check(lib.carlb_history_append(v, at, step, None if m is None else m.data_ptr(), counter, work.data_ptr(), size,
                                            self._stream()))
        self._written(self._pages, self._dropped)

    def free(self, mask: torch.Tensor) -> None:
        """Empties the rows with mask[r]; a page is free when no row names it any more."""
        m = self._mask(mask, "mask")
        if self._view.n_rows:
            capi.check(capi.load().carlb_history_free(self._view, m.data_ptr(), self._stream()))
            self._written()

    def compact(self) -> torch.Tensor:
        """Moves the live pages to the front and returns their number, int32 [1] on the
        device: of L live pages, the k-th highest goes to the k-th free page below L.
        pages[:L] is then all that the history holds."""
        v = self._view
        size = _workspaces(v.n_rows, v.row_pages, v.n_pages, v.page_len)[1]
        work = torch.empty(size, dtype=torch.uint8, device=self._device)
        live = torch.empty(1, dtype=torch.int32, device=self._device)
        capi.check(capi.load().carlb_history_compact(v, live.data_ptr(), work.data_ptr(), size, self._stream()))
        self._written(self._pages)
        return live

    def read(self, steps: int, rows: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The last `steps` records of the rows (all, or int64 row indices of any shape):
        records [*rows, steps, *record], oldest first, zeros behind a row's last, and
        their number, int32 [*rows].  A row index outside [0, n_rows) counts 0."""
        steps = int(steps)
        if steps < 1:
            raise ValueError("steps must be positive")
        r = None if rows is None else self._indices(rows, "rows")
        shape = torch.Size((self._view.n_rows,)) if r is None else r.shape
        counts = torch.empty(shape, dtype=torch.int32, device=self._device)
        n = counts.numel()
        if n * steps > 1 << 33 or steps > 0x7fffffff:
            raise ValueError("too many records")
        out = torch.empty((*shape, steps, *self._pages.shape[2:]), dtype=self._pages.dtype, device=self._device)
        if n:
            capi.check(capi.load().carlb_history_read(self._view, None if r is None else r.data_ptr(), n, steps,
                                                      out.data_ptr(), counts.data_ptr(), self._stream()))
        return out, counts
