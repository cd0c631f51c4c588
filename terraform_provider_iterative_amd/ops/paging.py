"""Pages of a paged cache: copying, forking, extending, freeing and compacting.

A cache of many sequences is kept in pages of ``page_tokens`` tokens; page ``i`` is row ``i`` of
each of a set of tensors (keys and values of every layer).  :class:`PagePool` keeps the books on
the device beside it -- which pages a sequence has, how many sequences name a page, which pages
are free -- and moves pages' bytes in all tensors with one launch.  No operation waits for the
host, so they can be captured into a graph; the host reads the books when it asks
(:meth:`PagePool.status`).

Results are the same on every run and on the host (``csrc/hip/pages.hip``,
``csrc/native/pages.cpp``): free pages are taken lowest number first, in the order in which
sequences are named.

The books are one int32 tensor (:attr:`PagePool.meta`).  ``TrainingState(paged={"kv": pool})``
checkpoints it with the pool's tensors, after the live pages have been moved together and the
dead ones cleared: those cost a spill through the codec next to nothing.
"""
from __future__ import annotations

import struct
from typing import Any, Dict, List, Optional, Sequence, Union

import numpy as np
import torch

from ._loader import native, torch_hip
from .packing import canonical_view

HEADER, CHUNK_UNITS = 16, 1024  # TPI_PAGES_HEADER, TPI_PAGE_UNITS
_POOL = struct.Struct("<8Q6i")  # tpi_pages
_CHUNK = np.dtype([("base", "<u8"), ("page_stride", "<i8"), ("row_stride", "<i8"),  # tpi_page_chunk
                   ("row_bytes", "<u4"), ("rows", "<u4"), ("row_units", "<u4"), ("pad", "<u4")])
_FREE, _ERROR, _SHAPE = 0, 1, 8  # words of the header
_ERRORS = {1: "not enough free pages", 2: "a slot is out of range",
           3: "a fork's destination holds a sequence (or is its source)",
           4: "a sequence would be longer than a row of the table",
           5: "a page is out of range", 6: "a slot is named twice",
           7: "a negative number of tokens", 8: "the pool's books contradict themselves"}

Numbers = Union[Sequence[int], torch.Tensor]


class PageError(RuntimeError):
    """A pool refused an operation."""


def _pad4(words: int) -> int:
    return (words + 3) // 4 * 4


def _has_memory(t: torch.Tensor) -> bool:
    """Whether all elements lie in memory of the tensor's own: those of a wrapper (DTensor, fake,
    jagged) or of a freed storage do not, and the kernels go by addresses."""
    if t.layout is not torch.strided or t.is_nested or torch._is_zerotensor(t):
        return False
    span = t.storage_offset() + 1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride()))
    return t.data_ptr() != 0 and span * t.element_size() <= t.untyped_storage().nbytes()


class PagePool:
    """The pages of ``tensors`` and the ``slots`` sequences that hold them.

    ``tensors``: one or more tensors of one device whose first dimension is the page, all with the
    same number of pages and none sharing memory; a page's bytes are one contiguous run, or
    several with one stride between them (``[heads, pages, ...]`` storage seen pages first).
    ``page_tokens``: tokens of a page.  ``width``: pages that one sequence can have (default: all).

    * :attr:`table` ``[slots, width]`` int32: pages of each slot's sequence, -1 behind its end
    * :attr:`lengths` ``[slots]`` int32: its tokens; 0: the slot is free
    * :attr:`refs` ``[pages]`` int32: table entries that name the page; 0: the page is free

    They are views of :attr:`meta` for kernels to read; change them through the methods (or
    :meth:`bind`) only.  Operations are enqueued on the current stream of the pool's device; two
    on one pool must not run at the same time, on two streams or in two graphs.  Slots and pages
    are given as lists, or as int32 / int64 tensors on the pool's device, read when the kernel
    runs.  An operation that cannot be done as a whole changes nothing: numbers given as lists
    that are out of range or named twice raise ``ValueError`` at once; what only the device can
    see (too few free pages, say) raises :class:`PageError` at the next :meth:`check`, on the host
    at once.
    """

    def __init__(self, tensors: Sequence[torch.Tensor], page_tokens: int, slots: int,
                 width: Optional[int] = None):
        tensors = list(tensors)
        if not tensors or not all(isinstance(t, torch.Tensor) for t in tensors):
            raise ValueError("a pool needs at least one tensor")
        if not all(map(_has_memory, tensors)):
            raise ValueError("a pool's tensors must be strided ones with memory of their own")
        self.device = tensors[0].device
        if self.device.type not in ("cuda", "cpu"):
            raise ValueError("a pool's tensors must be on the GPU or the host")
        self._on_device = self.device.type == "cuda"
        if any(t.dim() < 2 or t.numel() == 0 for t in tensors):
            raise ValueError("a pool's tensors need a page dimension and bytes in each page")
        if len({(t.device, t.shape[0]) for t in tensors}) != 1:
            raise ValueError("a pool's tensors must be on one device, with as many pages each")
        self.pages, self.page_tokens, self.slots = tensors[0].shape[0], int(page_tokens), int(slots)
        self.width = self.pages if width is None else int(width)
        if not 1 <= self.page_tokens <= 1 << 20:
            raise ValueError("page_tokens must be in [1, 2^20]")
        if self.slots < 1 or self.width < 1:
            raise ValueError("slots and width must be positive")
        # what one launch of the kernels can number
        if self.pages >= 1 << 30 or self.slots >= 1 << 23 or self.width >= 1 << 30:
            raise ValueError("too many pages, slots or pages of a sequence")
        if any(t.requires_grad for t in tensors):
            raise ValueError("a pool's tensors are written in place: none may require a gradient")
        self.tensors = tensors
        self._lay_out_tensors()
        words = (self.pages + 31) // 32
        self._sizes = [HEADER, _pad4(self.pages), _pad4(self.slots), _pad4(self.slots * self.width),
                       _pad4(words), _pad4(words)]
        self.meta = torch.empty(sum(self._sizes), dtype=torch.int32, device=self.device)
        self._bind_meta(words)
        self._scratch = torch.empty(4 * self.pages + 5 * self.slots, dtype=torch.int32,
                                    device=self.device)
        at = [t.data_ptr() for t in (self._header, self.refs, self.lengths, self.table,
                                     self._free_bits, self._stale_bits, self._scratch,
                                     self._chunk)]
        self._args = _POOL.pack(*at, self.pages, self.slots, self.width, self.page_tokens,
                                self._chunks, 0)
        self._streams = set()  # that use the memory: the one that it was allocated on, to begin with
        if self._on_device:
            self._streams.add(torch_hip().stream_and_capture(self.device.index)[0])
        self._write_books(np.full((self.slots, self.width), -1, np.int32),
                          np.zeros(self.slots, np.int32))

    # The kernels' arguments are addresses: a deep or unpickled copy is built around its own tensors
    # and books, a shallow one is another name for the same.
    def __reduce__(self):
        return PagePool._rebuilt, (self.tensors, self.page_tokens, self.slots, self.width, self.meta)

    def __copy__(self) -> "PagePool":
        out = object.__new__(type(self))
        out.__dict__.update(self.__dict__)
        return out

    @staticmethod
    def _rebuilt(tensors, page_tokens, slots, width, meta) -> "PagePool":
        pool = PagePool(tensors, page_tokens, slots, width)
        pool.meta.copy_(meta)
        return pool

    def _lay_out_tensors(self) -> None:
        parts, layouts = [], {}  # tensors mostly share one layout: cut it once
        for t in self.tensors:
            key = t.shape, t.stride(), t.element_size()
            if key not in layouts:
                layouts[key] = self._cut_page(t)
            part = layouts[key].copy()
            part["base"] += t.data_ptr()
            parts.append(part)
        chunks = np.concatenate(parts)
        if len(chunks) >= 1 << 23:
            raise ValueError("the pages are too large")
        self._chunks = len(chunks)
        self._chunk = torch.from_numpy(chunks.view(np.uint8)).to(self.device)

    def _cut_page(self, t: torch.Tensor) -> np.ndarray:
        """Chunks of a page of ``t``, from its first byte."""
        elem = t.element_size()
        strides = sorted((st, size) for st, size in zip(t.stride(), t.shape) if size > 1)
        if any(st <= 0 or (i and st < strides[i - 1][0] * strides[i - 1][1])
               for i, (st, _) in enumerate(strides)):
            raise ValueError("a pool's tensors must not overlap themselves")
        dims = canonical_view(t.shape[1:], t.stride()[1:])
        if dims[-1][1] != 1:  # elements with gaps between them: runs of one element
            dims.append((1, 1))
        if len(dims) > 2:
            raise ValueError("a page's bytes must be contiguous runs with one stride between "
                             "them, not %s with strides %s" % (tuple(t.shape), t.stride()))
        runs, run_stride = dims[0] if len(dims) == 2 else (1, 0)
        return self._cut(t.stride(0) * elem, runs, run_stride * elem, dims[-1][0] * elem)

    @staticmethod
    def _cut(page_stride: int, runs: int, run_stride: int, run: int) -> np.ndarray:
        """Chunks of a page: whole runs while several fit, pieces of one otherwise."""
        units = -(-run // 16)
        if units <= CHUNK_UNITS:
            step = CHUNK_UNITS // units
            rows = np.arange(0, runs, step)
            out = np.zeros(len(rows), _CHUNK)
            out["base"] = rows * run_stride
            out["rows"] = np.minimum(step, runs - rows)
            out["row_bytes"], out["row_units"] = run, units
        else:
            step = CHUNK_UNITS * 16
            starts = np.arange(0, run, step)
            ends = np.minimum(starts + step, run)
            starts = np.minimum(starts, run - 16)  # not less than one unit
            out = np.zeros(runs * len(starts), _CHUNK)
            out["base"] = (np.arange(runs)[:, None] * run_stride + starts).reshape(-1)
            out["rows"] = 1
            out["row_bytes"] = np.tile(ends - starts, runs)
            out["row_units"] = (out["row_bytes"] + 15) // 16
        out["page_stride"], out["row_stride"] = page_stride, run_stride
        return out

    def _bind_meta(self, words: int) -> None:
        parts = self.meta.split(self._sizes)
        self._header = parts[0]
        self.refs, self.lengths = parts[1][:self.pages], parts[2][:self.slots]
        self.table = parts[3][:self.slots * self.width].view(self.slots, self.width)
        self._free_bits, self._stale_bits = parts[4][:words], parts[5][:words]

    # -- books from the host ------------------------------------------------------------------
    def bind(self, table, lengths) -> "PagePool":
        """Take over sequences whose pages are already in the tensors: ``table`` ``[slots, <=
        width]`` and ``lengths`` ``[slots]``.  Sequences may share full pages; a partial last page is
        written by the next extension, so no other entry may name it.  Waits for the device."""
        table = torch.as_tensor(table).cpu().numpy().astype(np.int64)
        lengths = torch.as_tensor(lengths).cpu().numpy().astype(np.int64)
        if table.ndim != 2 or table.shape[0] != self.slots or table.shape[1] > self.width \
                or lengths.shape != (self.slots,):
            raise ValueError("table must be [%d, <= %d], lengths [%d]" % (
                self.slots, self.width, self.slots))
        if (lengths < 0).any() or (lengths > min(table.shape[1] * self.page_tokens,
                                                 (1 << 31) - 1)).any():
            raise ValueError("a length is negative or longer than its row of the table")
        held = np.arange(table.shape[1]) < -(-lengths // self.page_tokens)[:, None]
        if ((table < 0) | (table >= self.pages))[held].any():
            raise ValueError("a page of the table is out of range")
        books = np.full((self.slots, self.width), -1, np.int32)
        books[:, :table.shape[1]] = np.where(held, table, -1)
        part = (lengths % self.page_tokens != 0).nonzero()[0]
        named = np.bincount(books[books >= 0], minlength=self.pages)
        if (named[books[part, lengths[part] // self.page_tokens]] > 1).any():
            raise ValueError("a partial last page is named twice: give each sequence a copy")
        self._write_books(books, lengths.astype(np.int32))
        return self

    def _write_books(self, table: np.ndarray, lengths: np.ndarray) -> None:
        refs = np.bincount(table[table >= 0].astype(np.int64), minlength=self.pages)
        free = refs == 0
        words = self._free_bits.numel()
        packed = np.packbits(np.pad(free, (0, 32 * words - self.pages)), bitorder="little")
        meta = np.zeros(self.meta.numel(), np.int32)
        header, refs_, lengths_, table_, free_, stale_ = np.split(meta, np.cumsum(self._sizes)[:-1])
        header[_FREE] = int(free.sum())
        header[_SHAPE:_SHAPE + 4] = self._shape()
        refs_[:self.pages] = refs
        lengths_[:self.slots] = lengths
        table_[:table.size] = table.reshape(-1)
        free_[:words] = stale_[:words] = packed.view(np.int32)
        self.meta.copy_(torch.from_numpy(meta))

    # -- operations ---------------------------------------------------------------------------
    def _numbers(self, what: str, values: Numbers, limit: int, distinct: bool = False):
        """``values`` as a contiguous integer tensor on the pool's device."""
        if isinstance(values, torch.Tensor):
            if values.dtype not in (torch.int32, torch.int64) or values.dim() != 1:
                raise TypeError("%s must be a one-dimensional int32 or int64 tensor" % what)
            if values.device != self.device:
                raise ValueError("%s must be on %s" % (what, self.device))
            out = values.contiguous()
            if out.numel() and not out.data_ptr():  # a wrapper's, or of a freed storage
                raise ValueError("%s must have memory of their own" % what)
            if self._on_device:
                return out
            out = out.to(torch.int64)
        else:
            out = torch.tensor([int(v) for v in values], dtype=torch.int64)
        host = out.tolist()
        if any(not 0 <= v < limit for v in host):
            raise ValueError("%s must be in [0, %d)" % (what, limit))
        if distinct and len(set(host)) != len(host):
            raise ValueError("%s must be distinct" % what)
        return out.to(self.device)

    def _enqueue(self, name: str, *args) -> None:
        if self._on_device:
            stream = getattr(torch_hip(), "pages_" + name)(self._args, self.device.index, *args)
            if stream not in self._streams:  # a pool that is dropped keeps its memory until it is done
                self._streams.add(stream)
                for t in (self.meta, self._scratch, self._chunk, *self.tensors):
                    t.record_stream(torch.cuda.current_stream(self.device))
            return
        getattr(native(), "pages_" + name)(self._args, *args)
        self.check()

    def _pair(self, name: str, src, dst) -> None:
        if src.shape != dst.shape:
            raise ValueError("%s needs as many sources as destinations" % name)
        if src.dtype != dst.dtype:
            src, dst = src.to(torch.int64), dst.to(torch.int64)
        args = (src.data_ptr(), dst.data_ptr(), src.numel())
        if self._on_device:
            args += (int(src.dtype == torch.int64),)
        self._enqueue(name, *args)

    def _limit(self, name: str, count: int) -> None:
        if count > self.slots:  # some slot is named twice
            raise ValueError("%s of %d slots, the pool has %d" % (name, count, self.slots))

    def copy(self, src: Numbers, dst: Numbers) -> None:
        """Page ``src[i]`` to page ``dst[i]`` in every tensor; sequences and counts stay as they are (of
        a free page that is written, :meth:`compact` knows to clear it).  No page may be a
        destination twice, nor destination and source: of such a call on device numbers, those
        destinations' content is undefined.  A pair with a number out of range is left out."""
        known = not self._on_device or not (isinstance(src, torch.Tensor) or
                                                  isinstance(dst, torch.Tensor))
        if known and set(map(int, src)) & set(map(int, dst)):
            raise ValueError("a page is both source and destination")
        src = self._numbers("source pages", src, self.pages)
        dst = self._numbers("destination pages", dst, self.pages, distinct=True)
        self._pair("copy", src, dst)

    def fork(self, src: Numbers, dst: Numbers) -> None:
        """Slot ``dst[i]``, empty so far, becomes a copy of slot ``src[i]``'s sequence: it shares its
        full pages, and has a copy of a partial last page (either may go on writing).  A source may
        be named more than once; all are taken as they were before the call."""
        src = self._numbers("source slots", src, self.slots)
        dst = self._numbers("destination slots", dst, self.slots, distinct=True)
        self._limit("fork", dst.numel())
        self._pair("fork", src, dst)

    def extend(self, slots: Numbers, tokens: Union[int, Numbers]) -> None:
        """Slot ``slots[i]``'s sequence grows by ``tokens`` (``tokens[i]``) tokens: its row of the
        table gets the pages for them, lowest free number first.  The new tokens' bytes are
        whatever the pages held."""
        slots = self._numbers("slots", slots, self.slots, distinct=True)
        self._limit("extend", slots.numel())
        each, more = 0, None
        if isinstance(tokens, int):
            each = tokens
            if not 0 <= each < 1 << 31:
                raise ValueError("tokens must be in [0, 2^31)")
        else:
            more = self._numbers("tokens", tokens, 1 << 31)
            if more.shape != slots.shape:
                raise ValueError("extend needs as many token counts as slots")
        if self._on_device:
            wide = int(slots.dtype == torch.int64)
            if more is not None:
                wide |= 2 * int(more.dtype == torch.int64)
            self._enqueue("extend", slots.data_ptr(), slots.numel(), wide,
                          0 if more is None else more.data_ptr(), each)
            return
        if more is None:
            more = torch.full_like(slots, each)
        self._enqueue("extend", slots.data_ptr(), more.data_ptr(), slots.numel())

    def free(self, slots: Numbers) -> None:
        """The slots' sequences end: pages that no other sequence names become free.  A free slot
        stays free."""
        slots = self._numbers("slots", slots, self.slots, distinct=True)
        self._limit("free", slots.numel())
        args = (slots.data_ptr(), slots.numel())
        if self._on_device:
            args += (int(slots.dtype == torch.int64),)
        self._enqueue("free", *args)

    def compact(self, clear: bool = False) -> None:
        """Move the live pages to numbers 0, 1, ... (as few moves as there are holes among them) and
        rewrite the table.  ``clear``: also fill free pages with zeros, those that have been
        written since the last time."""
        self._enqueue("compact", int(clear) if self._on_device else bool(clear))

    def _shape(self) -> List[int]:
        return [self.pages, self.slots, self.width, self.page_tokens]

    # -- what the host may know ---------------------------------------------------------------
    def _read_header(self) -> List[int]:
        header = self._header.tolist()
        if header[_SHAPE:_SHAPE + 4] != self._shape():
            raise PageError("the books are those of a pool of %d pages, %d slots of %d pages and %d "
                            "tokens a page" % tuple(header[_SHAPE:_SHAPE + 4]))
        return header

    def resumed(self) -> None:
        """The books and the tensors have been restored from a checkpoint: raise
        :class:`PageError` if they are another pool's.  A refusal that the saved run had not asked
        for changed nothing, so it fails no resume: it stays for the next :meth:`check`, as it
        would have without the preemption (on the host, whose operations raise their own refusals
        at once, it is reported here as a warning)."""
        code = self._read_header()[_ERROR]
        if code and not self._on_device:
            import warnings

            self._header[_ERROR] = 0
            warnings.warn("the checkpoint's pool had refused an operation: %s"
                          % _ERRORS.get(code, "error %d" % code), stacklevel=2)

    def check(self) -> None:
        """Raise :class:`PageError` if an operation has been refused since the last check, or the
        books are not this pool's (of a checkpoint of another one).  Waits for the device."""
        code = self._read_header()[_ERROR]
        if code:
            self._header[_ERROR] = 0
            raise PageError(_ERRORS.get(code, "error %d" % code))

    def status(self) -> Dict[str, Any]:
        """``{"pages", "free", "live", "error"}``; waits for the device."""
        free, code = self._header[:2].tolist()
        return {"pages": self.pages, "free": free, "live": self.pages - free,
                "error": _ERRORS.get(code, "error %d" % code) if code else None}
