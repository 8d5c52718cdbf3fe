"""Page pool of a paged cache whose bookkeeping lives on the device.

Sequences of one prompt share its pages: ``fork`` starts continuations, ``extend`` grows them
for the next rows, ``truncate`` takes back rejected rows, ``free`` ends them, ``compact`` packs
the live pages to the front of the pool.  All of it runs on the current stream with no host
round trip, so the calls can sit inside a CUDA graph with the attention that reads
``page_table`` and ``seq_len``.  Pages are handed out lowest free id first in request order:
every call has one result.

Errors that only the device can see (a slot out of range or named twice, a child that is not
empty, too few free pages) set ``err`` (``check()`` reads it); a ``fork`` or ``extend`` with
such a request changes nothing.
"""

from __future__ import annotations

import torch

from . import _ext

FORK, EXTEND, TRUNCATE, COMPACT, COPY = range(5)
_ERRORS = {3: "a request the pool cannot serve (slot, parent or length)", 6: "too few free pages"}


def _aligned(n: int) -> int:
    return (n + 31) // 32 * 32


class PagePool:
    """``caches``: device tensors [layers, pages, ...] of one page count (``paged_caches()`` of a
    runner); ``page_table`` [num_slots, max_pages] and ``seq_len`` [num_slots] are views of the
    pool's one int32 ``state`` tensor.  Page 0 is the padding page and stays taken."""

    def __init__(self, caches: list[torch.Tensor], num_slots: int, max_pages: int, page_size: int = 16):
        if not caches:
            raise ValueError("a page pool needs at least one cache")
        pages = int(caches[0].shape[1])
        if any(c.dim() < 2 or int(c.shape[1]) != pages for c in caches):
            raise ValueError("caches must be [layers, pages, ...] with one page count")
        if num_slots < 1 or max_pages < 1 or page_size < 1 or pages < 2:
            raise ValueError("num_slots, max_pages and page_size must be positive, and pages at least 2")
        self.C = _ext.load()
        self.caches = list(caches)
        self.page_size = page_size
        self.num_pages, self.num_slots, self.max_pages = pages, num_slots, max_pages
        dev = caches[0].device
        words = (pages + 31) // 32
        sizes = [_aligned(pages), _aligned(words), _aligned(num_slots), num_slots * max_pages]
        self.state = torch.zeros(sum(sizes), dtype=torch.int32, device=dev)
        ref, bits, lens, table = self.state.split(sizes)
        self.refcount, self.free_bits, self.seq_len = ref[:pages], bits[:words], lens[:num_slots]
        self.page_table = table.view(num_slots, max_pages)
        self.err = torch.zeros(1, dtype=torch.int32, device=dev)
        self._scratch = torch.zeros(self.C.pool_scratch_ints(pages, num_slots), dtype=torch.int32, device=dev)
        self.refcount[0] = 1
        self._count_free()

    def _count_free(self) -> None:
        """free_bits from refcount."""
        free = torch.zeros(self.free_bits.numel() * 32, dtype=torch.int64, device=self.state.device)
        free[:self.num_pages] = self.refcount == 0
        bits = (free.view(-1, 32) << torch.arange(32, device=free.device)).sum(1)
        self.free_bits.copy_(torch.where(bits >= 1 << 31, bits - (1 << 32), bits))

    def adopt(self, seq_len: torch.Tensor, page_table: torch.Tensor) -> None:
        """Take over sequences whose pages are filled: lengths [num_slots] and their table rows
        [num_slots, <= max_pages].  Replaces what the pool held."""
        if seq_len.shape != self.seq_len.shape or page_table.dim() != 2 or page_table.shape[0] != self.num_slots \
                or page_table.shape[1] > self.max_pages:
            raise ValueError("adopt needs seq_len [num_slots] and page_table [num_slots, <= max_pages]")
        width = page_table.shape[1]
        used = torch.arange(width, device=self.state.device)[None, :] < \
            ((seq_len + self.page_size - 1) // self.page_size)[:, None].to(self.state.device)
        ids = page_table.to(self.state.device)[used].long()
        if ids.numel() and (int(ids.min()) < 1 or int(ids.max()) >= self.num_pages):
            raise ValueError("adopt: a page id outside the pool")
        if int(seq_len.max()) > width * self.page_size:
            raise ValueError("adopt: a sequence is longer than its table row")
        if int(seq_len.min()) < 0:
            raise ValueError("adopt: a negative length")
        self.page_table.zero_()
        self.page_table[:, :width].copy_(torch.where(used, page_table.to(self.state.device), 0))
        self.seq_len.copy_(seq_len)
        self.refcount.copy_(torch.bincount(ids, minlength=self.num_pages))
        self.refcount[0] = 1
        self._count_free()

    def _call(self, which: int, slots=None, parents=None, lens=None) -> None:
        if which != COMPACT and (slots is None or which in (FORK, COPY) and parents is None):
            raise ValueError("a page pool call needs its slots (or pages)")
        self.C.pool_call(which, self.refcount, self.free_bits, self.seq_len, self.page_table, self.page_size,
                         self.caches, slots, parents, lens, self._scratch, self.err)

    def fork(self, parents: torch.Tensor, children: torch.Tensor, share: torch.Tensor | None = None) -> None:
        """Empty slot ``children[i]`` becomes a copy of slot ``parents[i]``: the whole pages below
        ``share[i]`` tokens (all of them by default) are shared, the others copied.  A parent
        that is itself a child of the same call counts as empty."""
        self._call(FORK, children, parents, share)

    def extend(self, slots: torch.Tensor, new_len: torch.Tensor) -> None:
        """Grow distinct slots to ``new_len`` tokens (no effect where they are that long): fresh
        pages are appended, and a partly filled last page that other slots also refer to is
        copied first."""
        if new_len is None:
            raise ValueError("extend needs new_len")
        self._call(EXTEND, slots, None, new_len)

    def truncate(self, slots: torch.Tensor, new_len: torch.Tensor) -> None:
        """Cut slots to ``new_len`` tokens (no effect where they are that short) and drop the pages past them."""
        if new_len is None:
            raise ValueError("truncate needs new_len (free ends a sequence)")
        self._call(TRUNCATE, slots, None, new_len)

    def free(self, slots: torch.Tensor) -> None:
        """End the sequences in ``slots``."""
        self._call(TRUNCATE, slots)

    def compact(self) -> None:
        """Move the n live pages to ids 0..n-1 (the j-th live page from id n on to the j-th free
        page below n), with their data and every table entry."""
        self._call(COMPACT)

    def copy(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Copy pages ``src[i]`` to ``dst[i]`` in every layer of every cache.  No page may be both
        a source and a destination.  A source or destination 0 is skipped."""
        self._call(COPY, src, dst)

    def check(self) -> None:
        """Raise if a call since the last check failed (reads the device's error word)."""
        code = int(self.err.item())
        if code:
            self.err.zero_()
            raise RuntimeError(f"page pool: {_ERRORS.get(code, f'error {code}')}")
