"""A paged 4-bit prefix cache for many sequences: page accounting on the host, one pool for
all layers on the GPU (the pages' bytes: include/b200_kv4.h).

The reference fills one dense bf16 cache per prompt and one for the CFG negative
(src/pipeline.rs:154-155).  Here sequences share pages: a fork takes no memory (n images of
one prompt, one negative prompt for every request), extending a fork copies its unfinished
last page first, and freed pages are taken again, lowest first; ``compact`` moves the live
pages to the front of the pool.
"""
from __future__ import annotations

import contextlib
import copy
import functools
import heapq
import threading
from typing import Callable, Dict, List, Optional, Sequence, Tuple

import b200attn
from b200attn import KV4_BLOCK_BYTES, KV4_PAGE_TOKENS as PAGE

Copies = List[Tuple[int, int]]  # (source page, destination page)


class OutOfPages(RuntimeError):
    """The pool has too few free pages; nothing was changed."""


def _locked(call):
    """The method, holding the object's lock."""
    @functools.wraps(call)
    def held(self, *args, **kwargs):
        with self.lock:
            return call(self, *args, **kwargs)
    return held


class PageTables:
    """Which pages hold which sequence's tokens (host only; moves no data).  Calls that need
    page contents moved return the copies, whose sources and destinations are disjoint.
    Threads may share the tables: each call holds ``lock``."""

    def __init__(self, num_pages: int):
        if num_pages < 0:
            raise ValueError("num_pages must not be negative")
        self.num_pages = num_pages
        self.lock = threading.RLock()
        self._free = list(range(num_pages))  # a heap
        self._uses = [0] * num_pages         # sequences that hold the page
        self._pages: Dict[int, List[int]] = {}
        self._length: Dict[int, int] = {}
        self._next = 0

    def __getstate__(self):
        with self.lock:  # copies and pickles carry the accounting, not the lock
            return {k: copy.copy(v) for k, v in self.__dict__.items() if k != "lock"}

    def __setstate__(self, state):
        self.__dict__.update(state, lock=threading.RLock())

    @property
    def free_pages(self) -> int:
        return len(self._free)

    @_locked
    def pages(self, seq: int) -> List[int]:
        return list(self._pages[seq])

    @_locked
    def length(self, seq: int) -> int:
        return self._length[seq]

    def _take(self, n: int) -> List[int]:
        if n > len(self._free):
            raise OutOfPages(f"{n} pages wanted, {len(self._free)} free of {self.num_pages}")
        got = [heapq.heappop(self._free) for _ in range(n)]
        for p in got:
            self._uses[p] = 1
        return got

    def _give_back(self, pages: Sequence[int]) -> None:
        for p in pages:
            self._uses[p] -= 1
            if self._uses[p] == 0:
                heapq.heappush(self._free, p)

    @_locked
    def add(self, length: int) -> int:
        """A new sequence with room for `length` tokens; returns its id."""
        if length < 0:
            raise ValueError("a length must not be negative")
        pages = self._take(-(-length // PAGE))
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._length[seq] = pages, length
        return seq

    @_locked
    def fork(self, seq: int) -> int:
        """A new sequence with the same tokens, on the same pages."""
        pages = self._pages[seq]
        for p in pages:
            self._uses[p] += 1
        new, self._next = self._next, self._next + 1
        self._pages[new], self._length[new] = list(pages), self._length[seq]
        return new

    @_locked
    def extend(self, seqs: Sequence[int], counts: Sequence[int],
               move: Optional[Callable[[Copies], None]] = None) -> Copies:
        """Room for counts[i] more tokens behind sequence seqs[i] (each named once).  A last
        page that is not full and that another sequence holds too is replaced by a copy of
        its own.  All or nothing; `move` is given the copies before anything changes, and if
        it raises, nothing does."""
        if len(set(seqs)) != len(seqs) or len(seqs) != len(counts) or any(n < 0 for n in counts):
            raise ValueError("seqs must be distinct, with one count of at least 0 each")
        uses: Dict[int, int] = {}
        plan = []
        for seq, n in zip(seqs, counts):
            pages, length = self._pages[seq], self._length[seq]
            own = None
            if n and length % PAGE:
                last = pages[-1]
                if uses.setdefault(last, self._uses[last]) > 1:
                    uses[last] -= 1  # of several forks extended together, one keeps the page
                    own = last
            plan.append((seq, n, own, -(-(length + n) // PAGE) - len(pages)))
        got = self._take(sum(more + (own is not None) for _, _, own, more in plan))
        fresh = iter(got)
        copies = [(own, next(fresh)) for _, _, own, _ in plan if own is not None]
        if move is not None:
            try:
                move(copies)
            except BaseException:
                self._give_back(got)
                raise
        into = iter(copies)
        for seq, n, own, more in plan:
            pages = self._pages[seq]
            if own is not None:
                pages[-1] = next(into)[1]
                self._uses[own] -= 1
            pages += [next(fresh) for _ in range(more)]
            self._length[seq] += n
        return copies

    @_locked
    def free(self, seq: int) -> None:
        """Forgets a sequence; pages that no other sequence holds are free again."""
        self._give_back(self._pages.pop(seq))
        del self._length[seq]

    @_locked
    def compact(self, move: Optional[Callable[[Copies], None]] = None) -> Copies:
        """Moves the live pages onto the first ids: afterwards page i is live exactly if i <
        num_pages - free_pages.  `move` as in extend."""
        live = self.num_pages - len(self._free)
        holes = sorted(p for p in self._free if p < live)
        high = [p for p in range(live, self.num_pages) if self._uses[p]]
        to = dict(zip(high, holes))
        copies = list(to.items())
        if move is not None:
            move(copies)
        for src, dst in copies:
            self._uses[dst], self._uses[src] = self._uses[src], 0
        for seq, pages in self._pages.items():
            self._pages[seq] = [to.get(p, p) for p in pages]
        self._free = list(range(live, self.num_pages))
        return copies


class ReuseOrder:
    """Orders the reuse of pages between streams.  Pages become free while work that reads
    them may still be queued, and may be taken for another stream's work: ``released`` marks
    a stream's queue where it gave pages back (or queued copies of pages), and ``before_taking``
    makes a stream wait for all marks.  Streams are torch streams; `event` makes an event."""

    def __init__(self, event):
        self._event = event
        self._marks: Dict[int, Tuple] = {}  # a stream's handle -> (stream, its latest mark)

    def released(self, stream) -> None:
        mark = self._event()
        mark.record(stream)
        self._marks[stream.cuda_stream] = (stream, mark)

    def before_taking(self, stream) -> None:
        for _, mark in self._marks.values():
            stream.wait_event(mark)


class KV4Cache:
    """Pools of `layers` layers (uint8 [layers, num_pages, heads, 9216]) with the accounting
    above.  Work is enqueued on the current stream of the pool's device.

    Threads and streams may share a cache.  ``free`` may be called as soon as the last work
    that reads the sequences is queued on the current stream (or the current stream waits for
    it): pages are taken again, by ``add``, ``extend`` or ``compact`` on any stream, behind
    that work.  New pages are filled on the stream that took them, or behind it; a stream that
    reads, forks, extends or compacts what another one stored waits for that one first.  Calls
    made while a graph is captured are not ordered: that is for whoever replays it."""

    def __init__(self, layers: int, heads: int, num_pages: int, device="cuda"):
        import torch
        self.layers, self.heads = layers, heads
        self.tables = PageTables(num_pages)
        self.lock = self.tables.lock
        self.pool = torch.empty((layers, num_pages, heads, KV4_BLOCK_BYTES), dtype=torch.uint8,
                                device=device)
        self._order = ReuseOrder(torch.cuda.Event)

    @contextlib.contextmanager
    def _pages_move(self, takes: bool, releases: bool):
        """Holds the lock around a change of the tables and what it queues; orders the current
        stream behind others' use of free pages, and others behind this one's."""
        import torch
        with self.lock:
            stream = None
            if self.pool.is_cuda:
                with torch.cuda.device(self.pool.device):
                    if not torch.cuda.is_current_stream_capturing():
                        stream = torch.cuda.current_stream()
            if takes and stream is not None:
                self._order.before_taking(stream)
            try:
                yield
            finally:
                if releases and stream is not None:
                    self._order.released(stream)

    @staticmethod
    def pages_for(lengths: Sequence[int]) -> int:
        """Pages that sequences of these lengths take."""
        return sum(-(-n // PAGE) for n in lengths)

    def nbytes(self) -> int:
        return self.pool.numel()

    def add(self, lengths: Sequence[int]) -> List[int]:
        """New sequences of these lengths, to be filled with ``store`` (all or none)."""
        lengths = [int(n) for n in lengths]
        if any(n < 0 for n in lengths):
            raise ValueError("a length must not be negative")
        with self._pages_move(takes=True, releases=False):
            if self.pages_for(lengths) > self.tables.free_pages:
                raise OutOfPages(f"{self.pages_for(lengths)} pages wanted, {self.tables.free_pages} free")
            return [self.tables.add(n) for n in lengths]

    @_locked
    def fork(self, seqs: Sequence[int]) -> List[int]:
        """A fork of each sequence (all or none)."""
        for s in seqs:
            self.tables.length(s)
        return [self.tables.fork(s) for s in seqs]

    def free(self, seqs: Sequence[int]) -> None:
        """Forgets these sequences, each named once (all or none)."""
        with self._pages_move(takes=False, releases=True):
            for s in seqs:
                self.tables.length(s)
            if len(set(seqs)) != len(seqs):
                raise ValueError("a sequence is freed once")
            for s in seqs:
                self.tables.free(s)

    def _move(self, copies: Copies) -> None:
        if copies:
            b200attn.kv4_copy_pages(self.pool, [s for s, _ in copies], [d for _, d in copies])

    def extend(self, seqs: Sequence[int], counts: Sequence[int]) -> None:
        """Room for more tokens, to be filled with ``store`` from the old lengths on."""
        with self._pages_move(takes=True, releases=True):
            self.tables.extend(seqs, counts, self._move)

    def compact(self) -> int:
        """Moves the live pages to the front of the pool; returns how many pages were moved.
        Views taken before are stale."""
        with self._pages_move(takes=True, releases=True):
            return len(self.tables.compact(self._move))

    def view(self, seqs: Sequence[int]) -> "KV4View":
        """The page tables of a batch as they are now (stale after extend, free, compact)."""
        return KV4View(self, list(seqs))


class KV4View:
    """A batch of sequences of a KV4Cache: page table (int32 [B, pages]) and lengths on the
    device, for the cached steps that read it."""
    on_host = False

    def __init__(self, cache: KV4Cache, seqs: List[int]):
        import torch
        self.cache, self.seqs = cache, seqs
        with cache.lock:
            self.lengths = [cache.tables.length(s) for s in seqs]
            rows = [cache.tables.pages(s) for s in seqs]
        width = max([1] + [len(r) for r in rows])
        self.page_table = torch.tensor([r + [-1] * (width - len(r)) for r in rows], dtype=torch.int32,
                                       device=cache.pool.device).view(len(seqs), width)
        self.max_len = max(self.lengths, default=0)

    def pool(self, layer: int):
        return self.cache.pool[layer]

    def store(self, layer: int, k, v, start=None, count=None) -> None:
        """k, v bf16 [B, H, T, 128] into this layer's pages (see b200attn.kv4_store).  Pages
        that forks share are read by all of them: new tokens of a fork go behind its length
        of before ``extend``, whose copy makes that page its own."""
        b200attn.kv4_store(k, v, self.pool(layer), self.page_table, start=start, count=count)

    def load(self, layer: int, lengths=None):
        """This layer's (k, v) as bf16 [B, H, max_len, 128]; rows behind a sequence's end are
        zeros."""
        import torch
        if lengths is None:
            lengths = torch.tensor(self.lengths, dtype=torch.int32, device=self.page_table.device)
        return b200attn.kv4_load(self.pool(layer), self.page_table, lengths, self.max_len)
