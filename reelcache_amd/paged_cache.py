"""A KV cache in pages: sequences that share, fork, drop and compact their history.

A restored history is written into native cache slots (reelcache/restore_kernels.py:235-305); a
serving engine keeps such slots in pages so that continuations of one history share it.
:class:`PagedCache` holds the K and V pools of all layers and, on the host, the pages of each
sequence.  Every layer uses the same page of a sequence for the same tokens, so a page is copied in
all layers' K and V pools at once (``rch_pages_copy``), and the slots of new tokens are written as runs of
consecutive rows (``rch_runs_store``).

Pools are ``[layers, pages, page_tokens, heads, head_dim]`` (``layout="BTHD"``) or ``[layers, pages,
heads, page_tokens, head_dim]`` (``"BHTD"``): one layer's pool is a native cache tensor whose batch
axis counts pages, so a restore writes into consecutive pages through :meth:`PagedCache.view`, and a
caller's native caches serve as pools of one page (``PagedCache(k[None], v[None])``).

The page tables are host state.  Whatever allocates takes the lowest free pages, in the order of the
sequences given, and checks that there are enough before it changes anything.  Device work runs on the
current stream of the cache's device, in order: callers that use several streams order them, and threads
that share a cache take turns.
"""

from __future__ import annotations

import ctypes
import heapq
import struct
import weakref
from dataclasses import dataclass, field

import numpy as np
import torch

from . import _lib
from ._checks import count, in_memory, need, one_of
from .errors import CapacityError, ConfigurationError, StateError, UnsupportedError
from .restore_model import OUTPUT_DTYPES, NativeView, Remembering
from .rotary import Launch, _span, addresses_of, capturing, entered, known_calls, need_gpu, position_fields, raw_stream

HOLE = -1
_LAYOUTS = ("BTHD", "BHTD")


@dataclass(eq=False)
class Slots(Remembering):
    """Where new tokens go: built by :meth:`PagedCache.extend` or :meth:`PagedCache.slots` once per
    step, used by :meth:`PagedCache.store` in every layer.  ``index``: int32 ``[tokens]`` on the device,
    page * page_tokens + row of each token, written on the stream that was current then (other streams
    wait for it)."""

    index: torch.Tensor
    tokens: int
    cache: "PagedCache"
    stamp: int
    stream: int


@dataclass(eq=False)
class Places(Slots):
    """The rows that tokens lie in, for reading them: built by :meth:`PagedCache.places`.  Their pages may be shared; no
    store takes them.  Stale once pages moved or were freed, and once a sequence of theirs goes on in a copy of its begun
    page (:meth:`PagedCache.extend`): the rows are another sequence's then."""

    pieces: tuple = field(default=(), repr=False)  # (sequence, its first page of theirs, the pages) of each
    copied: int = 0  # begun pages that the cache had copied when they last were the sequences'


@dataclass(frozen=True, eq=False)
class PageView(NativeView):
    """A restore destination in a sequence's pages (:meth:`PagedCache.view`).  A restore into it is refused
    once one of those pages moved, was dropped or freed, or is shared."""

    cache: "PagedCache | None" = field(default=None, repr=False)
    sequence: int = -1
    first: int = 0         # index of the first page in the sequence
    pages: tuple = ()      # the pages it had then
    item: "_Sequence | None" = field(default=None, repr=False)
    end: int = 0           # tokens that the sequence had to have

    def check(self):
        cache, item = self.cache, self.item
        if (cache._sequences.get(self.sequence) is not item or item.tokens < self.end
                or tuple(item.pages[self.first:self.first + len(self.pages)]) != self.pages
                or any(cache._uses[page] > 1 for page in self.pages)):
            raise StateError("pages moved, were freed or became shared after this view was made")


class _Sequence:
    __slots__ = ("pages", "tokens")

    def __init__(self, pages, tokens):
        self.pages, self.tokens = pages, tokens


# Tables of at most this many words travel in the arguments of one launch: 64 words take 6.5 us of the host
# so and 9.8 us through pinned memory, 960 words 7.7 and 10.0 us; at 1920 (two launches) it is 11.9 and 10.3 us.
_ARGUMENT_WORDS = 960
# Slots of at most this many runs (a run: the tokens of a sequence in one page) travel as runs in the arguments
# of a launch, more as an array: slots of one token take 9.9 and 16.6 us of the host, of 512 in two pages 11.2 and
# 19.4 us, of 1024 in 64 pages 20.6 and 26.1 us, of 2048 in 128 pages 30.8 and 30.9 us, of 4096 in 256 pages 51.6 and
# 40.7 us.
_FEW_RUNS = 128


def upload(values, device):
    """An int32 array on ``device``, written on its current stream without a host wait: small ones in
    launch arguments, larger ones from pinned memory (the block stays reserved until the copy has run)."""
    values = np.ascontiguousarray(values, dtype=np.int32)
    if values.size <= _ARGUMENT_WORDS:
        return upload_words(values.tobytes(), values.shape, device)
    _refuse_capture(device)
    return torch.from_numpy(values).pin_memory().to(device, non_blocking=True)


def upload_words(words, shape, device):
    """The same of a small table that the caller packed into bytes."""
    _refuse_capture(device)
    out = torch.empty(shape, dtype=torch.int32, device=device)
    _lib.check(_lib.function("rch_words_store")(out.data_ptr(), words, len(words) // 4, raw_stream(device)))
    return out


def upload_runs(runs, total, device):
    """An int32 array of runs of ascending values: ``runs`` is flat, (first value, count) of each."""
    _refuse_capture(device)
    out = torch.empty(total, dtype=torch.int32, device=device)
    _lib.check(_lib.function("rch_runs_store")(out.data_ptr(), _pack(runs), len(runs) // 2, total, raw_stream(device)))
    return out


def _refuse_capture(device):
    with entered(device):
        captured = capturing()
    if captured:
        raise ConfigurationError("page tables, slots and plans are built before a HIP-graph capture, not in it")


def _pack(words):
    return struct.pack(f"{len(words)}i", *words)


class PagedCache:
    """K and V pools of every layer, and the pages of each sequence.

    ``keys``, ``values``: pools as above, of one shape, dtype (bfloat16, float16, float32) and device,
    with unit stride over the channels; any other strides that keep elements apart.
    """

    _POOL_DTYPES, _POOL_TYPES = OUTPUT_DTYPES, "bfloat16, float16 or float32"
    #: What the pools hold besides values (RCH_CODES_*).
    codes = _lib.CODES_NONE

    def __init__(self, keys, values, *, layout="BTHD"):
        one_of(layout, _LAYOUTS, "pool layout")
        for pool, name in ((keys, "keys"), (values, "values")):
            in_memory(pool, name)
            need(pool.ndim == 5, f"{name} must be [layers, pages, ...] pools of five dimensions")
            need(pool.dtype in self._POOL_DTYPES, f"{name} must be {self._POOL_TYPES}")
            need(min(pool.shape) >= 1, f"{name} must not be empty")
            need(pool.stride(4) == 1 or pool.shape[4] == 1, f"{name} must have unit stride over the channels")
            need(_apart(pool), f"{name} must keep its elements apart")
            need(not pool.requires_grad, f"{name} must not require gradients")
        need(keys.shape == values.shape and keys.dtype == values.dtype and keys.device == values.device,
             "keys and values must match in shape, dtype and device")
        self.keys, self.values, self.layout = keys, values, layout
        token, head = (2, 3) if layout == "BTHD" else (3, 2)
        self.layers, self.pages = keys.shape[:2]
        self.page_tokens, self.heads, self.head_dim = keys.shape[token], keys.shape[head], keys.shape[4]
        need(self.pages * self.page_tokens < 1 << 31, "a pool holds fewer than 2**31 tokens")
        self.device, self.dtype = keys.device, keys.dtype
        self._axes = (1, token, head)
        self._layer_bytes = tuple(pool.stride(0) * pool.element_size() for pool in (keys, values))
        # What autograd may have saved (inference tensors count no updates).
        self._counted = tuple(pool for pool in (keys, values) if not pool.is_inference())
        # Bytes from a layer's first element to behind its last.
        self._reach = tuple(_reach(pool[0]) for pool in (keys, values))
        self._geometry = (layout, keys.shape[1:], keys.stride()[1:], values.stride()[1:], keys.dtype, keys.device)
        self._sequences: dict[int, _Sequence] = {}
        self._next = 0
        self._uses = [0] * self.pages
        self._free = list(range(self.pages))
        self._moved = 0   # counts what may move or reuse pages: plans and slots built before it are stale
        self._shared = 0  # counts what may share pages: slots built before it are stale
        self._copied = 0  # counts begun pages copied: places built before it may be another sequence's
        self._copies = None
        self._along = []  # what moves along with the pages

    @classmethod
    def allocate(cls, pages, page_tokens, heads, head_dim, *, layers=1, dtype=torch.bfloat16, device="cuda", layout="BTHD"):
        """A cache over new, uninitialised pools."""
        one_of(layout, _LAYOUTS, "pool layout")
        for value, name in ((pages, "pages"), (page_tokens, "page_tokens"), (heads, "heads"), (head_dim, "head_dim"),
                            (layers, "layers")):
            count(value, name, minimum=1)
        rows = (page_tokens, heads) if layout == "BTHD" else (heads, page_tokens)
        keys, values = (torch.empty((layers, pages, *rows, head_dim), dtype=dtype, device=device) for _ in range(2))
        return cls(keys, values, layout=layout)

    # -----------------------------------------------------------------------------------------
    # Sequences
    # -----------------------------------------------------------------------------------------

    @property
    def free_pages(self):
        return len(self._free)

    def _get(self, sequence):
        found = self._sequences.get(sequence) if type(sequence) is int else None
        if found is None:
            raise StateError(f"there is no sequence {sequence!r} in this cache")
        return found

    def _several(self, sequences):
        sequences = list(sequences)
        found = [self._get(s) for s in sequences]
        need(len(set(sequences)) == len(sequences), "a sequence is named twice")
        return found

    def tokens(self, sequence):
        return self._get(sequence).tokens

    def pages_of(self, sequence):
        """The pages of a sequence in order (:data:`HOLE` where one was dropped)."""
        return list(self._get(sequence).pages)

    def new(self):
        """A new, empty sequence."""
        self._sequences[self._next] = _Sequence([], 0)
        self._next += 1
        return self._next - 1

    def fork(self, sequence):
        """A new sequence with the same tokens: it shares every page.  A page that is not full is copied
        when the first of its sequences goes on."""
        source, uses, child = self._get(sequence), self._uses, self._next
        for page in source.pages:
            if page != HOLE:
                uses[page] += 1
        self._shared += 1
        self._sequences[child] = _Sequence(source.pages[:], source.tokens)
        self._next = child + 1
        return child

    def _release(self, pages):
        for page in pages:
            if page == HOLE:
                continue
            self._uses[page] -= 1
            if self._uses[page] == 0:
                heapq.heappush(self._free, page)

    def free(self, sequence):
        """Drop a sequence; pages that no other one shares become free."""
        pages = self._get(sequence).pages
        del self._sequences[sequence]
        self._release(pages)
        self._moved += 1

    def truncate(self, sequence, tokens):
        """Rewind a sequence to its first ``tokens`` tokens."""
        found = self._get(sequence)
        need(count(tokens, "tokens") <= found.tokens, "a sequence is truncated to what it has")
        keep = -(-tokens // self.page_tokens)
        if keep and found.pages[keep - 1] == HOLE:
            raise StateError("a sequence cannot end in a dropped page")
        self._release(found.pages[keep:])
        del found.pages[keep:]
        found.tokens = tokens
        self._moved += 1

    def drop(self, sequence, first, pages):
        """Drop ``pages`` pages of a sequence from its page ``first`` on (a rolling window): their tokens
        keep their positions and are not attended to any more.  The last page stays."""
        found = self._get(sequence)
        count(first, "first"), count(pages, "pages")
        need(first + pages < max(1, len(found.pages)), "the last page of a sequence cannot be dropped")
        self._release(found.pages[first:first + pages])
        found.pages[first:first + pages] = [HOLE] * pages
        self._moved += 1

    def extend(self, sequences, counts):
        """Room for ``counts[i]`` more tokens of ``sequences[i]``: new pages, and a copy (in every layer)
        of a begun page that other sequences share.  Returns the :class:`Slots` of the new tokens, packed
        sequence after sequence."""
        counts = list(counts)
        found = self._several(sequences)
        need(len(counts) == len(found), "extend takes one count for each sequence")
        for n in counts:
            count(n, "a token count")
        need_gpu(self.device, "a paged cache")
        _refuse_capture(self.device)
        size, in_use, shared = self.page_tokens, self._uses, {}
        wanted, total, most = [], 0, 0  # (rows of a begun page to copy, or 0; new pages) of each sequence
        for item, n in zip(found, counts):
            tokens = item.tokens
            more = -(-(tokens + n) // size) - len(item.pages)
            begun = tokens % size if n else 0
            if begun:
                last = item.pages[-1]
                owners = shared.get(last, in_use[last])
                if owners > 1:
                    shared[last] = owners - 1
                else:
                    begun = 0
            wanted.append((begun, more))
            total += more + (begun > 0)
            most += tokens + n
        need(most < 1 << 31, "a step covers fewer than 2**31 tokens")
        free = self._free
        if shared:
            self._need_copies()
        if total > len(free):
            raise CapacityError(f"{total} pages are needed and {len(free)} are free")
        moves, starts, stamp = [], [], self._shared
        try:
            for item, n, (begun, more) in zip(found, counts, wanted):
                pages = item.pages
                if begun:
                    page = heapq.heappop(free)
                    in_use[page] = 1
                    in_use[pages[-1]] -= 1
                    moves += (pages[-1], page, begun)
                    pages[-1] = page
                    self._shared += 1
                    self._copied += 1
                for _ in range(more):
                    page = heapq.heappop(free)
                    in_use[page] = 1
                    pages.append(page)
                starts.append(item.tokens)
                item.tokens += n
            self._copy(moves)
            return self._slots(found, starts, counts)
        except BaseException:  # no memory, or no launch: as if it had not been called
            shared = moves[::3]
            for item, tokens, (begun, more) in zip(found, starts, wanted):
                pages, item.tokens = item.pages, tokens
                self._release(pages[len(pages) - more - (begun > 0):])
                del pages[len(pages) - more:]
                if begun:
                    pages[-1] = shared.pop(0)
                    in_use[pages[-1]] += 1
            self._shared = stamp
            raise

    def slots(self, sequences, starts, counts):
        """The :class:`Slots` of tokens ``starts[i] .. starts[i] + counts[i]`` that ``sequences[i]`` has
        (rows to write again).  Their pages must not be shared."""
        return self._slots(*self._stretches(sequences, starts, counts, "slots", False))

    def places(self, sequences, starts, counts):
        """The :class:`Places` of tokens ``starts[i] .. starts[i] + counts[i]`` that ``sequences[i]`` has, to read them.
        Their pages may be shared."""
        found, starts, counts = self._stretches(sequences, starts, counts, "places", True)
        made = self._slots(found, starts, counts, Places)
        size = self.page_tokens
        made.pieces = tuple((item, start // size, tuple(item.pages[start // size:-(-(start + n) // size)]))
                            for item, start, n in zip(found, starts, counts) if n)
        made.copied = self._copied
        return made

    def _stretches(self, sequences, starts, counts, what, shared):
        """Checked (sequences, starts, counts) of tokens that lie in pages."""
        found = self._several(sequences)
        starts, counts = list(starts), list(counts)
        need(len(starts) == len(counts) == len(found), f"{what} take one start and count for each sequence")
        for item, start, n in zip(found, starts, counts):
            need(count(start, "a start") + count(n, "a token count") <= item.tokens, f"{what} lie within the sequence")
            if n == 0:
                continue
            for page in item.pages[start // self.page_tokens:(start + n - 1) // self.page_tokens + 1]:
                if page == HOLE:
                    raise StateError(f"the {what}' page was dropped")
                if self._uses[page] > 1 and not shared:
                    raise StateError(f"the {what}' page is shared with another sequence")
        need(sum(counts) < 1 << 31, f"{what} cover fewer than 2**31 tokens")
        need_gpu(self.device, "a paged cache")
        return found, starts, counts

    def _slots(self, found, starts, counts, kind=Slots):
        size = self.page_tokens
        pieces = sum([-(-(start + n) // size) - start // size for start, n in zip(starts, counts) if n])
        if pieces <= _FEW_RUNS:
            runs = []
            for item, at, left in zip(found, starts, counts):
                while left:
                    page, row = divmod(at, size)
                    n = min(left, size - row)
                    runs += (item.pages[page] * size + row, n)
                    at += n
                    left -= n
            with entered(self.device):
                return self._made(upload_runs(runs, sum(counts), self.device), kind)
        pages, base = [], []  # the pages of all tokens, and where each sequence's page 0 would lie among them
        for item, start, n in zip(found, starts, counts):
            first = start // size
            base.append(len(pages) - first)
            pages += item.pages[first:-(-(start + n) // size)]
        counts = np.asarray(counts, dtype=np.int64)
        ends = np.cumsum(counts)
        total = int(ends[-1]) if len(ends) else 0
        at = np.arange(total) + np.repeat(np.asarray(starts, dtype=np.int64) - ends + counts, counts)
        page = at // size
        index = at - page * size
        if total:
            index += np.asarray(pages, dtype=np.int64)[page + np.repeat(np.asarray(base, dtype=np.int64), counts)] * size
        with entered(self.device):
            return self._made(upload(index, self.device), kind)

    def _made(self, index, kind):
        stamp = self._moved if kind is Places else self._moved + self._shared
        return kind(index, index.shape[0], self, stamp, raw_stream(self.device))

    def _current(self, slots):
        """Refuses slots and places of other caches, and those that pages have moved behind."""
        if not isinstance(slots, Slots) or slots.cache is not self:
            raise ConfigurationError("slots come from this cache")
        if not isinstance(slots, Places):
            if slots.stamp != self._moved + self._shared:
                raise StateError("pages moved, were freed or became shared after these slots were built")
            return
        if slots.stamp != self._moved:
            raise StateError("pages moved or were freed after these places were built")
        if slots.copied != self._copied:
            # Sequences went on in copies of their begun pages: these ones, or others.
            if any(tuple(item.pages[first:first + len(pages)]) != pages for item, first, pages in slots.pieces):
                raise StateError("a begun page was copied after these places were built")
            slots.copied = self._copied

    # -----------------------------------------------------------------------------------------
    # Page copies
    # -----------------------------------------------------------------------------------------

    def _need_copies(self):
        """Refuses (before anything changes) what the page copy cannot take."""
        if self.page_tokens * self.heads * self.head_dim * self.keys.element_size() >= 1 << 31:
            raise UnsupportedError("pages of 2 GiB or more cannot be copied")

    def _copy(self, moves):
        """Copies pages in every pool: ``moves`` is flat, (source, destination, leading rows) of each."""
        if not moves:
            return
        along = [(each, pool) for each in self._along if (pool := each.pool()) is not None]
        self._along = [each for each, _ in along]
        with entered(self.device):
            # A copied cache has pools of its own, and others may have come or gone.
            where = self.keys.data_ptr(), self.values.data_ptr(), *[(each, pool.data_ptr()) for each, pool in along]
            if self._copies is None or self._copies[0] != where:
                self._copies = where, [(1, *_pools(pool, self._axes, self.pages, self.page_tokens))
                                       for pool in self._joined_pools()]
                self._copies[1].extend((each.tokens, *_pools((pool,), each.axes, self.pages, pool.shape[each.axes[1]]))
                                       for each, pool in along)
            stream, tables = raw_stream(self.device), {}
            for tokens, pools, fields, streams in self._copies[1]:
                if tokens not in tables:  # a row may stand for several tokens: the begun one moves too
                    tables[tokens] = _pack([-(-word // tokens) if i % 3 == 2 else word for i, word in enumerate(moves)])
                if stream not in streams:  # the allocator learns of a stream that the table was not made on
                    pools.record_stream(torch.cuda.current_stream(self.device))
                    streams.add(stream)
                _lib.check(_lib.function("rch_pages_copy")(fields, tables[tokens], len(moves) // 3, stream))
            torch.autograd.graph.increment_version((*self._counted, *[pool for _, pool in along if not pool.is_inference()]))

    def _take_along(self, pool, axes, tokens=1):
        """Page copies move a further pool ``[layers, pages, rows or heads, .., width]`` from now on, for as long as it lives:
        ``axes`` as of the cache's pools, ``tokens`` of a row."""
        self._along.append(_Along(pool, axes, tokens))

    def _joined_pools(self):
        """K and V pools as one group where their strides agree (one launch), else as two."""
        if self.keys.stride() == self.values.stride():
            return [(self.keys, self.values)]
        return [(self.keys,), (self.values,)]

    def compact(self):
        """Move pages down until those in use are the lowest ones (the highest in use go to the lowest
        free, in order).  Returns the moves as (from, to) pairs."""
        n = self.pages - len(self._free)  # pages in use
        uses = self._uses
        return self._relocate([page for page in range(n, self.pages) if uses[page]], sorted(page for page in self._free if page < n))

    def make_contiguous(self, sequence):
        """Move a sequence's pages to the lowest run of consecutive free pages (for :meth:`view`); pages
        shared with other sequences move for them too.  Nothing moves when they are consecutive."""
        pages = self._get(sequence).pages
        if any(page == HOLE for page in pages):
            raise StateError("a sequence with dropped pages has no consecutive ones")
        if all(b == a + 1 for a, b in zip(pages, pages[1:])):
            return []
        start = run = 0
        for page in sorted(self._free):
            run = run + 1 if run and page == start + run else 1
            start = page if run == 1 else start
            if run == len(pages):
                return self._relocate(list(pages), list(range(start, start + run)))
        raise CapacityError(f"there is no run of {len(pages)} free pages")

    def _relocate(self, source, target):
        """Copies pages ``source[i]`` to the free pages ``target[i]`` and renames them in every sequence."""
        if not source:
            return []
        need_gpu(self.device, "a paged cache")
        _refuse_capture(self.device)
        self._need_copies()
        size, uses, names = self.page_tokens, self._uses, {}
        self._copy([word for a, b in zip(source, target) for word in (a, b, size)])  # where it fails, nothing has changed
        for a, b in zip(source, target):
            uses[b], uses[a] = uses[a], 0
            names[a] = b
        for item in self._sequences.values():
            pages = item.pages
            for at, page in enumerate(pages):
                if page in names:
                    pages[at] = names[page]
        self._free = [page for page, n in enumerate(uses) if not n]  # ascending: a heap
        self._moved += 1
        return list(names.items())

    def load_tables(self, tables):
        """Start over with sequences 0, 1, ... of ``(pages, tokens)`` each (e.g. saved with
        :meth:`pages_of`); the pools keep what they hold.  Sequences may share pages."""
        loaded, uses = {}, [0] * self.pages
        for number, (pages, tokens) in enumerate(tables):
            pages = list(map(int, pages))
            need(len(pages) == -(-count(tokens, "tokens") // self.page_tokens), "the pages do not hold the tokens")
            real = [page for page in pages if page != HOLE] if HOLE in pages else pages
            need(not real or (min(real) >= 0 and max(real) < self.pages), "a page lies outside the pool")
            need(len(set(real)) == len(real), "a sequence has a page twice")
            need(not pages or pages[-1] != HOLE, "the last page of a sequence cannot be a hole")
            for page in real:
                uses[page] += 1
            loaded[number] = _Sequence(pages, tokens)
        self._sequences, self._uses, self._next = loaded, uses, len(loaded)
        self._free = [page for page, n in enumerate(uses) if not n]
        self._moved += 1
        return list(loaded)

    def page_table(self, sequences):
        """int32 ``[sequences, most pages]`` on the device; :data:`HOLE` behind a sequence's last page."""
        tables = [self._get(s).pages for s in sequences]
        need_gpu(self.device, "a paged cache")
        width = max(map(len, tables), default=0)
        words = []
        for pages in tables:
            words += pages
            words += [HOLE] * (width - len(pages))
        shape = (len(tables), width)
        with entered(self.device):
            if len(words) <= _ARGUMENT_WORDS:
                return upload_words(_pack(words), shape, self.device)
            return upload(np.asarray(words, dtype=np.int32).reshape(shape), self.device)

    # -----------------------------------------------------------------------------------------
    # Contents
    # -----------------------------------------------------------------------------------------

    def _layer(self, layer):
        need(count(layer, "layer") < self.layers, "there is no such layer")
        return self.keys[layer], self.values[layer]

    def view(self, layer, target, sequence, start, tokens):
        """The slot of ``tokens`` tokens of a sequence as a restore destination: a
        :class:`~reelcache_amd.restore_model.NativeView` (:class:`PageView`) of the layer's K (``target="k"``)
        or V (``"v"``) pool, which a restore takes as long as its pages are the sequence's alone.  The tokens
        lie in one page, or in consecutive pages of a ``"BTHD"`` pool whose token rows follow each other across
        pages (:meth:`make_contiguous`)."""
        one_of(target, ("k", "v"), "target")
        pool = self._layer(layer)[target == "v"]
        found = self._get(sequence)
        need(count(start, "start") + count(tokens, "tokens", minimum=1) <= found.tokens, "the view lies within the sequence")
        first, last = start // self.page_tokens, (start + tokens - 1) // self.page_tokens
        pages = found.pages[first:last + 1]
        if HOLE in pages:
            raise StateError("the view's page was dropped")
        if any(self._uses[page] > 1 for page in pages):
            raise StateError("the view's page is shared with another sequence")
        offset = start - first * self.page_tokens
        where = self, sequence, first, tuple(pages), found, start + tokens
        if first == last:
            return PageView(pool, self.layout, offset, pages[0], *where)
        joined = self.layout == "BTHD" and pool.stride(0) == self.page_tokens * pool.stride(1)
        if not joined or any(b != a + 1 for a, b in zip(pages, pages[1:])):
            raise StateError("the view's pages do not follow each other; see make_contiguous")
        flat = pool.as_strided((self.pages * self.page_tokens, self.heads, self.head_dim), pool.stride()[1:])
        return PageView(flat, "THD", pages[0] * self.page_tokens + offset, 0, *where)

    def store(self, layer, slots, keys, values, *, positions=None, grid=None):
        """Write new tokens into their slots (a backward pass that saved a pool notices): ``keys`` turned by
        ``positions`` (interleaved pairs, which need an even ``head_dim``, as :func:`reelcache_amd.rotary.rotate`;
        ``None`` stores them as they are) and ``values``, both
        ``[tokens, heads, head_dim]`` of the cache's dtype, any strides (rows of the pools themselves are
        copied first).  With a ``grid`` the tokens are one chunk."""
        if type(layer) is not int or not 0 <= layer < self.layers:
            raise ConfigurationError("there is no such layer")
        self._current(slots)
        if isinstance(slots, Places):
            raise ConfigurationError("a store takes slots, not places")
        shape = (slots.tokens, self.heads, self.head_dim)
        for x, name in ((keys, "keys"), (values, "values")):
            in_memory(x, name)
            if x.shape != shape or x.dtype != self.dtype or x.device != self.device:
                raise ConfigurationError(f"{name} must be [tokens, heads, head_dim] of the cache's dtype and device")
            if x.requires_grad and torch.is_grad_enabled():
                raise ConfigurationError("a store is not differentiable; run it under torch.no_grad()")
        if slots.tokens == 0:
            return
        need_gpu(self.device, "a paged cache")
        grid = None if grid is None else tuple(grid)
        with entered(self.device):
            sources = [x if x.stride(2) == 1 or self.head_dim == 1 else x.contiguous() for x in (keys, values)]
            known = known_calls(slots if positions is None else positions)
            key = (slots.tokens, grid, self._geometry, *[x.stride() for x in sources])
            call = known.get(key)
            if call is None:
                call = known[key] = (self._store_launch(sources, positions, grid, slots.tokens), *map(_reach, sources))
            launch, *reach = call
            stream = raw_stream(self.device)
            k_bytes, v_bytes = self._layer_bytes
            pools = [self.keys.data_ptr() + layer * k_bytes, self.values.data_ptr() + layer * v_bytes]
            if pools[0] == pools[1]:
                raise ConfigurationError("a store needs keys and values in pools of their own")
            k, v = sources[0].data_ptr(), sources[1].data_ptr()
            for pool, room in zip(pools, self._reach):
                if (k < pool + room and pool < k + reach[0]) or (v < pool + room and pool < v + reach[1]):
                    # Rows of the pool itself, which are written while others are still read: of copies.
                    return self.store(layer, slots, *[x.clone(memory_format=torch.contiguous_format) for x in (keys, values)],
                                      positions=positions, grid=grid)
            self._launch_store(launch, layer, (k, v), pools, addresses_of(positions, self.device, stream),
                               slots.index.data_ptr(), stream)
            if stream != slots.stream:  # the allocator learns of a stream that the index was not made on
                slots.index.record_stream(torch.cuda.current_stream(self.device))
            torch._C._increment_version(self._counted)

    def _launch_store(self, launch, layer, sources, pools, turned, slots, stream):
        launch([(sources[0], pools[0], True), (sources[1], pools[1], False)], *turned, slots, stream)

    def _store_launch(self, sources, positions, grid, tokens):
        turned = position_fields(positions, grid, tokens, 1, self.head_dim, self.device)
        jobs = []
        for x, pool, (pairs, place) in zip(sources, (self.keys, self.values), (turned, (0, (0,) * 16))):
            page, token, head = (pool.stride(axis) for axis in self._axes)
            jobs.append((0, 0, 1, tokens, self.heads, self.head_dim, pairs, 0, x.stride(0), x.stride(1), page, token, head,
                         *place, 0, self.pages * self.page_tokens, self.page_tokens, 0, 0))
        return Launch(jobs, self.dtype, "interleaved")

    # -----------------------------------------------------------------------------------------
    # Attention
    # -----------------------------------------------------------------------------------------

    def plan(self, sequences, queries, *, heads, block=None, window=None, scale=None):
        """The :class:`~reelcache_amd.attention.AttentionPlan` of one step: ``queries[i]`` new tokens (the
        last ones) of ``sequences[i]`` attend to it.  Built once, used by :meth:`attend` in every layer."""
        from .attention import AttentionPlan

        return AttentionPlan(self, sequences, queries, heads=heads, block=block, window=window, scale=scale)

    def attend(self, layer, q, plan, *, out=None, return_lse=False):
        """:func:`reelcache_amd.attention.attend` over one layer."""
        from .attention import AttentionPlan, attend, run

        if type(layer) is not int or not 0 <= layer < self.layers:
            raise ConfigurationError("there is no such layer")
        if not isinstance(plan, AttentionPlan) or plan.cache is not self or plan._block_tokens:
            return attend(q, *self._layer(layer), plan, out=out, return_lse=return_lse)
        k_bytes, v_bytes = self._layer_bytes
        return run(q, self.keys.data_ptr() + layer * k_bytes, self.values.data_ptr() + layer * v_bytes, plan, out, return_lse,
                   self._pools(), self._scales(layer))

    def _pools(self):
        """What no output may overlap."""
        return self.keys, self.values

    def _scales(self, layer):
        """Addresses of a layer's scales, of pools in codes."""
        return 0, 0

    def _scale_strides(self):
        """(page, head) strides of the keys' and the values' scales."""
        return 0, 0, 0, 0

    def index(self, block_tokens):
        """A new :class:`~reelcache_amd.sparse_attention.BlockIndex` of the keys, in blocks of ``block_tokens``."""
        from .sparse_attention import BlockIndex

        return BlockIndex.allocate(self, block_tokens)


class _Along:
    """A further pool that moves with the pages: its owner keeps it, not the cache."""

    def __init__(self, pool, axes, tokens):
        self.pool = weakref.ref(pool) if pool is not None else _gone
        self.axes, self.tokens = axes, tokens

    def __reduce__(self):  # copies are of the pool's copy
        return _Along, (self.pool(), self.axes, self.tokens)


def _gone():
    return None


def _apart(pool):
    """Whether every element of a strided tensor has a place of its own (strides sorted, each at least the
    reach of those below it)."""
    reach = 1
    for stride, size in sorted((stride, size) for size, stride in zip(pool.shape, pool.stride()) if size > 1):
        if stride < reach:
            return False
        reach = stride * (size - 1) + reach
    return True


def _reach(x):
    """Bytes from a strided tensor's first element to behind its last."""
    low, high = _span(x)
    return high - low


def _pools(group, axes, pages, page_tokens):
    """(device table of pool addresses, ``rch_pages`` fields, streams the table is known to) of pools with the
    same strides."""
    size = group[0].element_size()
    stride = group[0].stride()
    page, token, head = (stride[axis] * size for axis in axes)
    heads, row = group[0].shape[axes[2]], group[0].shape[4] * size
    addresses = [pool.data_ptr() + layer * stride[0] * size for pool in group for layer in range(pool.shape[0])]
    table = torch.tensor(addresses, dtype=torch.int64).to(group[0].device)  # waits: usable on every stream
    joined = head == row or heads == 1  # a token's heads are one run
    segments, segment, width = (1, 0, heads * row) if joined else (heads, head, row)
    mix = 0
    for address in addresses:
        mix |= address
    fields = (table.data_ptr(), len(addresses), pages, page if pages > 1 else 0, page_tokens, segments, segment,
              token if page_tokens > 1 else width, width, mix)
    return table, (ctypes.c_int64 * len(fields))(*fields), {raw_stream(group[0].device)}


__all__ = ["HOLE", "PageView", "PagedCache", "Places", "Slots"]
