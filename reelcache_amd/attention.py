"""Attention of new tokens over a paged cache.

The tokens of a step (a chunk of a video, a prompt, one token of each of many sequences) attend to the
pages of their sequence, themselves included once they are stored.  :class:`AttentionPlan` lays the
step's work out on the host once: which rows of queries meet which keys in which workgroup, so that the
card is filled whatever the lengths; every layer's :func:`attend` then runs that plan
(``rch_attend_run``).

Masks: a query at place ``p`` of its sequence (the last query stands at the last token) sees every key
of the sequence, or with ``block`` those before the end of its own block of that many tokens
(``block=1``: causal; ``block=frame tokens``: causal over frames), and with ``window`` only keys after
``p - window``.  Dropped pages are not seen.  A query that sees nothing gets zeros.  Keys and values
that a query does not see have no influence on it, whatever their slots hold.
"""

from __future__ import annotations

import ctypes
import math
import struct

import numpy as np
import torch

from . import _lib
from ._checks import count, in_memory, need
from .errors import ConfigurationError, StateError, UnsupportedError
from .rotary import _DTYPE_CODES, _span, changed, entered, known_calls, need_gpu, raw_stream

#: Keys of a tile: the step of every split of a sequence's keys.
KEY_TILE = 64
#: Query rows (tokens x heads of a key head) of one workgroup's tile, per form.
GENERAL_ROWS, ROW_TILE = 16, 128
# What a workgroup's start, end and partial results cost in key tiles, per form (tiled: a step of six sequences of
# 211 to 5003 tokens takes 58.0 us at 0, 55.4 at 3, 54.8 at 6 and 55.0 at 8; others do not change by more than 2 %).
_OVERHEAD = {"general": 1, "rows": 6}
_CUS = 256
# At most this many rows are joined a workgroup to a row, whatever their parts, in one launch (512 rows of 4 parts take
# 4.1 us so, 4.1-5.1 us with a thread per eight channels; a second launch costs 5 us).
_FEW_ROWS = 512
_XCDS = 8
_MOST_KEYS = 2 ** 31 - 4096
# Scales that stay normal fp32 numbers with log2(e) in them.
_LEAST_SCALE, _MOST_SCALE = 2.0 ** -126, 2.0 ** 127


class _Work:
    """The row blocks of a step: parallel int64 arrays, one entry per (sequence, key head, row block)."""

    def __init__(self):
        self.parts = []

    def add(self, sequence, kv_heads, rows, tile, keys_of):
        begin = np.arange(0, rows, tile, dtype=np.int64)
        end = np.minimum(begin + tile, rows)
        first, last = keys_of(begin, end)
        block = np.stack([np.full_like(begin, sequence), begin, end, first, last], axis=1)
        heads = np.repeat(np.arange(kv_heads, dtype=np.int64), len(block))
        self.parts.append(np.concatenate([np.tile(block, (kv_heads, 1)), heads[:, None]], axis=1))

    def rows(self):
        """int64 [n, 6]: sequence, row begin, row end, first key, last key, key head."""
        return np.concatenate(self.parts) if self.parts else np.empty((0, 6), np.int64)


def _share_out(tiles, owner, resident, overhead):
    """The parts of row blocks of ``tiles`` key tiles (``rch_attend_share``): int64 [parts, 4] of (block,
    first tile, last tile, XCD), block after block.  The blocks of one ``owner`` (they share keys) go to one
    XCD as far as the XCDs stay evenly loaded, and are cut so that an XCD's workgroups end together."""
    tiles, owner = (np.ascontiguousarray(x, dtype=np.int64) for x in (tiles, owner))
    parts = np.empty((len(tiles) + 2 * resident + 16, 4), np.int64)
    count = ctypes.c_int64(0)
    _lib.check(_lib.function("rch_attend_share")(tiles.ctypes.data, owner.ctypes.data, len(tiles), resident, overhead,
                                                 parts.ctypes.data, len(parts), ctypes.byref(count)))
    return parts[:count.value]


class AttentionPlan:
    """The work of one step: ``queries[i]`` new tokens of ``sequences[i]`` of a
    :class:`~reelcache_amd.paged_cache.PagedCache` attend to it with ``heads`` query heads (a multiple of
    the cache's), packed sequence after sequence.

    ``block``, ``window``: see the module docstring (``None``: no such bound).  ``scale``: a positive
    factor of the scores (default ``head_dim ** -0.5``).  The plan is bound to the pages that the
    sequences have now; it is stale once pages move or are freed, and it keeps reading a begun page that a
    later ``extend`` copies for its sequence (plans are made after the step's ``extend``).  Its tables are
    written on the stream
    that is current (other streams wait for it).  A captured graph keeps its plan's tables as they are:
    keep the plan as long as the graph.
    """

    def __init__(self, cache, sequences, queries, *, heads, block=None, window=None, scale=None):
        found = cache._several(sequences)
        queries = [count(n, "a query count") for n in queries]
        need(len(queries) == len(found), "a plan takes one query count for each sequence")
        count(heads, "heads", minimum=1)
        need(heads % cache.heads == 0, "query heads must be a multiple of the cache's heads")
        for value, name in ((block, "block"), (window, "window")):
            need(value is None or count(value, name, minimum=1) < 1 << 31, f"{name} must be below 2**31")
        scale = cache.head_dim ** -0.5 if scale is None else scale
        need(isinstance(scale, (int, float)) and not isinstance(scale, bool) and _LEAST_SCALE <= scale <= _MOST_SCALE,
             "scale must be a positive number that fp32 holds")
        if cache.head_dim > _lib.ATTEND_MAX_DIM:
            raise UnsupportedError(f"attention takes at most {_lib.ATTEND_MAX_DIM} channels to a head")
        need_gpu(cache.device, "attention")
        # The kernels step over keys and pages in 32 bits, up to a few tiles past a sequence's last page.
        need(all(len(item.pages) * cache.page_tokens <= _MOST_KEYS for item in found),
             f"attention takes sequences of at most {_MOST_KEYS} tokens, their last page whole")
        self.cache, self.heads, self.queries = cache, heads, sum(queries)
        self.group = heads // cache.heads
        need(self.queries * self.group < 1 << 31, "a step has fewer than 2**31 query rows")
        self.block, self.window, self.scale = block, window, float(scale)
        self._stamp = cache._moved
        self._lay_out(found, queries)

    # -----------------------------------------------------------------------------------------

    def _keys_of(self, length, queries):
        """Function of row ranges: the keys that any row of a range may see (empty: first == last)."""
        group, block, window = self.group, self.block, self.window

        def keys(begin, end):
            place0, place1 = (length - queries + at // group for at in (begin, end - 1))
            first, last = np.zeros_like(begin), np.full_like(begin, length)
            if block:
                last = np.minimum(last, np.where(place1 < 0, 0, (place1 // block + 1) * block))
            if window:
                first = np.clip(place0 - window + 1, 0, length)
            return first, np.maximum(first, last)

        return keys

    def _form(self):
        """The kernels that take the cache: "rows", which tile for the matrix cores, or "general"."""
        cache = self.cache
        size = cache.keys.element_size()
        aligned = all(pool.data_ptr() % 16 == 0 and all(pool.stride(a) * size % 16 == 0 for a in range(4))
                      for pool in (cache.keys, cache.values))
        if not (aligned and cache.head_dim * size % 16 == 0 and cache.head_dim <= _lib.ATTEND_FAST_DIM):
            return "general"
        if max(cache.keys.stride(cache._axes[1]), cache.values.stride(cache._axes[1])) > 1 << 22:
            return "general"
        return "rows"

    def _lay_out(self, found, queries):
        cache = self.cache
        form, work = self._form(), _Work()
        tile = ROW_TILE if form == "rows" else GENERAL_ROWS
        table, at, lengths, starts = [], [], [], []
        words, row = _lib.ATTEND_ZEROS, 0
        for number, (item, n) in enumerate(zip(found, queries)):
            lengths.append(item.tokens)
            starts.append(row)
            at.append(words)
            table.extend(item.pages)
            words += len(item.pages)
            row += n
            if n:
                work.add(number, cache.heads, n * self.group, tile, self._keys_of(item.tokens, n))
        need(words < 1 << 30, "the step's page tables are too large")
        self._at = np.asarray(at, dtype=np.int64)
        self._lengths, self._starts = np.asarray(lengths, dtype=np.int64), np.asarray(starts, dtype=np.int64)
        self._counts = np.asarray(queries, dtype=np.int64)
        merges, self._partial_rows = [], 0
        items = self._split(form, work.rows(), merges)
        merges = np.concatenate(merges) if merges else np.empty((0, _lib.ATTEND_MERGE), np.int64)
        self._counts_of = (0, len(items)) if form == "rows" else (len(items), 0)
        first_item = _lib.ATTEND_ZEROS + len(table)
        self._items, self._merges = first_item, first_item + items.size
        # Merges that take a workgroup to a row come first (the kernels' rule).
        joined = form == "rows" and cache.head_dim % 8 == 0
        many = (merges[:, 5] > _lib.ATTEND_FEW_PARTS) | (not joined)
        if len(merges) * merges[:, 2].max(initial=0) <= _FEW_ROWS:
            many[:] = True
        merges = np.concatenate([merges[many], merges[~many]])
        self._n_merges, self._n_many = len(merges), int(many.sum())
        self._most_rows = [int(part[:, 2].max(initial=0)) for part in np.split(merges, [self._n_many])]
        self._holes = int(any(page < 0 for page in table))
        need(self._partial_rows < 1 << 31, "the step's partial results are too many")
        words = np.concatenate([np.zeros(_lib.ATTEND_ZEROS, np.int64), np.asarray(table, np.int64), items.ravel(),
                                merges.ravel()])
        from .paged_cache import upload

        self._tiled = self._counts_of[1]
        with entered(cache.device):
            self.buffer = upload(words, cache.device)
            self._stream = raw_stream(cache.device)

    def _unit(self):
        """Tokens that tiles of keys start over at: a page where tiles stay within pages, else a tile."""
        # Tiles that stay in a page leave the page's last one part empty; tiles across pages cost nothing more
        # where a wave's rows of a tile (16, fp32: 8) lie in one page, and 30 % more (an address for every row)
        # where they do not: a chunk's 2340 queries over 9360 keys, 12 heads, take 169-174 us either way, 225 us
        # with addresses, and 193 us in pages of 390 tokens, 230 us in pages of 200, 274 us in pages of 100.
        # The kernels look a tile's page up once where tiles stay within pages, so those hold a tile at least.
        size = self.cache.page_tokens
        if size < KEY_TILE:
            return KEY_TILE
        share = 16 if self.cache.keys.element_size() == 2 else 8
        held = -(-size // KEY_TILE) * KEY_TILE  # rows of tiles that a page takes
        return size if held == size or (size % share and 5 * held <= 6 * size) else KEY_TILE

    def _resident(self, form):
        """Workgroups of a form that the card holds at once."""
        if form == "general":
            return _CUS * 4
        dim = self.cache.head_dim  # its tiles fill LDS and registers
        return _CUS * (3 if dim <= 64 else 2 if dim <= 128 else 1)

    def _tile_of(self, key):
        """Index of the tile that holds ``key``, and the first key of a tile."""
        unit = self._unit()
        return key // unit * -(-unit // KEY_TILE) + key % unit // KEY_TILE

    def _key_of(self, tile):
        unit = self._unit()
        per = -(-unit // KEY_TILE)
        return tile // per * unit + tile % per * KEY_TILE

    def _split(self, form, blocks, merges):
        """Items of a form's row blocks, in launch order: the keys of a block in one part, or in as many as
        let the card's workgroups end together."""
        if not len(blocks):
            return np.empty((0, _lib.ATTEND_ITEM), np.int64)
        sequence, begin, end, first, last, head = blocks.T
        tile0 = self._tile_of(first)
        tiles = np.where(last > first, self._tile_of(np.maximum(last - 1, 0)) + 1 - tile0, 0)
        owner = sequence * self.cache.heads + head
        which, low, high, xcd = _share_out(tiles, owner, self._resident(form), _OVERHEAD[form]).T
        parts = np.bincount(which, minlength=len(blocks))
        part = np.arange(len(which)) - np.repeat(np.cumsum(parts) - parts, parts)
        n = parts[which]
        rows = (end - begin)[which]
        # Partial rows: part after part of a block, block after block.
        need_rows = np.where(parts > 1, parts * (end - begin), 0)
        base = self._partial_rows + np.cumsum(need_rows) - need_rows
        self._partial_rows += int(need_rows.sum())
        items = np.zeros((len(which), _lib.ATTEND_ITEM), np.int64)
        items[:, 0] = self._at[sequence][which]
        items[:, 1] = self._lengths[sequence][which]
        items[:, 2] = self._starts[sequence][which]
        items[:, 3] = self._counts[sequence][which]
        items[:, 4], items[:, 5], items[:, 6] = begin[which], end[which], head[which]
        items[:, 7] = np.where(part == 0, first[which], self._key_of(tile0[which] + low))
        items[:, 8] = np.where(part == n - 1, last[which], np.minimum(last[which], self._key_of(tile0[which] + high)))
        items[:, 9] = np.where(n > 1, base[which] + part * rows, -1)
        several = parts > 1
        if several.any():
            rows = (end - begin)[several]
            merge = np.zeros((len(rows), _lib.ATTEND_MERGE), np.int64)
            merge[:, 0], merge[:, 1], merge[:, 2] = self._starts[sequence[several]], begin[several], rows
            merge[:, 3], merge[:, 4], merge[:, 5] = head[several], base[several], parts[several]
            merges.append(merge)
        return self._ordered(items, high - low, xcd)

    @staticmethod
    def _ordered(items, cost, xcd):
        """Items in launch order: workgroup b runs on XCD b % 8, so the i-th longest item of XCD x stands at
        8 i + x; empty items fill up the XCDs that have fewer."""
        if len(items) <= _XCDS:
            return items[np.argsort(-cost, kind="stable")]
        buckets = [np.flatnonzero(xcd == x) for x in range(_XCDS)]
        out = np.zeros((max(len(bucket) for bucket in buckets), _XCDS, _lib.ATTEND_ITEM), np.int64)
        out[:, :, 9] = -1
        for x, bucket in enumerate(buckets):
            out[:len(bucket), x] = items[bucket[np.argsort(-cost[bucket], kind="stable")]]
        return out.reshape(-1, _lib.ATTEND_ITEM)

    # -----------------------------------------------------------------------------------------

    def _check(self, keys, values):
        cache = self.cache
        shape, k_stride, v_stride = cache.keys.shape[1:], cache.keys.stride()[1:], cache.values.stride()[1:]
        for pool, stride, name in ((keys, k_stride, "keys"), (values, v_stride, "values")):
            in_memory(pool, name)
            need(pool.shape == shape and pool.stride() == stride and pool.dtype == cache.dtype
                 and pool.device == cache.device, f"{name} must be a layer's pool like those of the plan's cache")
            need(self._tiled == 0 or pool.data_ptr() % 16 == 0, f"{name} must be aligned as the plan's cache is")
            need(not (pool.requires_grad and torch.is_grad_enabled()),
                 "attention over a cache is not differentiable; run it under torch.no_grad()")

    def _fields(self, q_stride, out_stride):
        """The ``rch_attend`` image of a call: everything but the addresses."""
        cache = self.cache
        page, token, head = cache._axes
        k, v = cache.keys.stride(), cache.values.stride()
        scale = struct.unpack("<i", struct.pack("<f", self.scale * math.log2(math.e)))[0]
        fields = (0, 0, 0, 0, 0, 0, 0, *q_stride, k[page], k[token], k[head], v[page], v[token], v[head], *out_stride,
                  self.group, self.heads, cache.head_dim, cache.page_tokens, cache.pages, self.block or 0, self.window or 0,
                  scale, self._partial_rows, self._items, *self._counts_of, self._merges, self._n_merges, self._n_many,
                  *self._most_rows, self._holes, self._unit())
        return bytes(_Image(*fields))


_Image = ctypes.c_int64 * len(_lib.ATTEND_FIELDS)


def attend(q, keys, values, plan, *, out=None, return_lse=False):
    """Attention of ``q`` over one layer's pools by ``plan``.

    ``q``: ``[rows, heads, head_dim]`` of the cache's dtype, any strides; its first ``plan.queries`` rows
    are the plan's.  ``keys``, ``values``: one layer of the plan's cache.  ``out``: where to write, of
    q's shape (rows behind the plan's stay as they are); without it a new tensor, zero behind them.
    ``return_lse``: also the fp32 ``[rows, heads]`` natural logs of the sums of exponentials (-inf for a
    query that sees nothing), by which the results over two caches join.  A query whose scores are all
    -inf gets NaN, as their softmax has no value (and a log of -inf).

    Scores, weights and sums are held in fp32; for the product with 16-bit values the weights are rounded to
    their type (half a step each, averaged over the keys), and the output is rounded once.  Keys meet the
    queries as the pools hold them: both are rotated before.  Runs on the current stream; not
    differentiable.  Returns ``out``, or ``(out, lse)``.
    """
    need(isinstance(plan, AttentionPlan), "attend needs an AttentionPlan")
    plan._check(keys, values)
    return run(q, keys.data_ptr(), values.data_ptr(), plan, out, return_lse, (keys, values))


def run(q, k_address, v_address, plan, out, return_lse, pools=None):
    """:func:`attend` over a layer's checked pools, given by their addresses."""
    cache = plan.cache
    if plan._stamp != cache._moved:
        raise StateError("pages moved or were freed after this plan was built")
    in_memory(q, "q")
    shape = q.shape
    if len(shape) != 3 or shape[0] < plan.queries or shape[1] != plan.heads or shape[2] != cache.head_dim:
        raise ConfigurationError("q must be [rows, heads, head_dim] with a row for every query of the plan")
    device = cache.device
    if q.dtype != cache.dtype or q.device != device:
        raise ConfigurationError("q must have the cache's dtype and device")
    if q.requires_grad and torch.is_grad_enabled():
        raise ConfigurationError("attention over a cache is not differentiable; run it under torch.no_grad()")
    with entered(device):
        given, q = q, _rows(q)
        more, given_out = shape[0] > plan.queries, out is not None
        result = out
        if out is None:
            result = out = torch.empty(shape, dtype=q.dtype, device=device)
            if more:
                out[plan.queries:].zero_()
        else:
            result = _output(out, given, pools or (cache.keys, cache.values))
        lse = None
        if return_lse:
            lse = torch.empty((shape[0], plan.heads), dtype=torch.float32, device=device)
            if more:
                lse[plan.queries:].fill_(-math.inf)
        if plan.queries:
            known = known_calls(plan)
            key = (q.stride(), result.stride())
            image = known.get(key)
            if image is None:
                image = known[key] = plan._fields(q.stride()[:2], result.stride()[:2])
            fields = _Image.from_buffer_copy(image)
            partials = None
            if plan._n_merges:
                partials = torch.empty(plan._partial_rows * (cache.head_dim + 2) + 1, dtype=torch.float32, device=device)
                fields[6] = partials.data_ptr()
            stream = raw_stream(device)
            if stream != plan._stream:  # the allocator learns of a stream that the tables were not made on
                plan.buffer.record_stream(torch.cuda.current_stream(device))
            fields[0], fields[1], fields[2], fields[3] = q.data_ptr(), k_address, v_address, result.data_ptr()
            fields[4], fields[5] = 0 if lse is None else lse.data_ptr(), plan.buffer.data_ptr()
            _lib.check(_lib.function("rch_attend_run")(fields, _DTYPE_CODES[q.dtype], stream))
            if result is not out:
                out[:plan.queries].copy_(result[:plan.queries])
            elif given_out:
                changed(out)
    return (out, lse) if return_lse else out


def _output(out, q, pools):
    """Where the kernels write for a given ``out``: itself, or a buffer when its rows are not aligned."""
    in_memory(out, "out")
    need(out.shape == q.shape and out.dtype == q.dtype and out.device == q.device, "out must match q")
    need(not out.requires_grad, "out must not require gradients")
    need(all(stride != 0 or size <= 1 for size, stride in zip(out.shape, out.stride())),
         "out with broadcast (zero) strides aliases itself")
    low, high = _span(out)
    for x in (q, *pools):
        same = x is q and out.data_ptr() == x.data_ptr() and out.stride() == x.stride()
        first, last = _span(x)
        need(same or high <= first or last <= low, "out overlaps an input without being q")
    return out if _aligned(out) else torch.empty(out.shape, dtype=out.dtype, device=out.device)


def _aligned(x):
    size = x.element_size()
    a, b, c = x.stride()
    return c == 1 and (x.data_ptr() | a * size | b * size) % 16 == 0


def _rows(q):
    """``q`` as the kernels read it in place (16-byte rows), else a copy; a head_dim whose rows cannot be
    16-byte aligned only runs in the general form, which needs unit stride alone."""
    if _aligned(q) or (q.shape[2] * q.element_size() % 16 and (q.stride(2) == 1 or q.shape[2] == 1)):
        return q
    return q.clone(memory_format=torch.contiguous_format)


__all__ = ["AttentionPlan", "attend"]
