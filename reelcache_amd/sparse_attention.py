"""Attention to chosen blocks of a paged cache: of a long history, the part that a cheap score finds worth its time.

:class:`BlockIndex` keeps the mean key of every block of ``block_tokens`` tokens (they divide a page) beside a cache's
pages, shared, copied and moved with them.  A step's queries are cut into runs of ``query_block`` tokens; for each run and
key head, :meth:`BlockIndex.select` scores the blocks by the sum of the run's query rows times the mean key
(``rch_blocks_select``), and :meth:`BlockIndex.attend` attends to the chosen ones (``rch_attend_run``).

Of the blocks that any query of a run sees, these are taken:

* those that not every query of the run sees whole (the run's own blocks under a causal mask, the borders of windows and
  frames) and those that are not full: their mean would tell of keys that a query does not see;
* the sequence's ``first`` leading blocks, and the ``recent`` blocks up to the one of the run's last query;
* of the others the ``top`` best scores; equal ones by the lower number, a NaN above all.

So no key that a query does not see has an influence on it, as in dense attention, and with ``top`` as large as the
history the result is the dense one.  Dropped pages are neither scored nor taken.  Scores are sums in FP64, so a choice
does not depend on the order of a sum; selection is not differentiable, nor is the attention.
"""

from __future__ import annotations

import ctypes

import numpy as np
import torch

from . import _lib
from ._checks import count, in_memory, need
from .attention import AttentionPlan, _ROWS, run
from .errors import ConfigurationError, StateError, UnsupportedError
from .paged_cache import HOLE
from .rotary import _DTYPE_CODES, entered, known_calls, need_gpu, raw_stream

_MOST_SCORED = 65535 * 128  # blocks of a run: one workgroup scores 128
# Blocks are scored in a launch of their own where a run scores more than _FEW_SCORED of them and there are fewer than
# _FEW_RUNS workgroups else (choice and attention, apart / together: 4 tokens of 8 key heads among 1000 blocks 29.7 / 38.9 us,
# 8 among 500 32.9 / 34.4, 4 among 125 27.2 / 23.7, 16 among 500 43.5 / 43.8, 39 runs of 12 heads among 270 150.9 / 139.9).
_FEW_SCORED, _FEW_RUNS = 256, 128
# Bytes of the numbers of blocks scored apart (8 for each block, run and key head; one run's at least): a step that needs more
# chooses run after run, in launches that follow each other (4680 runs of 12 key heads among 8192 blocks: 22.3 ms with 3.7 GB,
# 1 GB or this, 22.5 with 64 MiB, 24.0 with 16).
_SCORE_BYTES = 1 << 28
_Image = ctypes.c_int64 * len(_lib.BLOCKS_FIELDS)
_KEYS_AT, _SCALES_AT, _SLOTS_AT, _Q_AT, _PLAN_AT, _RUNS_AT, _SCORES_AT, _LISTS_AT = (
    _lib.BLOCKS_FIELDS.index(name)
    for name in ("keys_ptr", "scales_ptr", "slots_ptr", "q_ptr", "plan_ptr", "runs", "scores_ptr", "lists_ptr"))


class BlockPlan(AttentionPlan):
    """The work of one step of attention to chosen blocks: an :class:`~reelcache_amd.attention.AttentionPlan` whose queries
    are cut into runs (from a sequence's first new token on) that choose their blocks together.  Built by
    :meth:`BlockIndex.plan`, used by :meth:`BlockIndex.select` and :meth:`BlockIndex.attend` in every layer; stale once pages
    moved, and to be built after the step's ``extend``, as every plan.

    ``runs``: their number.  ``counts``: blocks that each takes (of every key head).  ``width``: the most of them.
    """

    def __init__(self, index, sequences, queries, *, heads, top, query_block=1, first=1, recent=1, block=None, window=None,
                 scale=None):
        self.index = index
        for value, name, least in ((top, "top", 0), (query_block, "query_block", 1), (first, "first", 0), (recent, "recent", 0)):
            need(count(value, name, minimum=least) < 1 << 31, f"{name} must be below 2**31")
        self.top, self.query_block, self.first, self.recent = top, query_block, first, recent
        self._block_tokens = index.block_tokens
        super().__init__(index.cache, sequences, queries, heads=heads, block=block, window=window, scale=scale)

    def _runs_of(self, length, queries):
        """The runs of one sequence: (first query, query behind the last, then blocks as pairs of first and last:
        seen by any query; full and seen whole by every query, and among them those taken anyway)."""
        size = self._block_tokens
        begin = np.arange(0, queries, self.query_block, dtype=np.int64)
        end = np.minimum(begin + self.query_block, queries)
        keys = self._keys_of(length, queries)
        group = self.group
        (low, high0), (low1, high) = (keys(at * group, at * group + 1) for at in (begin, end - 1))
        any_key = high > low
        seen = np.where(any_key, low // size, 0), np.where(any_key, -(-high // size), 0)
        # Whole blocks of every query; the leading ones are not scored.
        first = np.minimum(np.maximum(-(-low1 // size), np.maximum(seen[0], self.first)), seen[1])
        last = np.maximum(np.minimum(high0 // size, seen[1]), first)
        own = (length - queries + end - 1) // size  # floor: below 0 for places before the first key
        kept = np.clip(own - self.recent + 1, first, last), np.clip(own + 1, first, last)
        return begin, end, *seen, first, last, kept[0], np.maximum(*kept)

    def _lay_out(self, found, queries):
        cache, group, size = self.cache, self.group, self._block_tokens
        form = self._form_of(min(self.query_block, max(queries, default=0)))
        table = self._tables(found, queries)
        runs, counts = [], []
        for number, (item, n) in enumerate(zip(found, queries)):
            if not n:
                continue
            begin, end, *ranges = self._runs_of(item.tokens, n)
            # Blocks that lie in pages before each block.
            held = np.asarray(item.pages, dtype=np.int64) != HOLE
            held = np.concatenate([[0], np.cumsum(np.repeat(held, cache.page_tokens // size))])
            seen, scored, kept = (held[b] - held[a] for a, b in zip(ranges[::2], ranges[1::2]))
            scored -= kept
            counts.append(seen - scored + np.minimum(scored, self.top))
            fields = np.zeros((len(begin), _lib.BLOCKS_RUN), np.int64)
            fields[:, 0], fields[:, 1], fields[:, 2] = self._at[number], self._starts[number] + begin, end - begin
            fields[:, 3:9] = np.stack(ranges, axis=1)
            runs.append((fields, np.full_like(begin, number), begin, end))
        taken = np.concatenate(counts) if counts else np.zeros(0, np.int64)
        fields, sequence, begin, end = (np.concatenate(x) for x in zip(*runs)) if runs else (np.zeros((0, _lib.BLOCKS_RUN), np.int64),
                                                                                            *[taken] * 3)
        self.runs, self.counts, self.width = len(taken), taken.tolist(), int(taken.max(initial=0))
        self._scores = int((fields[:, 6] - fields[:, 5]).max(initial=0)) if self.top else 0
        # (or where a run's scores do not fit in LDS)
        self._apart = self._scores > (_FEW_SCORED if self.runs * cache.heads < _FEW_RUNS else _lib.BLOCKS_TOGETHER)
        if self._scores > _MOST_SCORED:
            raise UnsupportedError(f"a run scores at most {_MOST_SCORED} blocks")
        need(self.runs * cache.heads * max(1, self.width) < 1 << 31, "the step chooses too many blocks")
        # Row blocks: the rows of a run, in tiles, for each key head.
        tile = _ROWS[form]
        row0, row1 = begin * group, end * group
        pieces = -(-(row1 - row0) // tile)
        which = np.repeat(np.arange(self.runs), pieces)
        at = np.arange(len(which)) - np.repeat(np.cumsum(pieces) - pieces, pieces)
        low = row0[which] + at * tile
        high = np.minimum(low + tile, row1[which])
        heads = np.repeat(np.arange(cache.heads, dtype=np.int64), len(which))
        which, low, high = (np.tile(x, cache.heads) for x in (which, low, high))
        self._run_lists = (which * cache.heads + heads) * self.width
        tile = 32 if cache.dtype == torch.float32 or form == "single" else 64
        # Tiles run on over blocks of whole quarters of a tile (the rows of a wave's loads) that are no whole tiles.
        self._tile_unit = tile if form == "rows" and size % (tile // 4) == 0 and size % tile else size
        tiles = taken[which] * -(-size // tile) if self._tile_unit == size else -(-taken[which] * size // tile)
        self._run_taken, merges = taken[which], []
        items = np.empty((0, _lib.ATTEND_ITEM), np.int64)
        if len(which):
            items = self._cut(form, sequence[which], low, high, heads, tiles, lambda which, low, high, part, n: (low, high), merges)
        self._send(form, table, items, merges, fields.ravel())
        self._runs_at = self._merges + self._n_merges * _lib.ATTEND_MERGE

    def _lists_of(self, which):
        return self._run_lists[which], self._run_taken[which]

    def _unit(self):
        return self._tile_unit


class BlockIndex:
    """The mean keys of a cache's blocks.  ``means``: ``[layers, pages, page_tokens / block_tokens, heads, head_dim]``,
    contiguous, of the cache's dtype, on its device; page copies (``extend``, ``compact``, ``make_contiguous``) move it along
    with the pages from now on.  The mean of a block counts once it is full, and has to be up to date then:
    :meth:`update` after every store (and every restore into the pages) that completes or changes a block.
    """

    def __init__(self, cache, means):
        in_memory(means, "means")
        need(means.ndim == 5, "means must be [layers, pages, blocks of a page, heads, head_dim]")
        blocks = means.shape[2]
        need(blocks >= 1 and cache.page_tokens % blocks == 0
             and means.shape == (cache.layers, cache.pages, blocks, cache.heads, cache.head_dim)
             and means.dtype == cache.dtype and means.device == cache.device,
             "means must be [layers, pages, blocks of a page, heads, head_dim] of the cache's dtype and device, blocks dividing a page")
        need(means.is_contiguous(), "means must be contiguous")
        need(not means.requires_grad, "means must not require gradients")
        if cache.page_tokens // blocks > _lib.BLOCKS_TOKENS:
            raise UnsupportedError(f"a block has at most {_lib.BLOCKS_TOKENS} tokens")
        if cache.head_dim > _lib.ATTEND_MAX_DIM:
            raise UnsupportedError(f"an index takes at most {_lib.ATTEND_MAX_DIM} channels to a head")
        self.cache, self.means, self.block_tokens = cache, means, cache.page_tokens // blocks
        self._layer_bytes = means.stride(0) * means.element_size()
        cache._take_along(means, (1, 2, 3), self.block_tokens)

    @classmethod
    def allocate(cls, cache, block_tokens):
        """An index with means of zero."""
        need(cache.page_tokens % count(block_tokens, "block_tokens", minimum=1) == 0, "blocks must divide a page")
        shape = (cache.layers, cache.pages, cache.page_tokens // block_tokens, cache.heads, cache.head_dim)
        return cls(cache, torch.zeros(shape, dtype=cache.dtype, device=cache.device))

    def _layer(self, layer):
        if type(layer) is not int or not 0 <= layer < self.cache.layers:
            raise ConfigurationError("there is no such layer")
        return self.means.data_ptr() + layer * self._layer_bytes

    def _sizes(self):
        cache = self.cache
        return {"heads": cache.heads, "head_dim": cache.head_dim, "pages": cache.pages, "page_tokens": cache.page_tokens,
                "block_tokens": self.block_tokens}

    def update(self, layer, slots):
        """Writes the means of the blocks that hold tokens of ``slots`` (:class:`~reelcache_amd.paged_cache.Slots` or
        ``Places`` of the cache) anew, each over all its rows.  After the layer's ``store``, on the same stream."""
        cache, address = self.cache, self._layer(layer)
        cache._current(slots)
        need_gpu(cache.device, "a block index")
        if slots.tokens == 0:
            return
        with entered(cache.device):
            known = known_calls(slots)
            key = ("update", self.block_tokens)
            image = known.get(key)
            if image is None:
                page, token, head = cache._axes
                stride, strides = cache.keys.stride(), cache._scale_strides()
                image = known[key] = bytes(_fields(**self._sizes(), page_stride=stride[page], token_stride=stride[token],
                                                   head_stride=stride[head], codes=cache.codes, scale_page_stride=strides[0],
                                                   scale_head_stride=strides[1], tokens=slots.tokens))
            fields = _Image.from_buffer_copy(image)
            fields[0], fields[_KEYS_AT] = address, cache.keys.data_ptr() + layer * cache._layer_bytes[0]
            fields[_SCALES_AT], fields[_SLOTS_AT] = cache._scales(layer)[0], slots.index.data_ptr()
            stream = raw_stream(cache.device)
            _lib.check(_lib.function("rch_blocks_update")(fields, _DTYPE_CODES[cache.dtype], stream))
            if stream != slots.stream:  # the allocator learns of a stream that the index was not made on
                slots.index.record_stream(torch.cuda.current_stream(cache.device))
            if not self.means.is_inference():
                torch.autograd.graph.increment_version(self.means)

    def plan(self, sequences, queries, *, heads, top, query_block=1, first=1, recent=1, block=None, window=None, scale=None):
        """The :class:`BlockPlan` of one step: ``queries[i]`` new tokens (the last ones) of ``sequences[i]`` attend to chosen
        blocks of it.  ``top``, ``first``, ``recent``: see the module docstring.  ``query_block``: tokens of a run.  The
        others as in :class:`~reelcache_amd.attention.AttentionPlan`."""
        return BlockPlan(self, sequences, queries, heads=heads, top=top, query_block=query_block, first=first, recent=recent,
                         block=block, window=window, scale=scale)

    def _planned(self, plan):
        need(isinstance(plan, BlockPlan) and plan.index is self, "a BlockPlan of this index is needed")

    def _check(self, q, plan):
        cache = self.cache
        self._planned(plan)
        if plan._stamp != cache._moved:
            raise StateError("pages moved or were freed after this plan was built")
        in_memory(q, "q")
        if q.ndim != 3 or q.shape[0] < plan.queries or q.shape[1] != plan.heads or q.shape[2] != cache.head_dim:
            raise ConfigurationError("q must be [rows, heads, head_dim] with a row for every query of the plan")
        if q.dtype != cache.dtype or q.device != cache.device:
            raise ConfigurationError("q must have the cache's dtype and device")
        if q.requires_grad and torch.is_grad_enabled():
            raise ConfigurationError("a choice of blocks is not differentiable; run it under torch.no_grad()")

    def select(self, layer, q, plan):
        """The blocks that each run of queries and key head attends to: int32 ``[runs, key heads, width]``, numbers of blocks
        of the run's sequence in ascending order, -1 behind the last.  ``q``: as in :meth:`attend`.  Long histories are scored
        in scratch of at most 256 MiB (or what one run's blocks need)."""
        address = self._layer(layer)
        self._check(q, plan)
        cache = self.cache
        with entered(cache.device):
            blocks = torch.empty((plan.runs, cache.heads, plan.width), dtype=torch.int32, device=cache.device)
            if blocks.numel():
                if q.stride(2) != 1 and q.shape[2] > 1:
                    q = q.contiguous()
                known = known_calls(plan)
                key = ("select", q.stride())
                image = known.get(key)
                if image is None:
                    image = known[key] = bytes(_fields(**self._sizes(), q_token_stride=q.stride(0), q_head_stride=q.stride(1),
                                                       group=plan.group, runs=plan._runs_at, n_runs=plan.runs,
                                                       scores=plan._scores, width=plan.width, top=plan.top))
                fields = _Image.from_buffer_copy(image)
                scores, most = None, plan.runs  # runs of a launch
                if plan._apart:
                    most = min(most, max(1, _SCORE_BYTES // (8 * cache.heads * plan._scores)))
                    scores = torch.empty(most * cache.heads * plan._scores, dtype=torch.int64, device=cache.device)
                    fields[_SCORES_AT] = scores.data_ptr()
                fields[0], fields[_Q_AT], fields[_PLAN_AT] = address, q.data_ptr(), plan.buffer.data_ptr()
                stream = raw_stream(cache.device)
                if stream != plan._stream:  # the allocator learns of a stream that the tables were not made on
                    plan.buffer.record_stream(torch.cuda.current_stream(cache.device))
                for first in range(0, plan.runs, most):
                    fields[_RUNS_AT], fields[_RUNS_AT + 1] = plan._runs_at + first * _lib.BLOCKS_RUN, min(most, plan.runs - first)
                    fields[_LISTS_AT] = blocks.data_ptr() + 4 * first * cache.heads * plan.width
                    _lib.check(_lib.function("rch_blocks_select")(fields, _DTYPE_CODES[cache.dtype], stream))
        return blocks

    def attend(self, layer, q, plan, *, blocks=None, out=None, return_lse=False):
        """Attention of ``q`` over the chosen blocks of one layer.

        ``blocks``: what :meth:`select` gave for this plan, or a choice of the caller's own of the same shape and type
        (contiguous; of a run's ``width`` numbers the first ``plan.counts[run]`` are read; the same block twice counts twice; a
        number that is no block of the sequence, or in a dropped page, has no keys); without it, ``q`` and the layer's means choose.  The masks hold within the blocks.  ``q``, ``out``,
        ``return_lse`` and the result as in :func:`reelcache_amd.attention.attend`.
        """
        cache = self.cache
        if blocks is None:
            blocks = self.select(layer, q, plan)
        else:
            self._layer(layer)
            self._planned(plan)
            in_memory(blocks, "blocks")
            need(blocks.shape == (plan.runs, cache.heads, plan.width) and blocks.dtype == torch.int32
                 and blocks.device == cache.device and blocks.is_contiguous(),
                 "blocks must be contiguous int32 [runs, key heads, width] of the plan, on the cache's device")
        k_bytes, v_bytes = cache._layer_bytes
        # (a plan that chooses nothing has no list to point to, and reads none)
        return run(q, cache.keys.data_ptr() + layer * k_bytes, cache.values.data_ptr() + layer * v_bytes, plan, out, return_lse,
                   (*cache._pools(), self.means, blocks), cache._scales(layer), blocks.data_ptr() or plan.buffer.data_ptr())


def _fields(**values):
    return _Image(*(values.get(name, 0) for name in _lib.BLOCKS_FIELDS))


__all__ = ["BlockIndex", "BlockPlan"]
