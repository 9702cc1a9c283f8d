"""Host logic of 8-bit pages and chosen blocks (pools, places, plans) and their refusals, without a GPU."""

import contextlib
import copy
import ctypes
import math
import pickle
import re
import weakref
from pathlib import Path

import numpy as np
import pytest
import torch

from reelcache_amd import _lib, attention, paged_cache, quantized_cache, sparse_attention
from reelcache_amd.errors import ConfigurationError, StateError, UnsupportedError

import history_oracle as history

HEADER = Path(__file__).resolve().parents[1] / "include" / "reelcache_hip.h"


@pytest.fixture
def host(monkeypatch):
    """The host side alone: tables stay on the CPU; the C calls are noted, not made."""
    calls = []
    for module in (paged_cache, attention, quantized_cache, sparse_attention):
        monkeypatch.setattr(module, "need_gpu", lambda device, what: None)
        monkeypatch.setattr(module, "entered", lambda device: contextlib.nullcontext())
        monkeypatch.setattr(module, "raw_stream", lambda device: 0)
    monkeypatch.setattr(paged_cache, "capturing", lambda: False)
    monkeypatch.setattr(paged_cache, "upload", lambda values, device: torch.from_numpy(np.array(values, dtype=np.int32)))
    monkeypatch.setattr(paged_cache, "upload_words", lambda words, shape, device:
                        torch.from_numpy(np.frombuffer(words, dtype=np.int32).reshape(shape).copy()))
    monkeypatch.setattr(paged_cache, "upload_runs", lambda runs, total, device: torch.cat(
        [torch.arange(a, a + n, dtype=torch.int32) for a, n in zip(runs[::2], runs[1::2])] or [torch.empty(0, dtype=torch.int32)]))
    names = {"rch_codes_store": _lib.CODES_FIELDS, "rch_codes_read": _lib.CODES_FIELDS, "rch_blocks_update": _lib.BLOCKS_FIELDS,
             "rch_blocks_select": _lib.BLOCKS_FIELDS, "rch_attend_run": _lib.ATTEND_FIELDS}

    def function(name):
        def call(*arguments):
            fields = names.get(name)
            calls.append((name, dict(zip(fields, arguments[0])) if fields else arguments))
            return _lib.OK
        return call

    monkeypatch.setattr(_lib, "function", lambda name: getattr(_lib.library(), name) if name == "rch_attend_share" else function(name))
    return calls


def quantised(pages=8, size=4, heads=2, dim=16, layers=2, layout="BTHD", dtype=torch.bfloat16, codes=torch.int8):
    return quantized_cache.QuantizedCache.allocate(pages, size, heads, dim, codes=codes, layers=layers, dtype=dtype, device="cpu",
                                                   layout=layout)


def native(pages=8, size=4, heads=2, dim=16, layers=2, layout="BTHD", dtype=torch.bfloat16):
    rows = (size, heads) if layout == "BTHD" else (heads, size)
    return paged_cache.PagedCache(*(torch.zeros((layers, pages, *rows, dim), dtype=dtype) for _ in range(2)), layout=layout)


# ---------------------------------------------------------------------------------------------
# Pools in codes
# ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("layout", ["BTHD", "BHTD"])
@pytest.mark.parametrize("codes", quantized_cache.CODE_DTYPES)
def test_calls_carry_the_pools_addresses_and_strides(host, layout, codes):
    cache = quantised(layout=layout, codes=codes)
    slots = cache.extend([cache.new()], [6])
    k, v = (torch.zeros(6, 2, 16, dtype=torch.bfloat16) for _ in range(2))
    cache.store(1, slots, k, v)
    out = cache.read(1, slots)
    assert all(x.shape == (6, 2, 16) and x.dtype == torch.bfloat16 for x in out)
    (name, store), (other, read) = host[-2:]
    assert (name, other) == ("rch_codes_store", "rch_codes_read")
    for call, dense in ((store, (k, v)), (read, out)):
        assert (call["k_ptr"], call["v_ptr"]) == tuple(x.data_ptr() for x in dense)
        assert call["k_codes_ptr"] == cache.keys[1].data_ptr() and call["v_codes_ptr"] == cache.values[1].data_ptr()
        assert call["k_scales_ptr"] == cache.key_scales[1].data_ptr() and call["v_scales_ptr"] == cache.value_scales[1].data_ptr()
        token, head = (2, 3) if layout == "BTHD" else (3, 2)
        assert (call["k_page_stride"], call["k_row_stride"], call["k_codes_head_stride"]) == tuple(cache.keys.stride(a) for a in (1, token, head))
        assert (call["v_scale_page_stride"], call["v_scale_head_stride"]) == cache.value_scales.stride()[1:3]
        assert call["tokens"] == 6 and call["slots_ptr"] == slots.index.data_ptr() and call["pairs"] == 0
        assert call["format"] == (_lib.CODES_INT8 if codes == torch.int8 else _lib.CODES_E4M3)


def test_refused_pools(host):
    keys = torch.zeros(1, 4, 8, 2, 16, dtype=torch.int8)
    scales = torch.zeros(1, 4, 2, 8)
    make = quantized_cache.QuantizedCache
    make(keys, keys.clone(), scales, scales.clone())
    for arguments, words in (((keys.float(), keys, scales, scales.clone()), {}), ((keys, keys.clone(), scales, scales), {}),
                             ((keys, keys.clone(), scales[..., :4], scales.clone()), {}), ((keys, keys.clone(), scales.double(), scales.clone()), {}),
                             ((keys, keys.clone(), torch.zeros(1, 4, 8, 2).transpose(2, 3), scales.clone()), {}),
                             ((keys, keys.clone(), scales[:, :1].expand(-1, 4, -1, -1), scales.clone()), {}),
                             ((keys, keys.clone(), scales.clone().requires_grad_(True), scales.clone()), {}),
                             ((keys, keys.clone(), scales, scales.clone()), {"dtype": torch.float32}),
                             ((keys, keys.view(torch.uint8), scales, scales.clone()), {})):
        with pytest.raises(ConfigurationError):
            make(*arguments, **words)
    with pytest.raises(UnsupportedError, match="256"):
        quantised(dim=257)
    with pytest.raises(ConfigurationError):
        quantised(codes=torch.uint8)
    with pytest.raises(ConfigurationError):
        paged_cache.PagedCache(keys, keys.clone())


def test_refused_calls(host):
    cache = quantised()
    a = cache.new()
    slots = cache.extend([a], [6])
    k = torch.zeros(6, 2, 16, dtype=torch.bfloat16)
    for bad in (k.half(), k[:5], k.clone().requires_grad_(True)):
        with pytest.raises(ConfigurationError):
            cache.store(0, slots, bad, k)
    for layer in (-1, 2, True, 0.0):
        with pytest.raises(ConfigurationError):
            cache.read(layer, slots)
    other = quantised()
    with pytest.raises(ConfigurationError):
        other.read(0, slots)
    out = torch.zeros(2, 6, 2, 16, dtype=torch.bfloat16)
    for bad in ((out[0],), (out[0], out[0]), (out[0], out[1].half()), (out[0], out[1][:5]), (out[0][:1].expand(6, -1, -1), out[1]),
                (out[0], out[1].clone().requires_grad_(True)),
                (out[0], cache.keys.view(torch.bfloat16).flatten()[:192].view(6, 2, 16))):
        with pytest.raises(ConfigurationError):
            cache.read(0, slots, out=bad)
    with pytest.raises(UnsupportedError, match="store"):
        cache.view(0, "k", a, 0, 4)
    plan = cache.plan([a], [1], heads=4)
    q = torch.zeros(1, 4, 16, dtype=torch.bfloat16)
    cache.attend(0, q, plan)
    with pytest.raises(ConfigurationError, match="QuantizedCache.attend"):
        attention.attend(q, cache.keys[0], cache.values[0], plan)
    with pytest.raises(ConfigurationError):
        cache.attend(0, q, native().plan([], [], heads=4))
    with pytest.raises(ConfigurationError):
        cache.attend(0, q.float(), plan)
    cache.truncate(a, 2)
    with pytest.raises(StateError):
        cache.read(0, slots)
    with pytest.raises(StateError):
        cache.attend(0, q, plan)


def test_places_may_be_shared_and_slots_may_not(host):
    cache = quantised()
    a = cache.new()
    cache.extend([a], [6])
    b = cache.fork(a)
    with pytest.raises(StateError, match="shared"):
        cache.slots([a], [0], [6])
    places = cache.places([b, a], [1, 5], [4, 1])
    assert places.index.tolist() == [1, 2, 3, 4, 5] and isinstance(places, paged_cache.Places)
    k = torch.zeros(5, 2, 16, dtype=torch.bfloat16)
    with pytest.raises(ConfigurationError, match="places"):
        cache.store(0, places, k, k)
    cache.fork(a)  # sharing does not move rows
    cache.read(0, places)
    for starts, counts in (([0], [7]), ([-1], [2]), ([3, 1], [1])):
        with pytest.raises(ConfigurationError):
            cache.places([a], starts, counts)
    cache.free(b)
    with pytest.raises(StateError):
        cache.read(0, places)
    cache.drop(a, 0, 1)
    with pytest.raises(StateError, match="dropped"):
        cache.places([a], [0], [5])
    assert cache.places([a], [4], [2]).index.tolist() == [4, 5]


@pytest.mark.parametrize("who", ["quantised", "native"])
def test_places_are_stale_once_their_page_was_copied(host, who):
    """The sequence of the places goes on in a copy of its begun page: the old one is another sequence's, which may write
    it."""
    cache = quantised(size=8) if who == "quantised" else native(size=8)
    index = cache.index(4)
    a = cache.new()
    cache.extend([a], [13])
    b = cache.fork(a)
    begun, whole = cache.places([a], [8], [5]), cache.places([a, b], [0, 0], [8, 8])
    other = cache.places([b], [8], [5])
    host.clear()
    for places in (begun, whole, other):  # a fork alone moves no rows
        index.update(0, places)
    cache.extend([a], [1])
    assert cache.pages_of(a) == [0, 2] and cache.pages_of(b) == [0, 1]
    assert cache.slots([b], [8], [5]).index.tolist() == begun.index.tolist()  # b may write these rows now
    calls = len(host)
    with pytest.raises(StateError):
        index.update(0, begun)
    if who == "quantised":
        with pytest.raises(StateError):
            cache.read(0, begun)
    assert len(host) == calls  # nothing was launched
    for places in (whole, other):  # where the rows stayed, so does what stands for them
        for _ in range(2):
            index.update(0, places)
            if who == "quantised":
                cache.read(0, places)
    assert cache.places([a], [8], [6]).index.tolist() == [16, 17, 18, 19, 20, 21]


def test_places_of_several_sequences_are_checked_each(host):
    cache = quantised(size=8)
    a, c = cache.new(), cache.new()
    cache.extend([a, c], [13, 5])
    b = cache.fork(a)
    mixed = cache.places([c, a], [0, 3], [5, 10])
    cache.read(0, mixed)
    cache.extend([b], [1])  # b goes on elsewhere; a keeps its rows
    cache.read(0, mixed)
    d = cache.fork(a)
    cache.extend([a, d], [1, 1])
    for _ in range(2):
        with pytest.raises(StateError):
            cache.read(0, mixed)
    cache.read(0, cache.places([c, a], [0, 3], [5, 10]))


def test_places_stay_when_an_extension_fails(host, monkeypatch):
    """A copy that could not be launched changes nothing."""
    cache = quantised(size=8)
    a = cache.new()
    cache.extend([a], [13])
    cache.fork(a)
    places = cache.places([a], [8], [5])
    working = _lib.function

    def failing(name):
        if name == "rch_pages_copy":
            return lambda *arguments: _lib.E_LAUNCH
        return working(name)

    monkeypatch.setattr(_lib, "function", failing)
    with pytest.raises(Exception):
        cache.extend([a], [1])
    monkeypatch.setattr(_lib, "function", working)
    cache.read(0, places)


def test_copied_places_follow_the_copied_cache(host):
    cache = quantised(size=8)
    a = cache.new()
    cache.extend([a], [13])
    cache.fork(a)
    places = cache.places([a], [8], [5])
    other, moved = copy.deepcopy((cache, places))
    other.extend([a], [1])
    with pytest.raises(StateError):
        other.read(0, moved)
    cache.read(0, places)
    alone = pickle.loads(pickle.dumps(places))
    alone.cache.read(0, alone)
    alone.cache.extend([a], [1])
    with pytest.raises(StateError):
        alone.cache.read(0, alone)


def test_plans_of_codes_take_the_matrix_cores_where_rows_are_whole_pieces(host):
    for dim, tiled in ((16, True), (24, False), (128, True), (104, False), (7, False)):
        cache = quantised(dim=dim)
        a = cache.new()
        cache.extend([a], [9])
        general, rows = cache.plan([a], [3], heads=2)._counts_of
        assert (rows > 0 and general == 0) if tiled else (general > 0 and rows == 0)


def test_copied_and_pickled_caches(host):
    cache = quantised()
    index = cache.index(2)
    a = cache.new()
    slots = cache.extend([a], [6])
    cache.read(0, slots)
    other, moved = copy.deepcopy((cache, index))
    assert moved.cache is other and moved.means is other._along[-1].pool() and moved.means is not index.means
    assert pickle.loads(pickle.dumps(slots)).tokens == 6


# ---------------------------------------------------------------------------------------------
# Chosen blocks
# ---------------------------------------------------------------------------------------------


def _brute(length, queries, size, pages, page_tokens, first, recent, query_block, block, window):
    """(always, scored) blocks of each run, key by key."""
    class Zero:
        heads = 1

        def __call__(self, j, head):
            return torch.zeros(1, dtype=torch.float64)

    out = []
    q = torch.zeros(queries, 1, 1, dtype=torch.float64)
    arguments = dict(query_block=query_block, first=first, recent=recent, block=block, window=window)
    everything = history.choice(q, Zero(), pages, length, queries, size, page_tokens, top=1 << 20, **arguments)
    always = history.choice(q, Zero(), pages, length, queries, size, page_tokens, top=0, **arguments)
    for (start, n, taken), (_, _, least) in zip(everything, always):
        out.append((start, n, least[0], sorted(set(taken[0]) - set(least[0]))))
    return out


@pytest.mark.parametrize("seed", range(40))
def test_runs_and_items_of_a_plan(host, seed):
    """The ranges of every run against the rule stated key by key; every tile of every run's list in one part."""
    rng = np.random.default_rng(seed)
    size = int(rng.choice([1, 2, 5, 16, 40, 48, 64]))
    page_tokens = size * int(rng.integers(1, 5))
    dtype = [torch.bfloat16, torch.float32][seed % 2]
    dim, heads, group = int(rng.choice([16, 20, 128, 64, 7])), int(rng.integers(1, 4)), int(rng.integers(1, 4))
    lengths = [int(x) for x in rng.integers(0, 150, 4)] + [0, 1]
    queries = [int(rng.integers(0, 60)) for _ in lengths]
    cache = native(pages=sum(-(-n // page_tokens) for n in lengths) + 1, size=page_tokens, heads=heads, dim=dim, layers=1, dtype=dtype)
    sequences = [cache.new() for _ in lengths]
    cache.extend(sequences, lengths)
    for sequence in sequences:
        pages = len(cache.pages_of(sequence))
        if pages > 2 and rng.random() < 0.5:
            cache.drop(sequence, int(rng.integers(0, pages - 1)), 1)
    top, first, recent = int(rng.integers(0, 6)), int(rng.integers(0, 4)), int(rng.integers(0, 4))
    query_block = int(rng.choice([1, 3, 16, 50, 200]))
    block, window = [(None, None), (1, None), (30, None), (1, 25), (None, 40)][seed % 5]
    index = cache.index(size)
    plan = index.plan(sequences, queries, heads=heads * group, top=top, query_block=query_block, first=first, recent=recent,
                      block=block, window=window)
    words = plan.buffer.numpy()
    runs = words[plan._runs_at:].reshape(-1, _lib.BLOCKS_RUN)
    assert len(runs) == plan.runs
    at, widest, lists = 0, 0, {}
    starts = np.cumsum([0, *queries])
    for number, (length, n) in enumerate(zip(lengths, queries)):
        pages = cache.pages_of(sequences[number])
        for start, count, always, scored in _brute(length, n, size, pages, page_tokens, first, recent, query_block, block, window):
            table, q_row, tokens, low, high, s0, s1, k0, k1, *rest = runs[at].tolist()
            assert (q_row, tokens) == (starts[number] + start, count) and not any(rest)
            assert words[table:table + len(pages)].tolist() == pages
            assert 0 <= low <= high <= -(-length // size) and low <= s0 <= s1 <= high and s0 <= k0 <= k1 <= s1 and s1 - s0 <= max(plan._scores, 0 if top else 1 << 30)
            held = [j for j in range(low, high) if pages[j * size // page_tokens] >= 0]
            chosen = [j for j in held if s0 <= j < s1 and not k0 <= j < k1]
            assert chosen == scored and sorted(set(held) - set(chosen)) == always, (number, start)
            lists[at] = (number, start, count, len(always) + min(top, len(scored)))
            widest = max(widest, lists[at][3])
            at += 1
    assert at == plan.runs and widest == plan.width
    n_items = sum(plan._counts_of)
    items = words[plan._items:plan._items + n_items * _lib.ATTEND_ITEM].reshape(-1, _lib.ATTEND_ITEM)
    tile, seen = 32 if dtype == torch.float32 else 64, {}
    packed = plan._unit() != size
    assert packed == (plan._counts_of[1] > 0 and size % (tile // 4) == 0 and size % tile != 0)
    tiles_of = (lambda taken: -(-taken * size // tile)) if packed else (lambda taken: taken * -(-size // tile))
    for table, length, q_row, n, begin, end, head, low, high, part, at_list, entries in items.tolist():
        if begin >= end:
            continue
        run, h = divmod(at_list // max(1, plan.width), heads) if plan.width else (None, head)
        if plan.width:
            number, start, count, taken = lists[run]
            assert h == head and at_list % plan.width == 0 and (q_row, n, length) == (starts[number], queries[number], lengths[number])
            assert start * group <= begin < end <= (start + count) * group and 0 <= low <= high <= tiles_of(taken) and entries == taken
        for row in range(begin, end):
            seen.setdefault((q_row, head, row), []).append((low, high, run))
    for run, (number, start, count, taken) in lists.items():
        for head in range(heads):
            for row in range(start * group, (start + count) * group):
                parts = sorted(seen.pop((starts[number], head, row)))
                if plan.width:
                    assert parts[0][0] == 0 and parts[-1][1] == tiles_of(taken) and all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
                    assert all(p[2] == run for p in parts)
    assert not seen


def test_refused_indexes_and_plans(host):
    cache = native()
    for means in (torch.zeros(2, 8, 2, 2, 16), torch.zeros(2, 8, 3, 2, 16, dtype=torch.bfloat16), torch.zeros(2, 7, 2, 2, 16, dtype=torch.bfloat16),
                  torch.zeros(2, 8, 2, 16, 2, dtype=torch.bfloat16).transpose(3, 4), torch.zeros(2, 8, 2, 2, 16, dtype=torch.bfloat16, requires_grad=True),
                  torch.zeros(8, 2, 2, 16, dtype=torch.bfloat16), None):
        with pytest.raises(ConfigurationError):
            sparse_attention.BlockIndex(cache, means)
    for size in (3, 8, 0, True, 2.0):
        with pytest.raises(ConfigurationError):
            cache.index(size)
    with pytest.raises(UnsupportedError, match="256"):
        native(dim=264).index(2)
    index, other = cache.index(2), cache.index(4)
    a = cache.new()
    slots = cache.extend([a], [9])
    good = {"heads": 4, "top": 2}
    for bad in ({"top": -1}, {"top": 1.0}, {"query_block": 0}, {"first": -1}, {"recent": True}, {"heads": 3}, {"block": 0}, {"scale": 0.0},
                {"top": 1 << 31}, {"query_block": 1 << 31}):
        with pytest.raises(ConfigurationError):
            index.plan([a], [3], **{**good, **bad})
    plan = index.plan([a], [3], **good)
    q = torch.zeros(3, 4, 16, dtype=torch.bfloat16)
    blocks = index.select(0, q, plan)
    assert blocks.shape == (3, 2, plan.width) and blocks.dtype == torch.int32
    index.attend(0, q, plan, blocks=blocks)
    for call in (lambda: other.select(0, q, plan), lambda: cache.attend(0, q, plan), lambda: index.attend(0, q, cache.plan([a], [1], heads=4)),
                 lambda: attention.attend(q, cache.keys[0], cache.values[0], plan), lambda: index.attend(2, q, plan),
                 lambda: index.select(0, q.float(), plan), lambda: index.select(0, q[:2], plan),
                 lambda: index.select(0, q.clone().requires_grad_(True), plan), lambda: index.attend(0, q, plan, blocks=blocks[:, :1]),
                 lambda: index.attend(0, q, plan, blocks=blocks.long()), lambda: index.attend(0, q, plan, blocks=blocks.transpose(0, 1)),
                 lambda: index.attend(0, q, plan, out=index.means.flatten()[:192].view(3, 4, 16)),
                 lambda: index.update(2, slots), lambda: index.update(0, slots.index), lambda: index.update(0, native().places([], [], []))):
        with pytest.raises(ConfigurationError):
            call()
    cache.extend([a], [1])  # pages only added: the plan holds
    index.attend(0, q, plan)
    cache.truncate(a, 4)
    for call in (lambda: index.select(0, q, plan), lambda: index.attend(0, q, plan), lambda: index.attend(0, q, plan, blocks=blocks),
                 lambda: index.update(0, slots)):
        with pytest.raises(StateError):
            call()


def test_page_copies_take_the_scales_and_means_along(host, monkeypatch):
    """The launches of a copy: the codes, the scales and the means, with rows of tokens, tokens and blocks."""
    cache = quantised(size=8, layers=3)
    index = cache.index(4)
    a = cache.new()
    cache.extend([a], [13])
    b = cache.fork(a)
    host.clear()
    cache.extend([b], [1])
    copies = [(np.array(list(arguments[0])), np.frombuffer(arguments[1], dtype=np.int32).tolist()) for name, arguments in host if name == "rch_pages_copy"]
    fields = [dict(zip(_lib.PAGES_FIELDS, words.tolist())) for words, _ in copies]
    assert [table for _, table in copies] == [[1, 2, 5], [1, 2, 5], [1, 2, 5], [1, 2, 2]]
    assert [f["pools"] for f in fields] == [6, 3, 3, 3]
    assert [(f["page_rows"], f["segments"], f["row_bytes"]) for f in fields] == [(8, 1, 32), (8, 2, 4), (8, 2, 4), (2, 1, 64)]
    assert index.means._version == 1  # a saved one notices


def _copied(host, cache, sequence):
    """(table, rows of a page) of the launches of a fork's copy of its begun page."""
    b = cache.fork(sequence)
    host.clear()
    cache.extend([b], [1])
    found = [(np.frombuffer(arguments[1], dtype=np.int32).tolist()[2], dict(zip(_lib.PAGES_FIELDS, arguments[0]))["page_rows"])
             for name, arguments in host if name == "rch_pages_copy"]
    cache.free(b)
    return found


@pytest.mark.parametrize("sizes", [(4, 1, 2), (1, 4, 8)])
def test_indexes_of_several_block_sizes_move_by_rows_of_their_own(host, sizes):
    cache = native(size=8)
    indexes = [cache.index(n) for n in sizes]
    a = cache.new()
    cache.extend([a], [13])
    assert _copied(host, cache, a) == [(5, 8), *[(-(-5 // n), 8 // n) for n in sizes]]
    assert len(indexes) == len(cache._along)


def test_the_cache_keeps_no_index_that_its_owner_dropped(host):
    cache = quantised(size=8)
    a = cache.new()
    cache.extend([a], [13])
    kept, dropped = cache.index(4), cache.index(2)
    assert len(_copied(host, cache, a)) == 5
    means = weakref.ref(dropped.means)
    del dropped
    assert means() is None
    assert _copied(host, cache, a) == [(5, 8), (5, 8), (5, 8), (2, 2)] and kept.means is cache._along[-1].pool()
    other = copy.deepcopy(cache)  # without its index
    assert _copied(host, other, a) == [(5, 8)] * 3
    assert other._moving[0].data_ptr() == other.key_scales.data_ptr() != cache.key_scales.data_ptr()


def test_stores_refuse_what_overlaps_the_scales(host):
    cache = quantised(pages=64, size=4, heads=2, dim=16)
    slots = cache.extend([cache.new()], [2])
    dense = torch.zeros(2, 2, 16, dtype=torch.bfloat16)
    for scales in (cache.key_scales, cache.value_scales):
        over = scales.view(torch.bfloat16).flatten()[:64].view(2, 2, 16)
        for k, v in ((over, dense), (dense, over)):
            with pytest.raises(ConfigurationError, match="scales"):
                cache.store(1, slots, k, v)
    cache.store(1, slots, dense, dense)


def test_plans_count_the_blocks_that_each_run_takes(host):
    cache = native(pages=16, size=8)
    a, b = cache.new(), cache.new()
    cache.extend([a, b], [80, 20])
    plan = cache.index(8).plan([a, b], [1, 1], heads=2, top=3)
    assert (plan.runs, plan.counts, plan.width) == (2, [5, 3], 5)


def test_blocks_of_too_many_tokens_are_refused(host):
    pools = [torch.empty((1, 1, 1 << 25, 1, 1), dtype=torch.bfloat16) for _ in range(2)]
    cache = paged_cache.PagedCache(*pools)
    with pytest.raises(UnsupportedError, match="tokens"):
        cache.index(1 << 25)
    cache.index(1 << 24)


def test_header_matches_the_binding():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    for struct, fields in (("rch_codes", _lib.CODES_FIELDS), ("rch_blocks", _lib.BLOCKS_FIELDS)):
        body = re.search(r"typedef struct " + struct + r" \{(.*?)\}", text, flags=re.S).group(1)
        assert tuple(name.strip().split()[-1] for line in body.split(";") if line.strip() for name in line.split(",")) == fields
    defines = {name: int(value) for name, value in re.findall(r"#define (RCH_[A-Z0-9_]+) (\d+)\b", HEADER.read_text())}
    expected = {"RCH_CODES_NONE": _lib.CODES_NONE, "RCH_CODES_INT8": _lib.CODES_INT8, "RCH_CODES_E4M3": _lib.CODES_E4M3,
                "RCH_CODES_MAX_DIM": _lib.CODES_MAX_DIM, "RCH_BLOCKS_RUN": _lib.BLOCKS_RUN, "RCH_BLOCKS_TOGETHER": _lib.BLOCKS_TOGETHER}
    assert "#define RCH_BLOCKS_TOKENS (1 << 24)" in HEADER.read_text() and _lib.BLOCKS_TOKENS == 1 << 24
    assert {name: defines.get(name) for name in expected} == expected
    lib = _lib.library()
    assert lib.rch_codes_size() == 8 * len(_lib.CODES_FIELDS) and lib.rch_blocks_size() == 8 * len(_lib.BLOCKS_FIELDS)


def test_abi_refusals():
    """Bad arguments of the C entry points end in a status and a message, not in a launch."""

    def words(fields, **values):
        return (ctypes.c_int64 * len(fields))(*(values.get(f, 0) for f in fields))

    addresses = {name: 64 for name in ("k_ptr", "v_ptr", "k_codes_ptr", "v_codes_ptr", "k_scales_ptr", "v_scales_ptr", "slots_ptr")}
    good = dict(addresses, tokens=1, heads=1, head_dim=8, pages=1, page_tokens=1, format=1)
    for name in ("rch_codes_store", "rch_codes_read"):
        for bad, dtype, error in (({"format": 0}, 2, ConfigurationError), ({"format": 3}, 2, ConfigurationError), ({}, 0, UnsupportedError),
                                  ({"head_dim": 257}, 2, UnsupportedError), ({"head_dim": 0}, 2, ConfigurationError),
                                  ({"pages": 1 << 20, "page_tokens": 1 << 12}, 2, ConfigurationError), ({"pairs": 5}, 2, ConfigurationError),
                                  ({"pairs": 2}, 2, ConfigurationError), ({"slots_ptr": 0}, 2, ConfigurationError),
                                  ({"k_scales_ptr": 0}, 2, ConfigurationError), ({"tokens": -1}, 2, ConfigurationError)):
            with pytest.raises(error):
                _lib.call(name, words(_lib.CODES_FIELDS, **{**good, **bad}), dtype, None)
        _lib.call(name, words(_lib.CODES_FIELDS, **{**good, "tokens": 0}), 2, None)
    good = dict(means_ptr=64, keys_ptr=64, slots_ptr=64, q_ptr=64, plan_ptr=64, lists_ptr=64, scores_ptr=64, heads=1, head_dim=8, pages=1,
                page_tokens=4, block_tokens=2, tokens=1, group=1, n_runs=1, width=1, scores=1, top=1)
    for name, cases in (("rch_blocks_update", ({"block_tokens": 3}, {"codes": 3}, {"codes": 1}, {"tokens": -1}, {"keys_ptr": 0}, {"head_dim": 257})),
                        ("rch_blocks_select", ({"group": 0}, {"n_runs": -1}, {"scores_ptr": 0, "scores": 4097}, {"scores": 0}, {"scores_ptr": 4}, {"lists_ptr": 0}, {"top": -1},
                                               {"width": -1}, {"scores": 1 << 30}, {"block_tokens": 0}))):
        for bad in cases:
            with pytest.raises(ConfigurationError):
                _lib.call(name, words(_lib.BLOCKS_FIELDS, **{**good, **bad}), 2, None)
    with pytest.raises(UnsupportedError):
        _lib.call("rch_blocks_update", words(_lib.BLOCKS_FIELDS, **{**good, "codes": 1, "scales_ptr": 64}), 0, None)
    _lib.call("rch_blocks_update", words(_lib.BLOCKS_FIELDS, **{**good, "tokens": 0}), 2, None)
    _lib.call("rch_blocks_select", words(_lib.BLOCKS_FIELDS, **{**good, "n_runs": 0}), 2, None)
    step = dict(group=1, heads=1, head_dim=16, page_tokens=4, pages=1, n_general=1, scale_bits=0x3f800000, q_ptr=64, k_ptr=64, v_ptr=64,
                out_ptr=64, plan_ptr=64, k_scale_ptr=64, v_scale_ptr=64)
    for bad, dtype, error in (({"codes": 3}, 2, ConfigurationError), ({"codes": 1}, 0, UnsupportedError), ({"codes": 1, "k_scale_ptr": 0}, 2, ConfigurationError),
                              ({"single": 1}, 2, ConfigurationError), ({"single": 1, "codes": 1}, 2, ConfigurationError),
                              ({"single": 1, "codes": 1, "n_general": 0, "n_rows": 1, "group": 33}, 2, ConfigurationError),
                              ({"lists_ptr": 64}, 2, ConfigurationError), ({"lists_ptr": 64, "block_tokens": 3}, 2, ConfigurationError),
                              ({"lists_ptr": 64, "block_tokens": 2, "n_general": 0, "n_rows": 1, "tile_unit": 64}, 2, ConfigurationError),
                              ({"codes": 1, "n_general": 0, "n_rows": 1, "head_dim": 24, "tile_unit": 64}, 2, UnsupportedError)):
        with pytest.raises(error):
            _lib.call("rch_attend_run", words(_lib.ATTEND_FIELDS, **{**step, **bad}), dtype, None)


# ---------------------------------------------------------------------------------------------
# The oracle
# ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("codes", quantized_cache.CODE_DTYPES)
def test_the_plain_codes_are_the_nearest_ones(codes):
    """By search over all codes, at scales of several sizes."""
    every = torch.arange(256, dtype=torch.uint8).view(codes).double()
    every = every[every.isfinite() & (every.abs() <= (127 if codes == torch.int8 else 448))]
    x = torch.randn(60, 16, generator=torch.Generator().manual_seed(0)) * torch.exp2(torch.arange(60.0) - 40)[:, None]
    code, scale = history.encode(x, codes, torch.bfloat16)
    y = x.double() / scale.double()[:, None]
    best = (every - y[..., None]).abs().amin(dim=-1)
    assert ((code.double() - y).abs() <= best * (1 + 1e-6) + 1e-6).all()
    most = x.abs().amax(dim=1).double() / scale.double()
    assert (most <= (127 if codes == torch.int8 else 448) * (1 + 1e-6)).all() and (most > (126.9 if codes == torch.int8 else 224)).all()
    lost = history.encode(torch.tensor([[1.0, math.nan], [math.inf, 0.0]]), codes)
    assert lost[1].isnan().all() and not lost[0].float().any()


@pytest.mark.parametrize("source", ["attend_lists.hip", "attend_int8.hip"])
def test_resources_are_written_early_enough(source, tmp_path):
    """As for the other tiles that are fetched straight into LDS; and the registers of a base address."""
    import subprocess

    import test_kernel_code_host as machine
    from reelcache_amd.csrc import build as hip_build

    target = tmp_path / "kernels.s"
    subprocess.run([hip_build._hipcc(), *hip_build.FLAGS, "-w", "--cuda-device-only", "-S", str(hip_build.HERE / source), "-o",
                    str(target)], check=True, capture_output=True)
    text = target.read_text()
    assert text.count("offen lds") > 50 and machine.late_resources(text) == []
    if source != "attend_lists.hip":
        based = re.sub(r"global_load_lds_dwordx4 (v\d+), (s\[\d+:\d+\])", r"buffer_load_dwordx4 \1, \2, 0 offen lds", text)
        assert based.count("offen lds") > text.count("offen lds") + 50 and machine.late_resources(based) == []


@pytest.mark.parametrize("least", [0, 1 << 16])
def test_the_scratch_of_a_choice_is_bounded(host, monkeypatch, least):
    """Steps whose numbers need more than the bound choose run after run: every run once, each with its own list."""
    cache = native(pages=6000, size=1, heads=2, dim=8, layers=2)
    a = cache.new()
    cache.extend([a], [5500])
    index = cache.index(1)
    plan = index.plan([a], [4400], heads=4, top=3)  # every run scores all blocks but the last one's
    assert plan._apart and plan.runs == 4400 and plan._scores > _lib.BLOCKS_TOGETHER
    if least:  # a bound below a run's own need
        monkeypatch.setattr(sparse_attention, "_SCORE_BYTES", least, raising=False)
    bound = max(least or 1 << 28, cache.heads * plan._scores * 8)
    assert plan.runs * cache.heads * plan._scores * 8 > bound
    q = torch.zeros(4400, 4, 8, dtype=torch.bfloat16)
    host.clear()
    blocks = index.select(1, q, plan)
    at = 0
    for name, call in host:
        assert name == "rch_blocks_select" and call["n_runs"] >= 1
        assert call["n_runs"] * cache.heads * call["scores"] * 8 <= bound and call["scores"] == plan._scores and call["scores_ptr"]
        assert call["runs"] == plan._runs_at + at * _lib.BLOCKS_RUN and call["lists_ptr"] == blocks[at].data_ptr()
        assert call["q_ptr"] == q.data_ptr() and call["means_ptr"] == index.means[1].data_ptr()
        at += call["n_runs"]
    assert at == plan.runs


def test_a_choice_within_the_bound_is_one_call(host):
    cache = native(pages=600, size=1, heads=2, dim=8)
    a = cache.new()
    cache.extend([a], [500])
    index = cache.index(1)
    for queries, apart in ((20, True), (100, False)):
        plan = index.plan([a], [queries], heads=2, top=3)
        assert plan._apart == apart
        host.clear()
        blocks = index.select(0, torch.zeros(queries, 2, 8, dtype=torch.bfloat16), plan)
        (_, call), = host
        assert (call["runs"], call["n_runs"], call["lists_ptr"]) == (plan._runs_at, queries, blocks.data_ptr()) and bool(call["scores_ptr"]) == apart


@pytest.mark.parametrize("source", ["rotary.hip", "codes.hip", "blocks.hip"])
def test_kernels_keep_their_values_in_registers(source, tmp_path):
    """No scratch memory: places of rotated tokens written to an array cost every rotation and store 1 to 2 %."""
    import subprocess

    from reelcache_amd.csrc import build as hip_build

    target = tmp_path / "kernels.s"
    subprocess.run([hip_build._hipcc(), *hip_build.FLAGS, "-w", "--cuda-device-only", "-S", str(hip_build.HERE / source), "-o",
                    str(target)], check=True, capture_output=True)
    sizes = re.findall(r"\.private_segment_fixed_size: (\d+)", target.read_text())
    assert len(sizes) > 10 and set(sizes) == {"0"}


@pytest.mark.parametrize("dim", [64, 128, 144, 192, 256])
def test_single_tokens_over_codes_fill_the_card_by_parts_at_every_head_size(host, dim):
    """A form of single waves is cut into as many parts as it says, whatever the number of waves that its heads leave room for:
    one long sequence of 8 key heads takes half of the places."""
    cache = quantised(pages=1024, size=64, heads=8, dim=dim, layers=1)
    cache.load_tables([(list(range(1024)), 65536)])
    plan = cache.plan([0], [1], heads=32)
    assert plan._single
    items = plan.buffer.numpy()[plan._items:plan._items + plan._counts_of[1] * _lib.ATTEND_ITEM].reshape(-1, _lib.ATTEND_ITEM)
    parts = int((items[:, 5] > items[:, 4]).sum())
    shortest = -(-1024 // (plan._resident("single") // 16))  # tiles of a part, of a head's 1024
    assert parts >= 8 * (1024 // shortest), parts
    short = quantised(pages=64, size=64, heads=8, dim=dim, layers=1)
    short.load_tables([(list(range(8)), 512)])
    assert short.plan([0], [1], heads=32)._n_merges  # parts of single tiles
    assert "#define RCH_SHARE_WAVES (1LL << 32)" in HEADER.read_text() and _lib.SHARE_WAVES == 1 << 32
