"""Host logic of the cache operators (page tables, slots, plans) and their refusals, without a GPU."""

import contextlib
import copy
import gc
import heapq
import pickle
import re
import types
import weakref
from pathlib import Path

import numpy as np
import pytest
import torch

from reelcache_amd import _lib, attention, paged_cache, rotary
from reelcache_amd import restore_kernels as rk
from reelcache_amd.errors import CapacityError, ConfigurationError, StateError, UnsupportedError

import operator_oracle as oracle

HEADER = Path(__file__).resolve().parents[1] / "include" / "reelcache_hip.h"


@pytest.fixture
def host(monkeypatch):
    """The cache's host side alone: tables stay on the CPU, page copies are carried out by torch."""
    copies = []

    def copy(self, moves):
        moves = list(zip(*[iter(moves)] * 3))
        copies.extend(moves)
        for pool in (self.keys, self.values):
            for source, target, rows in moves:
                if self.layout == "BTHD":
                    pool[:, target, :rows] = pool[:, source, :rows]
                else:
                    pool[:, target, :, :rows] = pool[:, source, :, :rows]

    monkeypatch.setattr(paged_cache.PagedCache, "_copy", copy)
    for module in (paged_cache, attention):
        monkeypatch.setattr(module, "need_gpu", lambda device, what: None)
        monkeypatch.setattr(module, "entered", lambda device: contextlib.nullcontext())
        monkeypatch.setattr(module, "raw_stream", lambda device: 0)
    monkeypatch.setattr(paged_cache, "capturing", lambda: False)
    monkeypatch.setattr(paged_cache, "upload", lambda values, device: torch.from_numpy(np.array(values, dtype=np.int32)))
    monkeypatch.setattr(paged_cache, "upload_words", lambda words, shape, device:
                        torch.from_numpy(np.frombuffer(words, dtype=np.int32).reshape(shape).copy()))
    monkeypatch.setattr(paged_cache, "upload_runs", lambda runs, total, device: torch.cat(
        [torch.arange(a, a + n, dtype=torch.int32) for a, n in zip(runs[::2], runs[1::2])] or [torch.empty(0, dtype=torch.int32)]))
    return copies


def make(pages=8, size=4, heads=2, dim=8, layers=2, layout="BTHD", dtype=torch.float32):
    rows = (size, heads) if layout == "BTHD" else (heads, size)
    pools = [torch.randn((layers, pages, *rows, dim)).to(dtype) for _ in range(2)]
    return paged_cache.PagedCache(*pools, layout=layout)


def contents(cache, sequence):
    """The K rows of a sequence in layer 0, gathered through its pages."""
    pool = cache.keys[0] if cache.layout == "BTHD" else cache.keys[0].transpose(1, 2)
    return torch.cat([pool[page] for page in cache.pages_of(sequence)])[:cache.tokens(sequence)].clone()


def test_sequences_grow_share_and_copy(host):
    cache = make()
    a = cache.new()
    slots = cache.extend([a], [6])
    assert slots.index.tolist() == [0, 1, 2, 3, 4, 5] and slots.tokens == 6 and cache.pages_of(a) == [0, 1]
    b, c = cache.fork(a), cache.fork(a)
    before = contents(cache, a)
    slots = cache.extend([b, c, a], [3, 1, 1])
    # b and c copy the begun page; a is its last owner and goes on in it.
    assert host == [(1, 2, 2), (1, 4, 2)]
    assert [cache.pages_of(s) for s in (a, b, c)] == [[0, 1], [0, 2, 3], [0, 4]]
    assert slots.index.tolist() == [10, 11, 12, 18, 6]
    for s in (a, b, c):
        assert torch.equal(contents(cache, s)[:6], before)
    assert cache.free_pages == 3 and [cache.tokens(s) for s in (a, b, c)] == [7, 9, 7]
    cache.free(b)
    assert cache.free_pages == 5 and cache.pages_of(a) == [0, 1]
    assert cache.extend([a], [0]).tokens == 0


def test_a_full_last_page_is_not_copied(host):
    cache = make()
    a = cache.new()
    cache.extend([a], [8])
    b = cache.fork(a)
    assert cache.extend([b], [1]).index.tolist() == [8] and host == []
    cache.truncate(b, 5)  # now inside a page that a has too
    assert cache.extend([b], [1]).index.tolist() == [9] and host == [(1, 2, 1)]


def test_capacity_is_checked_before_anything_changes(host):
    cache = make(pages=3)
    a = cache.new()
    cache.extend([a], [6])
    b, c = cache.fork(a), cache.fork(a)
    with pytest.raises(CapacityError, match="2 pages are needed and 1 are free"):
        cache.extend([b, c], [1, 1])
    assert host == [] and [cache.tokens(s) for s in (a, b, c)] == [6, 6, 6] and cache.free_pages == 1


@pytest.mark.parametrize("layout", ["BTHD", "BHTD"])
def test_compact_moves_the_highest_pages_down(host, layout):
    cache = make(pages=10, layout=layout)
    cache.load_tables([([9, 3], 7), ([0, 7, 9], 12), ([5], 2)])
    kept = [contents(cache, s) for s in range(3)]
    assert cache.compact() == [(5, 1), (7, 2), (9, 4)]
    assert [cache.pages_of(s) for s in range(3)] == [[4, 3], [0, 2, 4], [1]]
    assert all(torch.equal(contents(cache, s), kept[s]) for s in range(3))
    assert cache.compact() == [] and cache.free_pages == 5
    cache.extend([cache.new()], [4])
    assert cache.pages_of(3) == [5]


def test_make_contiguous_and_view(host):
    cache = make(pages=10)
    cache.load_tables([([7, 0, 4], 11), ([8], 4)])
    kept = contents(cache, 0)
    with pytest.raises(StateError, match="make_contiguous"):
        cache.view(1, "k", 0, 0, 11)
    one = cache.view(1, "k", 0, 4, 4)
    assert one.layout == "BTHD" and one.batch_index == 0 and one.token_offset == 0
    assert torch.equal(one.slot(4), cache.keys[1, 0])
    assert cache.make_contiguous(0) == [(7, 1), (0, 2), (4, 3)]
    assert torch.equal(contents(cache, 0), kept) and cache.make_contiguous(0) == []
    view = cache.view(1, "v", 0, 2, 9)
    assert view.layout == "THD" and torch.equal(view.slot(9), cache.values[1, 1:4].flatten(0, 1)[2:11])
    view.slot(9).fill_(3)
    assert (cache.values[1, 1:4].flatten(0, 1)[2:11] == 3).all()
    with pytest.raises(CapacityError):
        small = make(pages=4)
        small.load_tables([([3, 0], 8)])
        small.fork(0)
        small.extend([small.new()], [4])
        small.make_contiguous(0)
    heads_first = make(layout="BHTD")
    heads_first.load_tables([([1, 2], 8)])
    with pytest.raises(StateError):
        heads_first.view(0, "k", 0, 0, 8)
    assert heads_first.view(0, "k", 0, 5, 3).layout == "BHTD"


def test_holes(host):
    cache = make()
    a = cache.new()
    cache.extend([a], [18])
    cache.drop(a, 1, 2)
    assert cache.pages_of(a) == [0, -1, -1, 3, 4] and cache.free_pages == 5
    with pytest.raises(ConfigurationError):
        cache.drop(a, 4, 1)
    with pytest.raises(StateError, match="dropped"):
        cache.slots([a], [3], [2])
    with pytest.raises(StateError, match="dropped"):
        cache.truncate(a, 6)
    with pytest.raises(StateError):
        cache.make_contiguous(a)
    b = cache.fork(a)
    assert cache.extend([b], [3]).index.tolist() == [1 * 4 + 2, 1 * 4 + 3, 2 * 4] and host == [(4, 1, 2)]
    assert cache.page_table([a, b]).tolist() == [[0, -1, -1, 3, 4, -1], [0, -1, -1, 3, 1, 2]]


def test_sequence_refusals(host):
    cache = make()
    a = cache.new()
    cache.extend([a], [5])
    for call in (lambda: cache.tokens(7), lambda: cache.fork("a"), lambda: cache.free(-1), lambda: cache.page_table([3])):
        with pytest.raises(StateError):
            call()
    for call in (lambda: cache.extend([a, a], [1, 1]), lambda: cache.extend([a], [1, 2]), lambda: cache.extend([a], [-1]),
                 lambda: cache.extend([a], [1.0]), lambda: cache.truncate(a, 6), lambda: cache.slots([a], [2], [4]),
                 lambda: cache.drop(a, 1, 1), lambda: cache.view(2, "k", a, 0, 1), lambda: cache.view(0, "q", a, 0, 1),
                 lambda: cache.load_tables([([0], 5)]), lambda: cache.load_tables([([0, 0], 5)]),
                 lambda: cache.load_tables([([8], 2)]), lambda: cache.load_tables([([-2], 2)]),
                 lambda: cache.load_tables([([0, -1], 5)])):
        with pytest.raises(ConfigurationError):
            call()
    assert cache.pages_of(a) == [0, 1]
    cache.fork(a)
    with pytest.raises(StateError, match="shared"):
        cache.slots([a], [0], [1])
    with pytest.raises(StateError, match="shared"):
        cache.view(0, "k", a, 0, 1)


def test_stale_slots_are_refused(host):
    cache = make()
    a, b = cache.new(), cache.new()
    slots = cache.extend([a], [5])
    x = torch.zeros(5, 2, 8)
    for change in (lambda: cache.fork(a), lambda: cache.free(b), cache.compact, lambda: cache.load_tables([([0, 1], 5)])):
        slots = cache.slots([a], [4], [1]) if cache.pages_of(a) and cache._uses[cache.pages_of(a)[-1]] == 1 else slots
        if change is cache.compact:  # nothing moves: nothing is stale
            change()
            continue
        change()
        with pytest.raises(StateError, match="after these slots"):
            cache.store(0, slots, x, x)
    other = make()
    with pytest.raises(ConfigurationError, match="come from this cache"):
        other.store(0, slots, x, x)
    slots = cache.slots([0], [0], [5])
    for call in (lambda: cache.store(2, slots, x, x), lambda: cache.store(0, slots, x[:4], x), lambda: cache.store(0, slots, x, x.half()),
                 lambda: cache.store(0, slots, x.clone().requires_grad_(True), x)):
        with pytest.raises(ConfigurationError):
            call()


def test_pool_refusals():
    good = torch.zeros(1, 2, 4, 2, 8)
    for keys, values in ((good[0], good[0]), (good, good.half()), (good, torch.zeros(1, 2, 4, 2, 16)),
                         (good.int(), good.int()), (good, good[..., :0]), (good.clone().requires_grad_(True), good), (good.expand(3, -1, -1, -1, -1), good.expand(3, -1, -1, -1, -1)),
                         (torch.zeros(300).as_strided((1, 2, 4, 2, 8), (256, 128, 32, 16, 2)),) * 2,
                         (torch.zeros(300).as_strided((1, 2, 4, 2, 8), (128, 32, 16, 8, 1)),) * 2):
        with pytest.raises(ConfigurationError):
            paged_cache.PagedCache(keys, values)
    with pytest.raises(ConfigurationError):
        paged_cache.PagedCache(good, good, layout="THD")
    with pytest.raises(ConfigurationError):
        paged_cache.PagedCache.allocate(0, 4, 2, 8, device="cpu")
    paged_cache.PagedCache(good[:, :, :, :, :4], good[:, :, :, :, :4])  # gaps are fine


def test_cpu_tensors_are_refused():
    cache = make()
    a = cache.new()
    table = rk.RopeTable(*oracle.tables(8, 4))
    x = torch.zeros(1, 6, 2, 8)
    for call in (lambda: cache.extend([a], [1]), lambda: cache.page_table([a]), lambda: cache.plan([a], [0], heads=2),
                 lambda: rotary.rotate(x, rk.RopePositions(table, 0), grid=(1, 2, 3))):
        with pytest.raises(UnsupportedError, match="GPU"):
            call()


def test_rotary_refusals(monkeypatch):
    monkeypatch.setattr(rotary, "need_gpu", lambda device, what: None)
    monkeypatch.setattr(rotary, "entered", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(rotary, "_table_pairs", lambda table, device, stream: 64)
    monkeypatch.setattr(rotary, "raw_stream", lambda device: 0)
    launches = []
    monkeypatch.setattr(rotary.Launch, "__call__", lambda self, addresses, *rest: launches.append((self, addresses)))
    cos, sin, sections = oracle.tables(8, 4)
    table, dense = rk.RopeTable(cos, sin, sections), rk.RopeTable(cos, sin)
    x, grid, at = torch.zeros(1, 6, 2, 8), (1, 2, 3), rk.RopePositions(table, 0)
    rows = torch.zeros(6, 3, dtype=torch.int32)
    rotary.rotate(x, at, grid=grid)
    rotary.rotate(x, rotary.TokenRows(table, rows))
    assert len(launches) == 2 and all(len(launch.image) == 8 * len(_lib.ROTARY_FIELDS) for launch, _ in launches)
    for call in (
            lambda: rotary.rotate(x, table, grid=grid), lambda: rotary.rotate(x, at), lambda: rotary.rotate(x, at, grid=(1, 2, 2)),
            lambda: rotary.rotate(x, at, grid=(0, 2, 3)), lambda: rotary.rotate(x, rk.RopePositions(table, (8, 0, 0)), grid=grid),
            lambda: rotary.rotate(x, rk.RopePositions(dense, 3)), lambda: rotary.rotate(x, rk.RopePositions(dense, 0), grid=grid),
            lambda: rotary.rotate(x, at, grid=grid, layout="HTD"), lambda: rotary.rotate(x[0], at, grid=grid),
            lambda: rotary.rotate(x, at, grid=grid, pairing="whole"), lambda: rotary.rotate(x.double(), at, grid=grid),
            lambda: rotary.rotate((x, x.half()), at, grid=grid), lambda: rotary.rotate((), at, grid=grid),
            lambda: rotary.rotate((x,) * 5, at, grid=grid), lambda: rotary.rotate(x[..., :6], at, grid=grid),
            lambda: rotary.rotate(x, rotary.TokenRows(table, rows[:5])), lambda: rotary.rotate(x, rotary.TokenRows(table, rows), grid=grid),
            lambda: rotary.TokenRows(table, rows.long()), lambda: rotary.TokenRows(table, rows[:, :2]),
            lambda: rotary.TokenRows(dense, torch.zeros(1, 2, 3, dtype=torch.int32)), lambda: rotary.TokenRows(None, rows),
            lambda: rotary.rotate(x, rotary.TokenRows(table, rows[None].expand(2, 6, 3))),
            lambda: rotary.rotate(x, at, grid=grid, out=x[..., :4]), lambda: rotary.rotate(x, at, grid=grid, out=(x, x)),
            lambda: rotary.rotate(x, at, grid=grid, out=torch.zeros(1, 6, 1, 8).expand(1, 6, 2, 8)),
            lambda: rotary.rotate(x, at, grid=grid, out=x.flip(1).as_strided(x.shape, x.stride()).requires_grad_(True))):
        with pytest.raises(ConfigurationError):
            call()
    storage = torch.zeros(200)
    a, b = (storage[i:i + 96].view(1, 6, 2, 8) for i in (0, 16))
    for call in (lambda: rotary.rotate(a, at, grid=grid, out=b), lambda: rotary.rotate((a, x), at, grid=grid, out=(x, a)),
                 lambda: rotary.rotate((x, x.clone()), at, grid=grid, out=(a, b))):
        with pytest.raises(ConfigurationError, match="overlap"):
            call()
    assert len(launches) == 2


def test_pages_too_large_to_copy_are_refused_before_anything_changes(host, monkeypatch):
    cache = make()
    a = cache.new()
    cache.extend([a], [5])
    b = cache.fork(a)
    monkeypatch.setattr(cache, "head_dim", 1 << 30)
    with pytest.raises(UnsupportedError, match="2 GiB"):
        cache.extend([b], [1])
    cache.truncate(b, 4)
    with pytest.raises(UnsupportedError, match="2 GiB"):
        cache.load_tables([([7], 2)])
        cache.compact()
    assert cache.pages_of(0) == [7] and host == []


def test_plan_refusals(host):
    cache = make()
    a = cache.new()
    cache.extend([a], [9])
    for call in (lambda: cache.plan([a], [1], heads=3), lambda: cache.plan([a], [1, 2], heads=2), lambda: cache.plan([a, a], [1, 1], heads=2),
                 lambda: cache.plan([a], [-1], heads=2), lambda: cache.plan([a], [1], heads=2, block=0),
                 lambda: cache.plan([a], [1], heads=2, window=0), lambda: cache.plan([a], [1], heads=2, scale=0.0),
                 lambda: cache.plan([a], [1], heads=2, scale=float("nan")), lambda: cache.plan([a], [1], heads=2, block=1 << 31)):
        with pytest.raises(ConfigurationError):
            call()
    with pytest.raises(UnsupportedError, match="256"):
        wide = make(dim=264)
        wide.plan([wide.new()], [0], heads=2)
    plan = cache.plan([a], [1], heads=2)
    cache.extend([a], [3])  # pages only added: the plan still holds
    plan._check(cache.keys[0], cache.values[0])
    with pytest.raises(ConfigurationError):
        plan._check(cache.keys[0][:4], cache.values[0])
    with pytest.raises(ConfigurationError, match="differentiable"):
        cache.attend(0, torch.zeros(1, 2, 8, requires_grad=True), plan)
    cache.truncate(a, 2)
    with pytest.raises(StateError, match="after this plan"):
        cache.attend(0, torch.zeros(1, 2, 8), plan)


def _items(plan):
    words = plan.buffer.numpy()
    n = sum(plan._counts_of)
    items = words[plan._items:plan._items + n * _lib.ATTEND_ITEM].reshape(n, _lib.ATTEND_ITEM)
    merges = words[plan._merges:plan._merges + plan._n_merges * _lib.ATTEND_MERGE].reshape(-1, _lib.ATTEND_MERGE)
    assert len(words) == plan._merges + merges.size and not words[:_lib.ATTEND_ZEROS].any()
    return items, merges


@pytest.mark.parametrize("size,dim,layout", [(16, 64, "BTHD"), (64, 128, "BTHD"), (100, 80, "BHTD"), (1560, 128, "BTHD"), (5, 20, "BTHD")])
@pytest.mark.parametrize("block,window", [(None, None), (1, None), (37, None), (None, 50), (1, 200)])
def test_plan_covers_every_visible_key_once(host, size, dim, layout, block, window):
    """Items of a plan: every row of every sequence and head once per visible key, keys of a part within
    its row block's range, parts of a block in disjoint partial rows, every split block merged once."""
    lengths, queries, group, kv_heads = [1, 333, 700, 40, 0, 2000], [1, 333, 1, 9, 2, 300], 2, 2
    pages = sum(-(-n // size) for n in lengths)
    cache = make(pages=pages, size=size, heads=kv_heads, dim=dim, layers=1, layout=layout, dtype=torch.bfloat16)
    sequences = [cache.new() for _ in lengths]
    cache.extend(sequences, lengths)
    plan = cache.plan(sequences, queries, heads=kv_heads * group, block=block, window=window)
    items, merges = _items(plan)
    words = plan.buffer.numpy()
    starts = np.cumsum([0, *queries])
    seen = {}
    partial_rows = []
    for table, length, q_row, n, begin, end, head, low, high, part, *_ in items.tolist():
        if begin >= end:  # filling
            continue
        number = [i for i in range(len(lengths)) if starts[i] == q_row and queries[i] == n and lengths[i] == length]
        assert len(number) == 1 and 0 <= begin < end <= n * group and 0 <= low <= high <= length
        assert words[table:table + -(-length // size)].tolist() == cache.pages_of(sequences[number[0]])
        for row in range(begin, end):
            seen.setdefault((number[0], head, row), []).append((low, high))
        if part >= 0:
            partial_rows += list(range(part, part + end - begin))
            merge = [m for m in merges.tolist() if m[0] == q_row and m[1] == begin and m[3] == head and m[2] == end - begin]
            assert len(merge) == 1 and (part - merge[0][4]) % (end - begin) == 0
            assert 0 <= (part - merge[0][4]) // (end - begin) < merge[0][5]
    assert sorted(partial_rows) == list(range(plan._partial_rows))
    for number, (length, n) in enumerate(zip(lengths, queries)):
        for head in range(kv_heads):
            for row in range(n * group):
                parts = sorted(seen.pop((number, head, row)))
                place = length - n + row // group
                last = min(length, (place // block + 1) * block) if block else length
                first = max(0, place - window + 1) if window else 0
                assert all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
                if first < last:
                    assert parts[0][0] <= first and parts[-1][1] >= last
    assert not seen


@pytest.mark.parametrize("seed", range(12))
def test_parts_cover_their_blocks_and_share_the_work(seed):
    """Every tile of every block lies in one part; the parts of an XCD end within a tenth (and one shortest
    part) of what its workgroups cannot do without."""
    rng = np.random.default_rng(seed)
    n, resident, overhead = int(rng.integers(1, 1500)), int(rng.choice([8, 64, 512])), int(rng.integers(0, 7))
    tiles = rng.integers(0, int(rng.choice([2, 20, 600])) + 1, n) if seed % 3 else np.full(n, int(rng.integers(1, 700)))
    parts = attention._share_out(tiles, np.arange(n) // int(rng.integers(1, 40)), resident, overhead)
    block, first, last, xcd = parts.T
    at = 0
    for index, (count, total) in enumerate(zip(np.bincount(block, minlength=n), tiles)):
        own = slice(at, at + count)
        assert count >= 1 and (block[own] == index).all() and first[at] == 0 and last[at + count - 1] == total
        assert (first[own][1:] == last[own][:-1]).all() and ((last[own] > first[own]) | (total == 0)).all()
        at += count
    assert at == len(parts) and xcd.min() >= 0 and xcd.max() < 8
    if n > resident // 2:
        return
    for x in range(8):
        costs = np.sort((last - first)[xcd == x])[::-1]
        loads = [0] * max(1, resident // 8)
        for cost in costs.tolist():
            heapq.heapreplace(loads, loads[0] + cost + overhead)
        least = max((costs.sum() + len(costs) * overhead) / len(loads), -(-int(tiles.max()) // 32))
        assert max(loads) <= 1.1 * least + 2 * (overhead + 6)


@pytest.mark.parametrize("scale", [1e-46, 2.0 ** -127, 1e39, 10 ** 400, -1.0, float("inf"), True, "1"])
def test_scales_that_fp32_does_not_hold_are_refused(host, scale):
    cache = make()
    a = cache.new()
    cache.extend([a], [1])
    with pytest.raises(ConfigurationError, match="scale"):
        cache.plan([a], [1], heads=2, scale=scale)
    cache.plan([a], [1], heads=2, scale=2.0 ** -126)


def test_pending_negations_are_refused(host, monkeypatch):
    """The imaginary part of a conjugate holds its values negated."""
    monkeypatch.setattr(rotary, "need_gpu", lambda device, what: None)
    negated = torch.randn(1, 2, 8, dtype=torch.complex64).conj().imag
    assert negated.is_neg()
    cache = make()
    a = cache.new()
    slots = cache.extend([a], [1])
    cos, sin, sections = oracle.tables(8, 4)
    plan = cache.plan([a], [1], heads=2)
    for call in (lambda: rotary.rotate(negated, rk.RopePositions(rk.RopeTable(cos, sin, sections), 0), grid=(1, 1, 1), layout="THD"),
                 lambda: cache.store(0, slots, negated, torch.zeros(1, 2, 8)), lambda: cache.attend(0, negated, plan),
                 lambda: paged_cache.PagedCache(negated[None, None], torch.zeros(1, 1, 1, 2, 8))):
        with pytest.raises(ConfigurationError, match="negation"):
            call()


def test_header_matches_the_binding():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    for struct, fields in (("rch_rotary_job", _lib.ROTARY_FIELDS), ("rch_pages", _lib.PAGES_FIELDS), ("rch_attend", _lib.ATTEND_FIELDS)):
        body = re.search(r"typedef struct " + struct + r" \{(.*?)\}", text, flags=re.S).group(1)
        assert tuple(name.strip().split()[-1] for line in body.split(";") if line.strip() for name in line.split(",")) == fields
    defines = {name: int(value) for name, value in re.findall(r"#define (RCH_[A-Z0-9_]+) (\d+)\b", HEADER.read_text())}
    expected = {"RCH_PAIRS_INTERLEAVED": _lib.PAIRS_INTERLEAVED, "RCH_PAIRS_HALF": _lib.PAIRS_HALF,
                "RCH_ATTEND_ITEM": _lib.ATTEND_ITEM, "RCH_ATTEND_MERGE": _lib.ATTEND_MERGE, "RCH_ATTEND_ZEROS": _lib.ATTEND_ZEROS,
                "RCH_ATTEND_MAX_DIM": _lib.ATTEND_MAX_DIM, "RCH_ATTEND_FEW_PARTS": _lib.ATTEND_FEW_PARTS, "RCH_ATTEND_FAST_DIM": _lib.ATTEND_FAST_DIM}
    assert {name: defines.get(name) for name in expected} == expected
    lib = _lib.library()
    assert lib.rch_rotary_size() == 8 * len(_lib.ROTARY_FIELDS) and lib.rch_attend_size() == 8 * len(_lib.ATTEND_FIELDS)


def test_abi_refusals():
    """Bad arguments of the C entry points end in a status and a message, not in a launch."""
    import ctypes

    def words(fields, **values):
        return (ctypes.c_int64 * len(fields))(*(values.get(f, 0) for f in fields))

    good = dict(src_ptr=64, dst_ptr=64, batch=1, tokens=1, heads=1, head_dim=8, pairs=0)
    for bad, count, dtype, pairing in ((dict(head_dim=0), 1, 0, 0), (dict(pairs=5), 1, 0, 0), (dict(pairs=2), 1, 0, 0),
                                       (dict(slots_ptr=64), 1, 0, 0), ({}, 0, 0, 0), ({}, 5, 0, 0), ({}, 1, 3, 0), ({}, 1, 0, 2)):
        with pytest.raises(ConfigurationError):
            _lib.call("rch_rotary", words(_lib.ROTARY_FIELDS, **{**good, **bad}), count, dtype, pairing, None)
    _lib.call("rch_rotary", words(_lib.ROTARY_FIELDS, **{**good, "tokens": 0}), 1, 0, 0, None)
    pools = dict(pools_ptr=64, pools=1, pages=4, page_stride=64, page_rows=4, segments=1, row_stride=16, row_bytes=16)
    for moves in ((0, 4, 1), (4, 0, 1), (-1, 0, 1), (0, 0, 1), (0, 1, 5), (0, 1, -1)):
        with pytest.raises(ConfigurationError, match="outside the pool"):
            _lib.call("rch_pages_copy", words(_lib.PAGES_FIELDS, **pools), (ctypes.c_int32 * 3)(*moves), 1, None)
    with pytest.raises(ConfigurationError):
        _lib.call("rch_pages_copy", words(_lib.PAGES_FIELDS, **{**pools, "row_stride": 8}), (ctypes.c_int32 * 3)(0, 1, 1), 1, None)
    with pytest.raises(UnsupportedError):
        _lib.call("rch_pages_copy", words(_lib.PAGES_FIELDS, **{**pools, "row_bytes": 1 << 30, "row_stride": 1 << 30}),
                  (ctypes.c_int32 * 3)(0, 1, 1), 1, None)
    _lib.call("rch_pages_copy", words(_lib.PAGES_FIELDS, **pools), None, 0, None)
    step = dict(group=1, heads=1, head_dim=8, page_tokens=4, pages=1, n_general=1)
    for bad, dtype in ((dict(head_dim=257), 0), (dict(page_tokens=0), 0), (dict(group=0), 0), (dict(n_merges=1), 0), ({}, 0),
                       (dict(n_general=-1), 0)):
        with pytest.raises(ConfigurationError):
            _lib.call("rch_attend_run", words(_lib.ATTEND_FIELDS, **{**step, **bad}), dtype, None)
    _lib.call("rch_attend_run", words(_lib.ATTEND_FIELDS, **{**step, "n_general": 0}), 0, None)
    tiles = (ctypes.c_int64 * 2)(5, 7)
    parts, found = (ctypes.c_int64 * 8)(), ctypes.c_int64(0)
    for arguments in ((tiles, tiles, 2, 0, 0, parts, 2), (tiles, tiles, -1, 8, 0, parts, 2), (None, tiles, 2, 8, 0, parts, 2),
                      ((ctypes.c_int64 * 2)(5, -1), tiles, 2, 8, 0, parts, 2), (tiles, tiles, 2, 8, 0, parts, 0)):
        with pytest.raises(ConfigurationError):
            _lib.call("rch_attend_share", *arguments, ctypes.byref(found))
    with pytest.raises(ConfigurationError):
        _lib.call("rch_words_store", None, (ctypes.c_int32 * 1)(1), 1, None)
    run = (ctypes.c_int32 * 2)(5, 3)
    for arguments in ((None, run, 1, 3), (64, None, 1, 3), (64, run, 1, 4), (64, run, 1, 2), (64, run, -1, 0), (64, (ctypes.c_int32 * 2)(5, -1), 1, -1),
                      (64, (ctypes.c_int32 * 2)(5, -1), 1, 0)):
        with pytest.raises(ConfigurationError):
            _lib.call("rch_runs_store", *arguments, None)
    _lib.call("rch_runs_store", None, None, 0, 0, None)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tiles_start_over_where_the_kernels_take_them(dtype):
    """Every page size gets tiles that the kernels accept: of 64 keys, or within pages that hold one."""
    plan = object.__new__(attention.AttentionPlan)
    for size in range(1, 2000):
        plan.cache = types.SimpleNamespace(page_tokens=size, keys=torch.empty(0, dtype=dtype))
        unit = plan._unit()
        assert unit == attention.KEY_TILE or (unit == size and size >= attention.KEY_TILE), (size, unit)


def test_outputs_of_overlapping_rows_have_their_channels_side_by_side(monkeypatch):
    """Rows that overlap in memory (a window of one step): the launch writes a head's channels one after another,
    so the output has them so."""
    monkeypatch.setattr(rotary, "need_gpu", lambda device, what: None)
    monkeypatch.setattr(rotary, "entered", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(rotary, "_table_pairs", lambda table, device, stream: 64)
    monkeypatch.setattr(rotary, "raw_stream", lambda device: 0)
    launches = []
    monkeypatch.setattr(rotary.Launch, "__call__", lambda self, addresses, *rest: launches.append(
        dict(zip(_lib.ROTARY_FIELDS, np.frombuffer(self.image, np.int64).tolist()))))
    cos, sin, sections = oracle.tables(40, 32)
    positions = rk.RopePositions(rk.RopeTable(cos, sin, sections), 0)
    x = torch.randn(200).as_strided((9, 1, 64), (1, 64, 1))
    for _ in range(2):
        out = rotary.rotate(x, positions, grid=(1, 3, 3), layout="THD")
        assert out.shape == x.shape and out.stride(-1) == 1
    assert len(launches) == 2
    for fields in launches:
        assert (fields["dst_token_stride"], fields["dst_head_stride"]) == out.stride()[:2]
        assert fields["src_token_stride"] == 1


@pytest.mark.parametrize("tokens", [False, True])
@pytest.mark.parametrize("which", ["cos", "sin"])
def test_tables_changed_before_the_backward_pass_are_refused(monkeypatch, tokens, which):
    monkeypatch.setattr(rotary, "need_gpu", lambda device, what: None)
    monkeypatch.setattr(rotary, "entered", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(rotary, "_table_pairs", lambda table, device, stream: 64)
    monkeypatch.setattr(rotary, "raw_stream", lambda device: 0)
    monkeypatch.setattr(rotary.Launch, "__call__", lambda self, addresses, *rest: None)
    cos, sin, sections = oracle.tables(8, 4)
    table = rk.RopeTable(cos, sin, sections)
    positions = rotary.TokenRows(table, torch.zeros(6, 3, dtype=torch.int32)) if tokens else rk.RopePositions(table, 0)
    x = torch.zeros(1, 6, 2, 8, requires_grad=True)
    call = lambda: rotary.rotate(x, positions, grid=None if tokens else (1, 2, 3)).sum()
    call().backward()
    out = call()
    getattr(table, which).mul_(0.5)
    with pytest.raises(StateError, match="table was changed"):
        out.backward()
    call().backward()


def test_forward_mode_tangents_are_refused(host, monkeypatch):
    monkeypatch.setattr(rotary, "need_gpu", lambda device, what: None)
    cache = make()
    a = cache.new()
    slots = cache.extend([a], [1])
    cos, sin, sections = oracle.tables(8, 4)
    positions = rk.RopePositions(rk.RopeTable(cos, sin, sections), 0)
    plan = cache.plan([a], [1], heads=2)
    plain = torch.randn(1, 2, 8)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(plain, torch.ones_like(plain))
        pool = torch.autograd.forward_ad.make_dual(cache.keys[0], torch.ones_like(cache.keys[0]))
        for call in (lambda: rotary.rotate(dual, positions, grid=(1, 1, 1), layout="THD"),
                     lambda: rotary.rotate(plain, positions, grid=(1, 1, 1), layout="THD", out=dual),
                     lambda: cache.store(0, slots, dual, plain), lambda: cache.store(0, slots, plain, dual),
                     lambda: cache.attend(0, dual, plan), lambda: attention.attend(plain, pool, cache.values[0], plan),
                     lambda: paged_cache.PagedCache(dual[None, None], plain[None, None])):
            with pytest.raises(ConfigurationError, match="tangent"):
                call()


@pytest.mark.parametrize("which", [0, 1])
def test_attention_refuses_pools_that_require_gradients(host, which):
    cache = make()
    a = cache.new()
    cache.extend([a], [1])
    plan = cache.plan([a], [1], heads=2)
    pools = [cache.keys[0].clone(), cache.values[0].clone()]
    plan._check(*pools)
    pools[which].requires_grad_(True)
    with pytest.raises(ConfigurationError, match="differentiable"):
        attention.attend(torch.zeros(1, 2, 8), *pools, plan)
    with torch.no_grad():
        plan._check(*pools)


def test_partial_results_are_aligned():
    """The statistics of partial rows are pairs of words at even ones, whatever the head size."""
    import ctypes

    step = dict(group=1, heads=1, head_dim=7, page_tokens=4, pages=1, n_general=1, n_merges=1, n_many=1, most_rows_many=1,
                partial_rows=3, scale_bits=0x3f800000, q_ptr=64, k_ptr=64, v_ptr=64, out_ptr=64, plan_ptr=64)
    for address in (0, 4, 8):
        with pytest.raises(ConfigurationError, match="merges"):
            _lib.call("rch_attend_run", (ctypes.c_int64 * len(_lib.ATTEND_FIELDS))(
                *({**step, "partial_ptr": 1024 + address if address else 0}.get(f, 0) for f in _lib.ATTEND_FIELDS)), 0, None)


def test_a_step_has_items_of_one_form(host):
    """The cache alone says which kernels take it, and a launch of both is refused."""
    import ctypes

    for dim, dtype, tiled in ((64, torch.bfloat16, True), (20, torch.bfloat16, False), (20, torch.float32, True), (7, torch.float32, False)):
        cache = make(pages=40, dim=dim, dtype=dtype, layers=1)
        sequences = [cache.new(), cache.new()]
        cache.extend(sequences, [9, 100])
        general, rows = cache.plan(sequences, [1, 90], heads=2)._counts_of
        assert (rows > 0 and general == 0) if tiled else (general > 0 and rows == 0)
    step = dict(group=1, heads=1, head_dim=8, page_tokens=4, pages=1, n_general=1, n_rows=1)
    with pytest.raises(ConfigurationError, match="item counts"):
        _lib.call("rch_attend_run", (ctypes.c_int64 * len(_lib.ATTEND_FIELDS))(*(step.get(f, 0) for f in _lib.ATTEND_FIELDS)), 0, None)


def test_rows_of_the_pools_are_copied_before_a_store(host, monkeypatch):
    """Sources in the memory that a store writes are read whole first; sources elsewhere are read where they are."""
    launches = []
    monkeypatch.setattr(rotary.Launch, "__call__", lambda self, addresses, *rest: launches.append(
        (addresses, np.frombuffer(self.image, np.int64).reshape(2, -1)[:, 8].tolist())))
    cache = make()
    a = cache.new()
    slots = cache.extend([a], [6])
    x, y = torch.zeros(6, 2, 8), torch.zeros(6, 2, 16)[..., :8]
    cache.store(1, slots, x, y)
    (((k, _, _), (v, _, _)), strides), = launches
    assert (k, v) == (x.data_ptr(), y.data_ptr()) and strides == [16, 32]
    rows = [pool[1].flatten(0, 1)[3:9] for pool in (cache.keys, cache.values)]
    size = cache.keys[1].numel() * 4
    inside = lambda at: any(pool[1].data_ptr() <= at < pool[1].data_ptr() + size for pool in (cache.keys, cache.values))
    for keys, values in ((rows[0], y), (x, rows[1]), (rows[1], y), (x, rows[0]), tuple(rows)):
        launches.clear()
        cache.store(1, slots, keys, values)
        (((k, to_k, _), (v, to_v, _)), _), = launches
        assert not inside(k) and not inside(v)
        assert (to_k, to_v) == (cache.keys[1].data_ptr(), cache.values[1].data_ptr())
    launches.clear()
    cache.store(0, slots, *rows)  # another layer's rows are not written
    assert launches[0][0][0][0] == rows[0].data_ptr()


def test_stores_and_copies_count_as_updates_of_the_pools(host, monkeypatch):
    """A backward pass that saved a pool notices what was written into it since."""
    monkeypatch.setattr(rotary.Launch, "__call__", lambda self, addresses, *rest: None)
    x = torch.zeros(1, 2, 8)
    with torch.inference_mode():  # pools that count nothing
        cache = make()
        cache.store(0, cache.extend([cache.new()], [1]), x, x)
    cache = make()
    slots = cache.extend([cache.new()], [1])
    weight = torch.ones(1, requires_grad=True)
    for pool in (cache.keys, cache.values):
        product = (weight * pool).sum()
        cache.store(0, slots, x, x)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.backward()


def _state(cache):
    return ([(number, item.pages[:], item.tokens) for number, item in cache._sequences.items()], sorted(cache._free),
            cache._uses[:], cache._moved + cache._shared)


@pytest.mark.parametrize("failing", ["_copy", "_made"])
def test_a_failed_extend_changes_nothing(host, monkeypatch, failing):
    """No memory for the slots, or no launch: sequences, pages and their counts are as before."""
    cache = make(pages=12)
    a = cache.new()
    cache.extend([a], [6])
    b, c, d = cache.fork(a), cache.fork(a), cache.new()
    cache.extend([d], [3])
    before = _state(cache)

    def fail(*arguments):
        raise RuntimeError("out of memory")

    with monkeypatch.context() as patch:
        patch.setattr(paged_cache.PagedCache, failing, fail)
        for sequences, counts in (([b, c, a, d], [3, 1, 7, 2]), ([d, a], [0, 1]), ([b], [12]), ([a, b, c], [1, 1, 1])):
            with pytest.raises(RuntimeError, match="memory"):
                cache.extend(sequences, counts)
            assert _state(cache) == before
    assert cache.extend([b, c, a, d], [3, 1, 7, 2]).index.tolist()[:4] == [3 * 4 + 2, 3 * 4 + 3, 4 * 4, 5 * 4 + 2]
    assert cache.pages_of(a)[:2] == [0, 1]


@pytest.mark.parametrize("call", ["compact", "make_contiguous"])
def test_failed_page_moves_change_nothing(host, monkeypatch, call):
    cache = make(pages=10)
    cache.load_tables([([9, 3], 7), ([0, 7, 9], 12), ([5], 2)])
    before = _state(cache)

    def fail(*arguments):
        raise RuntimeError("no launch")

    with monkeypatch.context() as patch:
        patch.setattr(paged_cache.PagedCache, "_copy", fail)
        with pytest.raises(RuntimeError, match="launch"):
            cache.compact() if call == "compact" else cache.make_contiguous(0)
        assert _state(cache) == before
    assert cache.compact() == [(5, 1), (7, 2), (9, 4)]


def test_positions_and_slots_can_be_pickled_after_their_calls(host, monkeypatch):
    """What calls prepared is no part of a position's or slots' state."""
    monkeypatch.setattr(rotary, "need_gpu", lambda device, what: None)
    monkeypatch.setattr(rotary, "entered", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(rotary, "_table_pairs", lambda table, device, stream: 64)
    monkeypatch.setattr(rotary, "raw_stream", lambda device: 0)
    monkeypatch.setattr(rotary.Launch, "__call__", lambda self, addresses, *rest: None)
    cos, sin, sections = oracle.tables(8, 4)
    table = rk.RopeTable(cos, sin, sections)
    x = torch.zeros(6, 2, 8)
    cache = make()
    slots = cache.extend([cache.new()], [6])
    cache.store(0, slots, x, x)
    for positions, grid in ((rk.RopePositions(table, (1, 0, 2)), (1, 2, 3)), (rotary.TokenRows(table, torch.ones(6, 3, dtype=torch.int32)), None)):
        rotary.rotate(x, positions, grid=grid, layout="THD")
        assert "_known_calls" in vars(positions)
        for again in (pickle.loads(pickle.dumps(positions)), copy.deepcopy(positions)):
            assert "_known_calls" not in vars(again) and type(again) is type(positions)
            assert torch.equal(torch.as_tensor(again.rows), torch.as_tensor(positions.rows))
            assert torch.equal(again.table.cos, cos)
            rotary.rotate(x, again, grid=grid, layout="THD")
    again = pickle.loads(pickle.dumps(slots))
    assert torch.equal(again.index, slots.index) and again.cache.pages_of(0) == [0, 1]
    again.cache.store(0, again, x, x)


def test_tables_of_captured_calls_are_kept(monkeypatch):
    """A graph reads a table's device copy on every replay: it outlives the table and its updates."""
    device, state = torch.device("cpu"), {"capturing": False}
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: state["capturing"], raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: None)
    monkeypatch.setattr(rotary, "_CAPTURED_TABLES", set())
    cos, sin, sections = oracle.tables(8, 4)
    table = rk.RopeTable(cos, sin, sections)

    def use():
        entry = table._kernel_block(device, None)
        rotary._TABLE_STREAMS[entry] = {0}
        assert rotary._table_pairs(table, device, 0) == entry.pairs.data_ptr()
        return weakref.ref(entry)

    eager = use()
    table.cos.mul_(0.5)
    state["capturing"] = True
    captured = use()
    state["capturing"] = False
    table.cos.mul_(0.5)
    later = use()
    table.invalidate()
    gc.collect()
    assert eager() is None and later() is None and captured() is not None


def test_restores_into_stale_views_are_refused(host):
    """A view is a restore destination as long as its pages are its sequence's alone."""
    cache = make(pages=12, size=4, heads=2, dim=8, layers=1)
    cache.load_tables([([7, 2], 8), ([11], 4), ([5], 3)])
    job = lambda view, tokens: rk.ReconstructionJob(rk.DenseSource(torch.randn(tokens, 16)), view, (1, 1, tokens))
    restore = rk.reconstruct_reference
    changes = {
        "fork": lambda c: c.fork(0), "free": lambda c: c.free(0), "compact": lambda c: c.compact(),
        "truncate": lambda c: c.truncate(0, 3), "drop": lambda c: c.drop(0, 0, 1), "contiguous": lambda c: c.make_contiguous(0),
        "load": lambda c: c.load_tables([([7, 2], 8)]),
    }
    for name, change in changes.items():
        cache.load_tables([([7, 2], 8), ([11], 4), ([5], 3)])
        first = job(cache.view(0, "k", 0, 0, 4), 4)
        kept = job(cache.view(0, "v", 1, 1, 3), 3)
        restore([first, kept])
        assert torch.equal(cache.keys[0, 7], first.source.values.view(4, 2, 8))
        change(cache)
        before = cache.keys.clone()
        with pytest.raises(StateError, match="after this view"):
            restore([first])
        with pytest.raises(StateError, match="after this view"):
            restore([job(first.destination, 4)])
        assert torch.equal(cache.keys, before)
        if name in ("fork", "free", "truncate", "drop", "contiguous"):  # other sequences' pages are as they were
            restore([kept])
            assert torch.equal(cache.values[0, 11, 1:], kept.source.values.view(3, 2, 8))
    # Growth of the sequence, and of others, leaves a view as it is.
    cache.load_tables([([7, 2], 8), ([11], 4), ([5], 3)])
    kept = job(cache.view(0, "k", 0, 0, 4), 4)
    other = cache.fork(2)
    cache.extend([0, other], [2, 1])
    restore([kept])
    assert torch.equal(cache.keys[0, 7], kept.source.values.view(4, 2, 8))
    with pytest.raises(StateError, match="after this view"):
        stale = job(cache.view(0, "k", 0, 8, 2), 2)
        cache.fork(0)
        restore([stale])


def test_sequences_whose_keys_32_bits_do_not_count_are_refused(host):
    """Dropped pages take no room, so a sequence may be longer than its pool."""
    size = 1 << 20
    cache = make(pages=2, size=size, heads=1, dim=1, layers=1)
    for pages, fits in ((2047, True), (2048, False)):
        cache.load_tables([([paged_cache.HOLE] * (pages - 1) + [1], (pages - 1) * size + 5)])
        if fits:
            cache.plan([0], [1], heads=1)
        else:
            with pytest.raises(ConfigurationError, match="tokens"):
                cache.plan([0], [1], heads=1)


def test_rotated_tensors_require_gradients_where_their_inputs_do(host, monkeypatch):
    """Keys without a gradient that turn beside queries with one: they can be stored."""
    monkeypatch.setattr(rotary, "need_gpu", lambda device, what: None)
    monkeypatch.setattr(rotary, "entered", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(rotary, "_table_pairs", lambda table, device, stream: 64)
    monkeypatch.setattr(rotary, "raw_stream", lambda device: 0)
    launches = []
    monkeypatch.setattr(rotary.Launch, "__call__", lambda self, addresses, *rest: launches.append(len(addresses)))
    cos, sin, sections = oracle.tables(8, 4)
    positions = rk.RopePositions(rk.RopeTable(cos, sin, sections), 0)
    queries, keys = torch.zeros(6, 4, 8, requires_grad=True), torch.zeros(6, 2, 8)
    q, k = rotary.rotate((queries, keys), positions, grid=(1, 2, 3), layout="THD")
    assert q.requires_grad and not k.requires_grad
    cache = make()
    cache.store(0, cache.extend([cache.new()], [6]), k, torch.zeros(6, 2, 8))
    launches.clear()
    (q.sum() + k.sum()).backward()
    assert launches == [1] and queries.grad.shape == queries.shape
    k, q = rotary.rotate((keys, queries), positions, grid=(1, 2, 3), layout="THD")
    assert q.requires_grad and not k.requires_grad


def test_a_store_into_one_pool_for_both_is_refused(host):
    """Keys and values that are one pool can be read and copied, but a store would write each place twice."""
    pool = torch.zeros(2, 4, 4, 2, 8)
    cache = paged_cache.PagedCache(pool, pool)
    slots = cache.extend([cache.new()], [1])
    with pytest.raises(ConfigurationError, match="pools of their own"):
        cache.store(1, slots, torch.zeros(1, 2, 8), torch.zeros(1, 2, 8))
