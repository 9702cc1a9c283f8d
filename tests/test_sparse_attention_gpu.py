"""``BlockIndex`` on the GPU: means of key blocks, their choice, attention to the chosen ones."""

import math

import numpy as np
import pytest
import torch

from reelcache_amd import paged_cache, quantized_cache, sparse_attention
from reelcache_amd.errors import ConfigurationError, StateError

import history_oracle as history
import operator_oracle as oracle

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
KINDS = [(torch.bfloat16, None), (torch.float16, None), (torch.float32, None), (torch.bfloat16, torch.int8),
         (torch.float16, torch.float8_e4m3fn)]


def _cache(device, lengths, size, heads, dim, dtype, codes=None, layout="BTHD", seed=0):
    """A cache of stored sequences in scattered pages; rows that no sequence has are (or stand for) NaN."""
    pages = sum(-(-n // size) for n in lengths) + 2
    if codes is None:
        rows = (size, heads) if layout == "BTHD" else (heads, size)
        cache = paged_cache.PagedCache(*(torch.full((1, pages, *rows, dim), math.nan, dtype=dtype, device=device) for _ in range(2)), layout=layout)
    else:
        cache = quantized_cache.QuantizedCache.allocate(pages, size, heads, dim, codes=codes, dtype=dtype, device=device, layout=layout)
        for pool, scales in ((cache.keys, cache.key_scales), (cache.values, cache.value_scales)):
            pool.view(torch.uint8).fill_(1), scales.fill_(math.nan)
    order, tables = np.random.default_rng(seed).permutation(pages).tolist(), []
    for n in lengths:
        tables.append((order[:-(-n // size)], n))
        order = order[-(-n // size):]
    cache.load_tables(tables)
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn((sum(lengths), heads, dim), generator=g).to(dtype).to(device) for _ in range(2))
    cache.store(0, cache.slots(list(range(len(lengths))), [0] * len(lengths), lengths), k, v)
    return cache


def _values(cache):
    """The layer's pools as values (tensors of the cache's dtype)."""
    if not cache.codes:
        return cache.keys[0], cache.values[0]
    return tuple(history.decode(pool[0], scales[0] if cache.layout == "BHTD" else scales[0].transpose(1, 2), cache.dtype)
                 for pool, scales in ((cache.keys, cache.key_scales), (cache.values, cache.value_scales)))


def _index(cache, size, lengths):
    index = sparse_attention.BlockIndex.allocate(cache, size)
    index.update(0, cache.places(list(range(len(lengths))), [0] * len(lengths), lengths))
    return index


class _Means:
    """A sequence's means in 64 bits, from the index."""

    def __init__(self, index, sequence):
        self.rows = index.means[0].double().cpu()
        self.pages, self.heads, self.blocks = index.cache.pages_of(sequence), index.cache.heads, self.rows.shape[1]

    def __call__(self, block, head):
        return self.rows[self.pages[block // self.blocks], block % self.blocks, head]


def _check(cache, index, lengths, queries, q, chosen=None, *, top, query_block=1, first=1, recent=1, **mask):
    """Chosen blocks against the rule, and the attention over them against 64 bits."""
    plan = index.plan(list(range(len(lengths))), queries, heads=q.shape[1], top=top, query_block=query_block, first=first,
                      recent=recent, **mask)
    blocks = index.select(0, q, plan)
    out, lse = index.attend(0, q, plan, blocks=blocks, return_lse=True)
    assert torch.equal(out.isnan(), torch.zeros_like(out, dtype=torch.bool)) or chosen is not None
    assert torch.equal(out, index.attend(0, q, plan))
    keys, values = _values(cache)
    group, size = q.shape[1] // cache.heads, index.block_tokens
    run, start, widest = 0, 0, 0
    scale = mask.pop("scale", None)
    for sequence, (length, n) in enumerate(zip(lengths, queries)):
        pages = cache.pages_of(sequence)
        k, v = (history.history(x, cache.layout, pages, length) for x in (keys, values))
        rows = q[start:start + n].double().cpu()
        want = history.choice(rows, _Means(index, sequence), pages, length, n, size, cache.page_tokens, top=top,
                              query_block=query_block, first=first, recent=recent, **mask)
        held = np.repeat(np.array([page >= 0 for page in pages], dtype=bool), cache.page_tokens)[:length]
        for at, count, per_head in want:
            seen = np.array([history.visible(length, length - n + at + i, **mask) for i in range(count)]).reshape(count, length) & held
            for head, expected in enumerate(per_head):
                assert blocks[run, head].tolist() == expected + [-1] * (plan.width - len(expected)), (sequence, at, head)
                widest = max(widest, len(expected))
                shown = np.zeros(length, dtype=bool)
                for j in expected:
                    shown[j * size:(j + 1) * size] = True
                for member in range(head * group, (head + 1) * group):
                    value, bound, log, log_bound = history.attend(rows[at:at + count, member], k[:, head], v[:, head],
                                                                  seen & shown, cache.dtype, scale)
                    place = slice(start + at, start + at + count)
                    assert oracle.worst(out[place, member], value, bound) <= 0, (sequence, at, member)
                    assert oracle.worst(lse[place, member], log, log_bound) <= 0, (sequence, at, member)
            run += 1
        start += n
    assert run == plan.runs and widest == plan.width
    return plan, blocks, out


def _queries(queries, heads, dim, dtype, device, seed=5):
    return torch.randn((sum(queries), heads, dim), generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


@pytest.mark.parametrize("dtype,codes", KINDS)
@pytest.mark.parametrize("size,block,heads,dim,layout", [(16, 16, 2, 64, "BTHD"), (64, 32, 3, 128, "BHTD"), (60, 20, 1, 80, "BTHD"),
                                                         (8, 1, 2, 20, "BTHD"), (12, 4, 9, 7, "BHTD"), (200, 100, 1, 200, "BTHD"),
                                                         (96, 96, 1, 256, "BTHD")])
def test_means(device, dtype, codes, size, block, heads, dim, layout):
    """Means of the touched blocks; the others stay."""
    lengths = [5 * size, 2 * size + size // 2, 1]
    cache = _cache(device, lengths, size, heads, dim, dtype, codes, layout)
    for pool in _values(cache):
        assert pool.isnan().any()
    index = sparse_attention.BlockIndex(cache, torch.full((1, cache.pages, size // block, heads, dim), 7.0, dtype=dtype, device=device))
    begin, count = size // 2, 2 * size
    slots = cache.slots([0, 1], [begin, size], [count, 1])
    index.update(0, slots)
    touched = sorted({s // block for s in slots.index.tolist()})
    rows = history.rows_of(_values(cache)[0], layout).double().cpu().flatten(0, 1)
    means = index.means[0].flatten(0, 1).double().cpu()
    for number in range(means.shape[0]):
        if number not in touched:
            assert (means[number] == 7.0).all()
            continue
        held = rows[number * block:(number + 1) * block]
        want = held.mean(dim=0)
        # A sum in 64 bits, rounded to fp32 and then to the type.
        bound = (oracle.U[dtype] + (0 if dtype == torch.float32 else oracle.F32) + 2.0 ** -40) * want.abs() * 1.01 + oracle.TINY[dtype]
        bound += 2.0 ** -45 * held.abs().nan_to_num().sum(dim=0)
        assert oracle.worst(means[number], want, bound.nan_to_num()) <= 0


@pytest.mark.parametrize("dtype,codes", KINDS)
@pytest.mark.parametrize("size,block,heads,group,dim,layout", [
    (16, 16, 2, 1, 64, "BTHD"), (64, 32, 1, 4, 128, "BTHD"), (60, 20, 2, 2, 80, "BHTD"), (96, 96, 1, 3, 96, "BTHD"), (8, 2, 1, 2, 20, "BTHD"),
    (130, 65, 1, 1, 128, "BHTD"), (16, 8, 1, 1, 7, "BTHD"), (200, 100, 1, 2, 208, "BTHD"), (64, 64, 2, 1, 104, "BTHD"),
])
def test_single_tokens(device, dtype, codes, size, block, heads, group, dim, layout):
    """Single tokens over histories of one token up to many blocks."""
    lengths = [1, 2, 31, 64, 65, 129, 700]
    queries = [1] * len(lengths)
    cache = _cache(device, lengths, size, heads, dim, dtype, codes, layout)
    index = _index(cache, block, lengths)
    q = _queries(queries, heads * group, dim, dtype, device)
    for top, first, recent in ((3, 1, 1), (0, 0, 1), (2, 0, 0), (1000, 2, 2)):
        _check(cache, index, lengths, queries, q, top=top, first=first, recent=recent)


@pytest.mark.parametrize("dtype,codes", KINDS)
@pytest.mark.parametrize("block,window", [(None, None), (1, None), (50, None), (1, 90), (None, 70)])
@pytest.mark.parametrize("size,length,heads,group,dim,query_block", [(64, 16, 1, 1, 64, 16), (64, 32, 1, 4, 128, 33), (60, 20, 2, 1, 80, 7),
                                                                     (100, 100, 1, 1, 128, 150), (8, 4, 1, 2, 20, 10),
                                                                     (96, 48, 1, 2, 96, 30)])
def test_chunks(device, dtype, codes, block, window, size, length, heads, group, dim, query_block):
    """Chunks alone and behind histories, in runs shorter and longer than a block, and rows that see nothing."""
    lengths, queries = [70, 333, 260, 90, 3], [70, 129, 75, 1, 9 if block else 3]
    cache = _cache(device, lengths, size, heads, dim, dtype, codes)
    index = _index(cache, length, lengths)
    q = _queries(queries, heads * group, dim, dtype, device)
    for top, first, recent in ((3, 1, 1), (1, 0, 2)):
        _check(cache, index, lengths, queries, q, top=top, query_block=query_block, first=first, recent=recent, block=block, window=window)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_histories(device, dtype):
    """Hundreds of blocks: choices by more than the first eight bits, and lists in several parts."""
    lengths, queries = [20000, 9001], [1, 1]
    cache = _cache(device, lengths, 64, 1, 32, dtype)
    index = _index(cache, 16, lengths)
    q = _queries(queries, 4, 32, dtype, device)
    for top in (1, 40, 250, 700, 1249):
        _check(cache, index, lengths, queries, q, top=top)


@pytest.mark.parametrize("codes", [None, torch.int8])
def test_dropped_pages(device, codes):
    """Holes are neither scored nor taken, whatever their means and rows hold."""
    dtype, size, lengths, queries = torch.bfloat16, 32, [500, 96], [40, 1]
    cache = _cache(device, lengths, size, 1, 64, dtype, codes)
    index = _index(cache, 16, lengths)
    dropped = cache.pages_of(0)[2:9] + cache.pages_of(1)[:2]
    cache.drop(0, 2, 7)
    cache.drop(1, 0, 2)
    index.means[:, dropped] = math.nan
    if codes is None:
        cache.keys[:, dropped], cache.values[:, dropped] = math.nan, math.inf
    q = _queries(queries, 2, 64, dtype, device)
    for mask in ({}, {"block": 1}, {"window": 200}):
        _check(cache, index, lengths, queries, q, top=2, query_block=16, **mask)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_and_numbers_that_are_none(device, dtype):
    """Equal scores go to the lower block, zeros of either sign are equal, infinities rank as such and a NaN above all."""
    lengths, queries = [330], [1]
    cache = _cache(device, lengths, 16, 1, 32, dtype)
    index = _index(cache, 16, lengths)
    q = torch.ones((1, 1, 32), dtype=dtype, device=device)
    means = index.means[0]
    pages = cache.pages_of(0)
    def choose(scores, top):
        for j, value in enumerate(scores):
            means[pages[j], 0] = 0
            means[pages[j], 0, 0, 3] = value
        plan = index.plan([0], queries, heads=1, top=top, first=0, recent=1)
        return [j for j in index.select(0, q, plan)[0, 0].tolist() if 0 <= j < 20]
    assert choose([5.0] * 20, 3) == [0, 1, 2]
    assert choose([0.0, -0.0] * 10, 5) == [0, 1, 2, 3, 4]
    assert choose([1.0] * 10 + [2.0] * 10, 12) == [0, 1] + list(range(10, 20))
    assert choose([-1.0] * 19 + [-math.inf], 19) == list(range(19))
    assert choose([-math.inf] * 20, 4) == [0, 1, 2, 3]
    assert choose([1.0, math.inf, 2.0, math.nan] + [0.0] * 16, 1) == [3]
    assert choose([1.0, math.inf, 2.0, math.nan] + [0.0] * 16, 2) == [1, 3]
    assert choose([3.0, 3.0 + 8 * float(torch.finfo(dtype).eps)] * 10, 10) == list(range(1, 20, 2))
    assert choose([float(j) for j in range(20)], 20) == list(range(20))


def test_a_means_block_that_hides_a_key_is_not_scored(device):
    """NaN keys that a causal mask hides: their blocks are taken where seen in part, and change nothing elsewhere."""
    dtype, size = torch.bfloat16, 16
    cache = _cache(device, [200], size, 1, 64, dtype)
    q = _queries([100], 1, 64, dtype, device)
    index = _index(cache, size, [200])
    arguments = {"heads": 1, "top": 2, "query_block": 10, "block": 1}
    plan = index.plan([0], [100], **arguments)
    expected, blocks = index.attend(0, q, plan), index.select(0, q, plan)
    page = cache.pages_of(0)[150 // size]
    cache.keys[0, page, 150 % size], cache.values[0, page, 150 % size] = math.nan, math.nan
    index.update(0, cache.slots([0], [150], [1]))
    out, now = index.attend(0, q, plan), index.select(0, q, plan)
    assert torch.equal(now[:5], blocks[:5]) and torch.equal(out[:50], expected[:50]) and out[50:].isnan().any()


@pytest.mark.parametrize("dtype,codes", KINDS)
def test_choices_of_the_callers_own(device, dtype, codes):
    """Any lists: without order, with numbers that are no blocks, empty ones."""
    lengths, queries, size = [300, 50], [20, 1], 16
    cache = _cache(device, lengths, 32, 1, 64, dtype, codes)
    index = _index(cache, size, lengths)
    q = _queries(queries, 2, 64, dtype, device)
    plan = index.plan([0, 1], queries, heads=2, top=4, query_block=8)
    own = torch.full((plan.runs, 1, plan.width), -1, dtype=torch.int32)
    lists = [[7, 2, 18], [0], [], [3, 1]]
    for run, numbers in enumerate(lists):
        own[run, 0, :len(numbers)] = torch.tensor(numbers, dtype=torch.int32)
    own[2, 0] = torch.tensor([-5, 19, 1 << 30, -(1 << 31), 400] + [-1] * plan.width)[:plan.width]
    own[3, 0, 2] = 4  # behind the sequence
    out, lse = index.attend(0, q, plan, blocks=own.to(device), return_lse=True)
    keys, values = _values(cache)
    at = 0
    for sequence, first, n, numbers in ((0, 0, 8, lists[0]), (0, 8, 8, lists[1]), (0, 16, 4, []), (1, 20, 1, lists[3])):
        k, v = (history.history(x, "BTHD", cache.pages_of(sequence), lengths[sequence])[:, 0] for x in (keys, values))
        shown = np.zeros((n, lengths[sequence]), dtype=bool)
        for j in numbers:
            shown[:, j * size:(j + 1) * size] = True
        for member in range(2):
            want, bound, logs, log_bound = history.attend(q[first:first + n, member].double().cpu(), k, v, shown, dtype)
            assert oracle.worst(out[first:first + n, member], want, bound) <= 0
            assert oracle.worst(lse[first:first + n, member], logs, log_bound) <= 0


@pytest.mark.parametrize("dtype,codes", KINDS)
def test_means_move_with_the_pages(device, dtype, codes):
    """A fork's copied page, compaction and a copied cache: the means follow."""
    lengths = [100, 70, 33]
    cache = _cache(device, lengths, 32, 2, 64, dtype, codes)
    index = _index(cache, 8, lengths)
    q = _queries([1, 1], 4, 64, dtype, device)
    child = cache.fork(1)
    slots = cache.extend([child], [10])  # the begun page is copied with its means
    g = torch.Generator().manual_seed(8)
    cache.store(0, slots, *(torch.randn((10, 2, 64), generator=g).to(dtype).to(device) for _ in range(2)))
    index.update(0, slots)
    cache.free(0)
    assert cache.compact() or True
    sequences = [1, child]
    lengths = [cache.tokens(s) for s in sequences]
    plan = index.plan(sequences, [1, 1], heads=4, top=2)
    blocks = index.select(0, q, plan)
    for run, sequence in enumerate(sequences):
        want = history.choice(q[run:run + 1].double().cpu(), _Means(index, sequence), cache.pages_of(sequence), lengths[run], 1, 8, 32,
                              top=2, query_block=1, first=1, recent=1)
        assert [[j for j in row if j >= 0] for row in blocks[run].tolist()] == want[0][2]
    fresh = sparse_attention.BlockIndex.allocate(cache, 8)
    fresh.update(0, cache.places(sequences, [0, 0], lengths))
    for sequence, n in zip(sequences, lengths):
        for j in range(n // 8):
            page = cache.pages_of(sequence)[j // 4]
            assert torch.equal(fresh.means[0, page, j % 4], index.means[0, page, j % 4]), (sequence, j)


@pytest.mark.parametrize("sizes", [(16, 1, 4), (1, 32)])
def test_indexes_of_several_sizes_move_with_the_pages(device, sizes):
    """A fork's begun page moves in each index by its own rows."""
    cache = _cache(device, [100], 32, 2, 64, torch.bfloat16)
    cache.keys.nan_to_num_(0.0)
    indexes = [_index(cache, n, [100]) for n in sizes]
    spare = sparse_attention.BlockIndex.allocate(cache, 8)
    del spare  # moves no more
    child = cache.fork(0)
    cache.extend([child], [1])
    source, target = cache.pages_of(0)[3], cache.pages_of(child)[3]
    for n, index in zip(sizes, indexes):
        rows = -(-4 // n)
        assert source != target and torch.equal(index.means[0, target, :rows], index.means[0, source, :rows])


@pytest.mark.parametrize("dtype,codes", KINDS)
@pytest.mark.parametrize("size,block,dim,query_block", [(1, 1, 64, 1), (2, 1, 80, 5), (16, 1, 128, 64), (3, 3, 20, 2)])
def test_smallest_pages_and_blocks(device, dtype, codes, size, block, dim, query_block):
    lengths, queries = [70, 1, 9], [6, 1, 9]
    cache = _cache(device, lengths, size, 2, dim, dtype, codes)
    index = _index(cache, block, lengths)
    q = _queries(queries, 4, dim, dtype, device)
    _check(cache, index, lengths, queries, q, top=9, query_block=query_block, block=1)
    _check(cache, index, lengths, [1, 1, 1], q[:3], top=40, first=0, recent=3, window=50)


@pytest.mark.parametrize("dtype,codes", KINDS)
def test_a_run_of_steps(device, dtype, codes):
    """As a server uses them: a prompt over a history, then single tokens of it and of a fork: stored, their blocks' means
    brought up to date, and attended to, with one index, while pages are copied and moved."""
    size, block, heads, group, dim = 32, 16, 2, 4, 128
    cache = _cache(device, [200, 90], size, heads, dim, dtype, codes)
    index = _index(cache, block, [200, 90])
    g = torch.Generator().manual_seed(31)

    def step(counts):
        sequences = list(range(len(counts)))
        slots = cache.extend(sequences, counts)
        n = sum(counts)
        k, v = (torch.randn((n, heads, dim), generator=g).to(dtype).to(device) for _ in range(2))
        cache.store(0, slots, k, v)
        index.update(0, slots)
        q = torch.randn((n, heads * group, dim), generator=g).to(dtype).to(device)
        lengths = [cache.tokens(s) for s in sequences]
        _check(cache, index, lengths, counts, q, top=3, query_block=16, recent=2, block=1)

    step([20, 1])
    cache.fork(0)  # sequence 2 shares the history
    for _ in range(3):
        step([1, 1, 1])
    step([0, 1, 1])
    cache.compact()
    step([1, 1, 15])


def test_outputs_strides_and_other_rows(device):
    """``out`` with rows behind the plan's, queries of other orders, an empty plan."""
    dtype = torch.bfloat16
    lengths, queries = [300, 200], [5, 7]
    cache = _cache(device, lengths, 32, 2, 64, dtype)
    index = _index(cache, 16, lengths)
    q = _queries([20], 4, 64, dtype, device)
    plan = index.plan([0, 1], queries, heads=4, top=3, query_block=4, block=1)
    expected = index.attend(0, q, plan)
    assert not expected[12:].any()
    out = torch.full_like(q, 3.0)
    assert index.attend(0, q, plan, out=out) is out and torch.equal(out[:12], expected[:12]) and (out[12:] == 3).all()
    other = q.permute(1, 2, 0).contiguous().permute(2, 0, 1)
    assert torch.equal(index.attend(0, other, plan), expected)
    empty = index.plan([], [], heads=4, top=3)
    assert index.select(0, q[:0], empty).shape == (0, 2, 0) and index.attend(0, q[:0], empty).shape == (0, 4, 64)
    none = index.plan([0], [3], heads=4, top=0, first=0, recent=0)
    assert (index.select(0, q, none)[:, 0, 0] == 18).all()  # the block that is not full
    for call in (lambda: cache.attend(0, q, plan), lambda: index.attend(0, q, cache.plan([0], [1], heads=4)),
                 lambda: index.attend(0, q, plan, blocks=index.select(0, q, plan).long()),
                 lambda: index.attend(0, q, plan, out=q[1:])):
        with pytest.raises(ConfigurationError):
            call()
    cache.free(1)
    with pytest.raises(StateError):
        index.attend(0, q, plan)


def test_streams_and_captured_replays(device):
    """Update, choice and attention in two graphs with one plan, replayed in turn and at once, with eager work between."""
    dtype = torch.bfloat16
    cache = _cache(device, [3000, 130], 64, 2, 128, dtype)
    cache.keys.nan_to_num_(0.0), cache.values.nan_to_num_(0.0)
    index = _index(cache, 32, [3000, 130])
    slots = cache.slots([0], [2900], [100])
    plan = index.plan([0, 1], [100, 1], heads=4, top=5, query_block=25)
    q = _queries([101], 4, 128, dtype, device)
    k = torch.randn((100, 2, 128), generator=torch.Generator().manual_seed(1)).to(dtype).to(device)

    def step():
        cache.store(0, slots, k, k)
        index.update(0, slots)
        blocks = index.select(0, q, plan)
        return blocks, index.attend(0, q, plan, blocks=blocks)

    expected = step()
    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        other = step()
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, expected))
    graphs, outs = [], []
    for captured in (step, lambda: (index.select(0, q, plan), index.attend(0, q, plan))):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(captured())
        graphs.append(graph)
    for replay in range(3):
        for x in (k, q):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(10 + replay)))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize(device)
        found = [[t.clone() for t in out] for out in outs]
        want = step()
        for out in found:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    sides = [torch.cuda.Stream(device) for _ in graphs]
    torch.cuda.synchronize(device)
    for side in sides:  # the attention of both at once (the keys stay as they are)
        with torch.cuda.stream(side):
            graphs[1].replay() if side is sides[0] else index.attend(0, q, plan)
    torch.cuda.synchronize(device)
    assert all(torch.equal(a, b) for a, b in zip(outs[1], want))


@pytest.mark.parametrize("dtype,codes", [(torch.bfloat16, None), (torch.bfloat16, torch.int8), (torch.float16, torch.float8_e4m3fn)])
@pytest.mark.parametrize("size,block,dim,layout", [(1024, 32, 16, "BTHD"), (64, 2, 128, "BHTD"), (50, 25, 104, "BTHD")])
def test_pools_past_32_bits(device, dtype, codes, size, block, dim, layout):
    """Pages, scales and means that lie more than 2^32 bytes into their pools: the bits of the same sequence in a small
    cache, stored, read, indexed, chosen and attended to."""
    heads, n, queries = 2, 6 * size - 7, 130
    near = (1 << 30) // (size * heads) if dim == 16 else (1 << 32) // (size * heads * dim)  # (of 16 channels the scales lie as far)
    results = []
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn((n, heads, dim), generator=g).to(dtype).to(device) for _ in range(2))
    q = torch.randn((queries, 2 * heads, dim), generator=g).to(dtype).to(device)
    for pages in (9, near + 9):
        rows = (size, heads) if layout == "BTHD" else (heads, size)
        if codes is None:
            cache = paged_cache.PagedCache(*(torch.empty((1, pages, *rows, dim), dtype=dtype, device=device) for _ in range(2)), layout=layout)
        else:
            cache = quantized_cache.QuantizedCache.allocate(pages, size, heads, dim, codes=codes, dtype=dtype, device=device, layout=layout)
        cache.load_tables([([pages - 1 - i for i in range(6)], n)])
        slots = cache.slots([0], [0], [n])
        cache.store(0, slots, k, v)
        index = cache.index(block)
        index.update(0, slots)
        found = [*cache.read(0, slots)] if codes is not None else []
        for count in (queries, 1):
            plan = index.plan([0], [count], heads=2 * heads, top=5, query_block=16, block=1)
            blocks = index.select(0, q[:count], plan)
            found += [blocks, index.attend(0, q[:count], plan, blocks=blocks),
                      cache.attend(0, q[:count], cache.plan([0], [count], heads=2 * heads, block=1))]
        results.append([x.cpu() for x in found])
        far = max(pool[0, pages - 6:].data_ptr() - pool.data_ptr() for pool in (cache.keys, *([] if codes is None else [cache.key_scales])))
        assert (far > 1 << 32) == (pages > 9)
        del cache, index, slots, plan
    for small, large in zip(*results):
        assert not small.isnan().any() and torch.equal(small, large)


def _ranked(means, pooled, held, scored, always, top):
    """The rule for one run and key head, from exact scores: ``means`` float64 [blocks, D], ``scored`` ascending."""
    scored = scored[held[scored]]
    scores = means[scored] @ pooled
    none = np.isnan(scores)
    order = scored[np.lexsort((scored, np.where(none, 0.0, -scores), ~none))]
    return sorted([j for j in always if held[j]] + order[:top].tolist())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("blocks,queries,query_block,heads,group,dim", [
    (300, 70, 1, 2, 1, 16), (1000, 70, 1, 2, 2, 7), (4096, 64, 1, 2, 1, 8), (4100, 90, 1, 2, 1, 8), (3000, 260, 2, 1, 2, 64),  # a launch
    (300, 9, 1, 1, 2, 16), (4090, 3, 1, 2, 1, 8), (4500, 4, 1, 1, 1, 16), (4098, 70, 1, 2, 1, 8), (9001, 66, 1, 2, 1, 8),  # two launches
])
def test_choices_among_many_blocks(device, dtype, blocks, queries, query_block, heads, group, dim, monkeypatch):
    """Every path of a choice: numbers in LDS and in memory, in one launch and in two, with equal scores on both sides of every
    256th and 1024th block, holes and NaN.  Small whole numbers, so that the scores are exact and few."""
    size, length = 4, blocks * 4 - 1  # the last block is not full
    cache = paged_cache.PagedCache.allocate(blocks, size, heads, dim, dtype=dtype, device=device)
    order = np.random.default_rng(blocks).permutation(blocks).tolist()
    cache.load_tables([(order, length)])
    index = sparse_attention.BlockIndex.allocate(cache, size)
    g = torch.Generator().manual_seed(blocks)
    means = torch.randint(-1, 2, (blocks, heads, dim), generator=g).float()
    means[torch.randint(0, blocks, (3,), generator=g), 0, 0] = math.nan
    index.means[0, :, 0] = means[torch.tensor(order).argsort()].to(dtype).to(device)
    for first in (100, 255, 1023):
        if first < blocks - 2:
            cache.drop(0, first, 2)
    held = np.array(cache.pages_of(0)) >= 0
    q = torch.randint(-1, 2, (queries, heads * group, dim), generator=g).to(dtype).to(device)
    rows, exact = q.double().cpu().numpy(), means.double().numpy()
    for top, first, recent in ((1, 1, 1), (37, 0, 0), (blocks // 3, 2, 3), (blocks - 20, 0, 1), (blocks, 0, 0)):
        plan = index.plan([0], [queries], heads=heads * group, top=top, query_block=query_block, first=first, recent=recent)
        assert plan._scores == blocks - 1 - first
        found = index.select(0, q, plan)
        assert plan._apart == (plan._scores > (256 if plan.runs * heads < 128 else 4096))
        if plan._apart and plan.runs > 1:  # the same in several launches
            with monkeypatch.context() as patch:
                patch.setattr(sparse_attention, "_SCORE_BYTES", 8 * heads * plan._scores * 2 + 1)
                assert torch.equal(index.select(0, q, plan), found)
        found = found.cpu()
        for run in sorted({0, 1, plan.runs // 2, plan.runs - 1} & set(range(plan.runs))):
            begin, end = run * query_block, min((run + 1) * query_block, queries)
            own = (length - queries + end - 1) // size
            always = sorted({j for j in range(blocks) if j < first or own - recent < j <= own} | {blocks - 1})
            scored = np.setdiff1d(np.arange(blocks), always)
            for head in range(heads):
                pooled = rows[begin:end, head * group:(head + 1) * group].sum(axis=(0, 1))
                want = _ranked(exact[:, head], pooled, held, scored, always, top)
                assert found[run, head].tolist() == want + [-1] * (plan.width - len(want)), (top, run, head)


@pytest.mark.parametrize("dtype,codes", KINDS)
def test_means_and_choices_after_compaction(device, dtype, codes):
    """Pages that moved, each with its means."""
    lengths = [100, 70, 33]
    cache = _cache(device, lengths, 32, 2, 64, dtype, codes)
    index = _index(cache, 8, lengths)
    kept = [1, 2]
    before = [[index.means[0, cache.pages_of(s)[j // 4], j % 4].clone() for j in range(lengths[s] // 8)] for s in kept]
    q = _queries([1, 1], 4, 64, dtype, device)
    plan = index.plan(kept, [1, 1], heads=4, top=2)
    blocks, out = index.select(0, q, plan), index.attend(0, q, plan)
    pages = [cache.pages_of(s) for s in kept]
    cache.free(0)
    assert cache.compact() and [cache.pages_of(s) for s in kept] != pages
    for s, means in zip(kept, before):
        for j, mean in enumerate(means):
            assert torch.equal(index.means[0, cache.pages_of(s)[j // 4], j % 4], mean), (s, j)
    plan = index.plan(kept, [1, 1], heads=4, top=2)
    assert torch.equal(index.select(0, q, plan), blocks) and torch.equal(index.attend(0, q, plan), out)


@pytest.mark.parametrize("dtype,codes", [(torch.bfloat16, None), (torch.bfloat16, torch.float8_e4m3fn), (torch.float16, torch.int8)])
def test_graphs_and_eager_calls_at_once(device, dtype, codes):
    """Two captured steps and an eager one on streams of their own, at the same time: each has the results that it has alone.
    One graph stores into a cache of its own; the other and the eager step share a cache, an index and plans."""
    lengths, queries = [6000, 130], [60, 1]
    caches = [_cache(device, lengths, 64, 2, 128, dtype, codes, seed=seed) for seed in (0, 1)]
    for cache in caches:
        if codes is None:
            cache.keys.nan_to_num_(0.0), cache.values.nan_to_num_(0.0)
    indexes = [_index(cache, 16, lengths) for cache in caches]
    # Runs of 6000 / 16 blocks: 3 x 2 of them are scored in launches of their own, for single tokens too.
    plans = [index.plan([0, 1], queries, heads=8, top=200, query_block=30) for index in indexes]
    tokens = indexes[1].plan([0, 1], [1, 1], heads=8, top=200)
    assert plans[0]._apart and tokens._apart and plans[0]._n_merges
    qs = [_queries([61], 8, 128, dtype, device, seed=seed) for seed in range(3)]
    slots = caches[0].slots([0], [5940], [60])
    k = torch.randn((60, 2, 128), generator=torch.Generator().manual_seed(1)).to(dtype).to(device)

    def storing():
        caches[0].store(0, slots, k, k)
        indexes[0].update(0, slots)
        blocks = indexes[0].select(0, qs[0], plans[0])
        return (blocks, *indexes[0].attend(0, qs[0], plans[0], blocks=blocks, return_lse=True))

    def reading(q):
        return (indexes[1].select(0, q, plans[1]), *indexes[1].attend(0, q, plans[1], return_lse=True), indexes[1].attend(0, q[:2], tokens))

    torch.cuda.synchronize(device)
    sides = [torch.cuda.Stream(device) for _ in range(3)]
    graphs, outs = [], []
    storing(), reading(qs[1])
    torch.cuda.synchronize(device)
    for side, step in zip(sides, (storing, lambda: reading(qs[1]))):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(step())
        graphs.append(graph)
    for replay in range(4):
        for i, x in enumerate((k, *qs)):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(10 * replay + i)))
        torch.cuda.synchronize(device)
        want = [[t.clone() for t in step] for step in (storing(), reading(qs[1]), reading(qs[2]))]
        for out in outs:
            for t in out:
                t.zero_()
        torch.cuda.synchronize(device)
        for side, graph in zip(sides, graphs):
            with torch.cuda.stream(side):
                graph.replay()
        with torch.cuda.stream(sides[2]):
            eager = reading(qs[2])
        torch.cuda.synchronize(device)
        for found, expected in zip((*outs, eager), want):
            assert all(torch.equal(a, b) for a, b in zip(found, expected)), replay


@pytest.mark.parametrize("dtype,codes", KINDS)
@pytest.mark.parametrize("dim", [64, 20])
def test_runs_that_take_nothing(device, dtype, codes, dim):
    """No leading, recent or chosen block, and every block full: queries that attend to nothing, in every form."""
    lengths = [256, 64]
    cache = _cache(device, lengths, 64, 2, dim, dtype, codes)
    for block in (16, 64):
        index = _index(cache, block, lengths)
        for queries in ([1, 1], [40, 3]):
            q = _queries(queries, 4, dim, dtype, device)
            plan = index.plan([0, 1], queries, heads=4, top=0, first=0, recent=0, query_block=8)
            assert plan.width == 0 and index.select(0, q, plan).shape == (plan.runs, 2, 0)
            out, lse = index.attend(0, q, plan, return_lse=True)
            assert not out.any() and (lse == -math.inf).all()
            _check(cache, index, lengths, queries, q, top=1, first=0, recent=0, query_block=8)


def test_reads_follow_a_sequence_into_its_copied_page(device):
    """Two sequences of one history go on apart and rewrite their last rows: each is read as it is, and old places are refused."""
    dtype = torch.bfloat16
    cache = quantized_cache.QuantizedCache.allocate(8, 16, 2, 64, codes=torch.int8, dtype=dtype, device=device)
    index = cache.index(8)
    a = cache.new()
    slots = cache.extend([a], [30])
    g = torch.Generator().manual_seed(2)
    rows = [torch.randn((30, 2, 64), generator=g).to(dtype).to(device) for _ in range(3)]
    cache.store(0, slots, rows[0], rows[0])
    index.update(0, slots)
    b = cache.fork(a)
    old = cache.places([a], [0], [30])
    cache.extend([a], [1])
    for sequence, x in ((a, rows[1]), (b, rows[2])):
        slots = cache.slots([sequence], [16], [14])
        cache.store(0, slots, x[:14], x[:14])
        index.update(0, slots)
    for call in (lambda: cache.read(0, old), lambda: index.update(0, old)):
        with pytest.raises(StateError):
            call()
    for sequence, x in ((a, rows[1]), (b, rows[2])):
        want = history.decode(*history.encode(torch.cat([rows[0][:16], x[:14]]), torch.int8), dtype)
        for found in cache.read(0, cache.places([sequence], [0], [30])):
            assert torch.equal(found.cpu(), want)
        # The mean of its block of rows 16 to 23: a sum in 64 bits, rounded to fp32 and then to the type.
        mean, exact = index.means[0, cache.pages_of(sequence)[1], 0].double().cpu(), want[16:24].double().mean(dim=0)
        assert ((mean - exact).abs() <= (oracle.U[dtype] + oracle.F32 + 2.0 ** -40) * 1.01 * exact.abs() + oracle.TINY[dtype]).all()
