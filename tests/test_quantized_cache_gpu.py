"""``QuantizedCache`` on the GPU: codes and scales, what they stand for, page copies, attention over them."""

import copy
import math

import numpy as np
import pytest
import torch

from reelcache_amd import paged_cache, quantized_cache, rotary
from reelcache_amd import restore_kernels as rk
from reelcache_amd.errors import ConfigurationError

import history_oracle as history
import operator_oracle as oracle

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]
CODES = [torch.int8, torch.float8_e4m3fn]
SHAPES = [(16, 2, 64, "BTHD"), (64, 3, 128, "BHTD"), (7, 1, 80, "BTHD"), (30, 5, 96, "BHTD"), (16, 2, 256, "BTHD"), (8, 2, 200, "BTHD"),
          (16, 1, 20, "BTHD"), (9, 3, 7, "BHTD"), (16, 9, 8, "BTHD"), (5, 1, 1, "BTHD"), (12, 2, 104, "BHTD"), (11, 1, 250, "BTHD")]


def _empty(device, pages, size, heads, dim, codes, dtype, layout="BTHD", layers=1):
    """A cache whose codes are 1 and whose scales are NaN, so that rows nobody wrote are seen."""
    cache = quantized_cache.QuantizedCache.allocate(pages, size, heads, dim, codes=codes, layers=layers, dtype=dtype, device=device,
                                                    layout=layout)
    for pool, scales in ((cache.keys, cache.key_scales), (cache.values, cache.value_scales)):
        pool.view(torch.uint8).fill_(1)
        scales.fill_(math.nan)
    return cache


def _random(shape, dtype, seed, device):
    """Values of several sizes: channels, rows of small and large ones, rows of zeros."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp2(torch.randint(-9, 9, (shape[0], shape[1], 1), generator=g).float())
    x *= torch.rand(shape[2], generator=g) + 0.1
    x[::5, 0] = 0
    return x.to(dtype).to(device)


def _rows(pool, scales, slots, layout):
    """(codes as numbers, scales) of slots, on the CPU."""
    codes = history.rows_of(pool, layout).float().cpu().flatten(0, 1)
    return codes[slots], scales.transpose(1, 2).cpu().flatten(0, 1)[slots]


def _same(a, b):
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size,heads,dim,layout", SHAPES)
def test_codes_scales_and_values(device, codes, dtype, size, heads, dim, layout):
    """Codes and scales are those that fp32 arithmetic defines, bit by bit; other rows stay; reading gives what they stand
    for."""
    cache = _empty(device, 12, size, heads, dim, codes, dtype, layout, layers=2)
    a, b = cache.new(), cache.new()
    cache.extend([a, b], [3, 1])
    slots = cache.extend([b, a], [2 * size + 1, size])
    k, v = (_random((slots.tokens, heads, dim), dtype, seed, device) for seed in (1, 2))
    cache.store(1, slots, k, v)
    index = slots.index.cpu().long()
    others = torch.ones(12 * size, dtype=torch.bool)
    others[index] = False
    for x, pool, scales in ((k, cache.keys, cache.key_scales), (v, cache.values, cache.value_scales)):
        code, scale = history.encode(x, codes)
        got, got_scale = _rows(pool[1], scales[1], index, layout)
        assert torch.equal(got, code.float()) and torch.equal(got_scale, scale)
        got, got_scale = _rows(pool[1], scales[1], others, layout)
        assert (got == torch.ones(1, dtype=torch.uint8).view(codes).float()).all() and got_scale.isnan().all()
        assert scales[0].isnan().all()
    for found, x in zip(cache.read(1, slots), (k, v)):
        assert found.dtype == dtype and _same(found.cpu(), history.decode(*history.encode(x, codes), dtype))
    # And within what the formats promise: half a step of m / 127 (a product and a reciprocal rounded: 2^-15 of a step
    # more), or 2^-4 of the value (2^-10 of the scale for small ones); then one rounding to the type.
    for found, x in zip(cache.read(1, slots), (k, v)):
        x, found = x.double().cpu(), found.double().cpu()
        scale = history.encode(x, codes)[1].double()[..., None]
        off = (0.5 + 2.0 ** -15) * scale if codes == torch.int8 else torch.maximum(x.abs() * 2.0 ** -4, scale * 2.0 ** -10)
        assert ((found - x).abs() <= off * 1.0001 + oracle.U[dtype] * found.abs() + oracle.TINY[dtype]).all()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size,heads,dim,layout,pairs", [(16, 2, 64, "BTHD", 32), (6, 5, 128, "BHTD", 64), (7, 1, 80, "BTHD", 24),
                                                         (16, 2, 256, "BTHD", 128), (9, 3, 7, "BHTD", 3), (16, 1, 22, "BTHD", 11)])
def test_keys_are_rotated_first(device, codes, dtype, size, heads, dim, layout, pairs):
    grid = (2, 3, 5)
    n = 30
    cos, sin, sections = oracle.tables(20, pairs)
    table = rk.RopeTable(cos, sin, sections)
    cache = _empty(device, 8, size, heads, dim, codes, dtype, layout)
    slots = cache.extend([cache.new()], [n])
    k, v = (_random((n, heads, dim), dtype, seed, device) for seed in (1, 2))
    rows = oracle.grid_rows((4, 1, 2), grid)
    want = history.encode(history.rotated(k, *oracle.token_angles(cos, sin, sections, rows)), codes, dtype)
    for positions, given in ((rk.RopePositions(table, (4, 1, 2)), grid), (rotary.TokenRows(table, rows.to(device)), None)):
        cache.keys.view(torch.uint8).fill_(1)
        cache.store(0, slots, k, v, positions=positions, grid=given)
        got, scale = _rows(cache.keys[0], cache.key_scales[0], slots.index.cpu().long(), layout)
        assert torch.equal(got, want[0].float()) and torch.equal(scale, want[1])
        assert _same(cache.read(0, slots)[1].cpu(), history.decode(*history.encode(v, codes), dtype))


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_largest_smallest_and_values_that_are_none(device, codes, dtype):
    """Rows at the ends of the type, at borders of the formats, and with infinities and NaN."""
    dim = 16
    most, least = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    rows = [[most, -most, 1.0], [least, -least], [least / 4], [0.0], [127.0, 63.5, -63.5, 0.5, 1.5, -0.5], [448.0, 449.0, 3.5],
            [447.0, 0.0009765625], [1.75, 1.7578125], [math.inf, 1.0], [1.0, -math.inf], [math.nan, 2.0], [2.0 ** -14, 1.0]]
    x = torch.zeros(len(rows), 1, dim)
    for i, row in enumerate(rows):
        x[i, 0, :len(row)] = torch.tensor(row)
    x = x.to(dtype).to(device)
    cache = _empty(device, 4, 4, 1, dim, codes, dtype)
    slots = cache.extend([cache.new()], [len(rows)])
    cache.store(0, slots, x, x.flip(2))
    code, scale = history.encode(x, codes)
    got, got_scale = _rows(cache.keys[0], cache.key_scales[0], slots.index.cpu().long(), "BTHD")
    assert torch.equal(got, code.float()) and _same(got_scale, scale)
    keys, values = (t.cpu() for t in cache.read(0, slots))
    assert _same(keys, history.decode(code, scale, dtype)) and _same(values, keys.flip(2))
    assert keys[8:11].isnan().all() and torch.isfinite(keys[:8]).all() and torch.isfinite(keys[11]).all()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dim", [64, 20])
def test_strided_sources_outputs_and_pools(device, codes, dim):
    """Sources and outputs of other orders, a pool with room behind its rows, scales with gaps."""
    dtype, heads, size, pages = torch.bfloat16, 3, 8, 6
    pools = [torch.zeros(2, pages, size, heads, dim + 16, dtype=torch.uint8, device=device)[..., :dim].view(codes) for _ in range(2)]
    scales = [torch.zeros(2, pages, heads, size + 3, device=device)[..., :size] for _ in range(2)]
    cache = quantized_cache.QuantizedCache(*pools, *scales, dtype=dtype)
    slots = cache.extend([cache.new()], [21])
    k = _random((heads, 21, dim), dtype, 1, device).transpose(0, 1)
    v = _random((21, dim, heads), dtype, 2, device).transpose(1, 2)
    cache.store(1, slots, k, v)
    want = [history.decode(*history.encode(x, codes), dtype) for x in (k, v)]
    out = torch.empty(heads, 21, dim, dtype=dtype, device=device).transpose(0, 1), torch.empty(21, dim, heads, dtype=dtype, device=device).transpose(1, 2)
    version = out[0]._version
    assert cache.read(1, slots, out=out) == out and out[0]._version > version
    for found in (out, cache.read(1, slots)):
        assert all(_same(a.cpu(), b) for a, b in zip(found, want))
    assert not cache.keys[0].view(torch.uint8).any() and not cache.key_scales[0].any()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("layout", ["BTHD", "BHTD"])
def test_pages_move_with_their_scales(device, codes, layout):
    """Forks that go on apart, and compaction, in every layer; a copied cache moves its own."""
    dtype, heads, size, dim, layers = torch.float16, 2, 8, 32, 3
    cache = _empty(device, 16, size, heads, dim, codes, dtype, layout, layers)
    spare = cache.new()
    cache.extend([spare], [3 * size])
    a = cache.new()
    slots = cache.extend([a], [2 * size + 3])
    stored = [[_random((2 * size + 3, heads, dim), dtype, 10 * layer + i, device) for i in range(2)] for layer in range(layers)]
    for layer, (k, v) in enumerate(stored):
        cache.store(layer, slots, k, v)
    b = cache.fork(a)
    more = cache.extend([b], [2])
    new = [_random((2, heads, dim), dtype, 90 + i, device) for i in range(2)]
    for layer in range(layers):
        cache.store(layer, more, *new)
    cache.free(spare)
    other = copy.deepcopy(cache)
    kept = [t.clone() for t in (cache.keys.view(torch.uint8), cache.key_scales, cache.values.view(torch.uint8), cache.value_scales)]
    assert other.compact()
    now = (cache.keys.view(torch.uint8), cache.key_scales, cache.values.view(torch.uint8), cache.value_scales)
    assert all(_same(x.float(), y.float()) for x, y in zip(kept, now))
    assert cache.compact()
    for which in (cache, other):
        for layer, pair in enumerate(stored):
            for sequence, tail in ((a, None), (b, new)):
                n = which.tokens(sequence)
                found = which.read(layer, which.places([sequence], [0], [n]))
                for i, x in enumerate(pair):
                    x = x if tail is None else torch.cat([x, tail[i]])
                    assert _same(found[i].cpu(), history.decode(*history.encode(x, codes), dtype))


def _filled(device, lengths, size, heads, dim, codes, dtype, layout="BTHD", seed=0):
    """A cache of stored sequences; rows that no sequence has stand for NaN."""
    pages = sum(-(-n // size) for n in lengths) + 2
    cache = _empty(device, pages, size, heads, dim, codes, dtype, layout)
    order = np.random.default_rng(seed).permutation(pages).tolist()
    tables = []
    for n in lengths:
        count = -(-n // size)
        tables.append((order[:count], n))
        order = order[count:]
    cache.load_tables(tables)
    numbers = list(range(len(lengths)))
    slots = cache.slots(numbers, [0] * len(lengths), lengths)
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn((sum(lengths), heads, dim), generator=g).to(dtype).to(device) for _ in range(2))
    cache.store(0, slots, k, v)
    return cache


def _native(cache):
    """The cache of the values that a quantised one's codes stand for."""
    pools = []
    for pool, scales in ((cache.keys, cache.key_scales), (cache.values, cache.value_scales)):
        scales = scales if cache.layout == "BHTD" else scales.transpose(2, 3)
        pools.append(history.decode(pool, scales, cache.dtype))
    native = paged_cache.PagedCache(*pools, layout=cache.layout)
    native.load_tables([(cache.pages_of(s), cache.tokens(s)) for s in cache._sequences])
    return native


def _check(cache, lengths, queries, q, **mask):
    """Against 64 bits over the values read back and, where both take the matrix cores, their bits."""
    native = _native(cache)
    plan = cache.plan(list(range(len(lengths))), queries, heads=q.shape[1], **mask)
    out, lse = cache.attend(0, q, plan, return_lse=True)
    start = 0
    for sequence, (length, n) in enumerate(zip(lengths, queries)):
        rows = slice(start, start + n)
        want, bound, logs, log_bound = oracle.attend(q[rows], native.keys[0], native.values[0], cache.pages_of(sequence), length, n,
                                                     cache.page_tokens, layout=cache.layout, **mask)
        assert oracle.worst(out[rows], want, bound) <= 0, (sequence, length, n)
        assert oracle.worst(lse[rows], logs, log_bound) <= 0, (sequence, length, n)
        start += n
    assert torch.equal(out, cache.attend(0, q, plan))
    if cache.head_dim % 16 == 0 and not plan._single:  # (single tokens take smaller tiles)
        same = native.plan(list(range(len(lengths))), queries, heads=q.shape[1], **mask)
        assert torch.equal(out, native.attend(0, q, same))
    return out


def _run(device, lengths, queries, size, heads, group, dim, codes, dtype, layout="BTHD", seed=0, **mask):
    cache = _filled(device, lengths, size, heads, dim, codes, dtype, layout, seed)
    q = torch.randn((sum(queries), heads * group, dim), generator=torch.Generator().manual_seed(seed + 1)).to(dtype).to(device)
    return _check(cache, lengths, queries, q, **mask)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size,heads,group,dim,layout", [
    (16, 2, 1, 64, "BTHD"), (64, 1, 4, 128, "BTHD"), (100, 2, 2, 80, "BHTD"), (7, 1, 3, 96, "BTHD"), (130, 3, 1, 128, "BHTD"),
    (16, 1, 2, 20, "BTHD"), (9, 2, 1, 208, "BTHD"), (16, 1, 1, 7, "BHTD"), (64, 1, 1, 16, "BTHD"), (33, 1, 2, 104, "BTHD"), (70, 1, 2, 256, "BTHD"),
])
def test_single_tokens(device, codes, dtype, size, heads, group, dim, layout):
    lengths = [1, 2, 31, 64, 65, 129, 300]
    _run(device, lengths, [1] * len(lengths), size, heads, group, dim, codes, dtype, layout)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block,window", [(None, None), (1, None), (40, None), (1, 33)])
@pytest.mark.parametrize("size,heads,group,dim,layout", [
    (16, 1, 1, 64, "BTHD"), (64, 1, 2, 128, "BTHD"), (100, 1, 1, 80, "BHTD"), (7, 1, 1, 128, "BTHD"), (16, 1, 1, 20, "BTHD"),
    (150, 1, 1, 96, "BTHD"), (60, 1, 1, 192, "BHTD"),
])
def test_chunks(device, codes, dtype, block, window, size, heads, group, dim, layout):
    """Chunks alone, behind a history, beside single tokens, and rows that see nothing."""
    _run(device, [70, 133, 260, 90, 40, 3], [70, 129, 75, 1, 33, 9 if block else 3], size, heads, group, dim, codes, dtype, layout,
         block=block, window=window)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dim,size", [(128, 16), (64, 64), (128, 100), (20, 8)])
def test_dropped_pages_and_hidden_rows(device, codes, dim, size):
    """Dropped pages are not seen; a row that stands for NaN harms only the queries that see it."""
    dtype, lengths, queries = torch.bfloat16, [8 * size + 3, 3 * size], [size + 3, 1]
    cache = _filled(device, lengths, size, 1, dim, codes, dtype)
    dropped = cache.pages_of(0)[2:5] + cache.pages_of(1)[:2]
    cache.drop(0, 2, 3)
    cache.drop(1, 0, 2)
    cache.key_scales[:, dropped], cache.value_scales[:, dropped] = math.nan, math.inf
    q = torch.randn((sum(queries), 2, dim), generator=torch.Generator().manual_seed(3)).to(dtype).to(device)
    for mask in ({}, {"block": 1}, {"window": size}):
        _check(cache, lengths, queries, q, **mask)
    cache = _filled(device, [210, 20], size, 1, dim, codes, dtype)
    q = torch.randn((170, 1, dim), generator=torch.Generator().manual_seed(3)).to(dtype).to(device)
    expected = cache.attend(0, q, cache.plan([0, 1], [150, 20], heads=1, block=1))
    bad = 150  # its query is row 90
    cache.value_scales[0, cache.pages_of(0)[bad // size], 0, bad % size] = math.nan
    out = cache.attend(0, q, cache.plan([0, 1], [150, 20], heads=1, block=1))
    assert torch.equal(out[:90], expected[:90]) and torch.equal(out[150:], expected[150:]) and out[90:150].isnan().all()


@pytest.mark.parametrize("codes", CODES)
def test_long_split_histories(device, codes):
    """Keys of single tokens in many parts, in pages of a tile and of less."""
    for size in (64, 16, 1560):
        cache = _filled(device, [9000, 4001], size, 2, 128, codes, torch.bfloat16)
        q = torch.randn((2, 8, 128), generator=torch.Generator().manual_seed(3)).bfloat16().to(device)
        native = _native(cache)
        plan = cache.plan([0, 1], [1, 1], heads=8)
        assert plan._n_merges and plan._single
        out, lse = cache.attend(0, q, plan, return_lse=True)
        k, v = (history.rows_of(x[0], "BTHD").double().cpu() for x in (native.keys, native.values))
        for sequence, length in ((0, 9000), (1, 4001)):
            pages = torch.tensor(cache.pages_of(sequence))
            for head in range(8):
                keys, values = (x[pages][:, :, head // 4].flatten(0, 1)[:length] for x in (k, v))
                want, bound, logs, log_bound = history.attend(q[sequence:sequence + 1, head].double().cpu(), keys, values,
                                                              np.ones((1, length), dtype=bool), torch.bfloat16)
                assert oracle.worst(out[sequence:sequence + 1, head], want, bound) <= 0
                assert oracle.worst(lse[sequence:sequence + 1, head], logs, log_bound) <= 0


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [16, 64, 96, 128, 192, 256])
def test_single_tokens_of_many_heads(device, codes, dtype, dim):
    """Groups of up to 32 heads, and more, over pages in one piece and in many; a window; keys that hide NaN."""
    for group in (1, 8, 32, 33):
        for size in (64, 16, 5):
            cache = _filled(device, [200, 33, 1], size, 1, dim, codes, dtype)
            q = torch.randn((3, group, dim), generator=torch.Generator().manual_seed(group)).to(dtype).to(device)
            _check(cache, [200, 33, 1], [1, 1, 1], q)
            _check(cache, [200, 33, 1], [1, 1, 1], q, window=70)
            plan = cache.plan([0], [1], heads=group, window=70)
            assert plan._single == (group <= 32)
            expected = cache.attend(0, q[:1], plan)
            for at in (0, 100, 129):  # hidden by the window
                page = cache.pages_of(0)[at // size]
                cache.key_scales[0, page, 0, at % size], cache.value_scales[0, page, 0, at % size] = math.nan, math.nan
            assert torch.equal(cache.attend(0, q[:1], plan), expected)


def test_scales_beyond_fp16(device):
    """Codes of values at the ends of fp16: the product with the scale is rounded, never the scale."""
    cache = _filled(device, [70], 16, 1, 64, torch.int8, torch.float16)
    cache.value_scales[0, cache.pages_of(0)[0]] = 2.0 ** -30
    cache.value_scales[0, cache.pages_of(0)[1]] = 500.0
    q = torch.randn((1, 2, 64), generator=torch.Generator().manual_seed(3)).half().to(device)
    _check(cache, [70], [1], q)


@pytest.mark.parametrize("codes", CODES)
def test_streams_and_captured_replays(device, codes):
    """Store, read and attention in one graph, replayed with new inputs; another stream beside it."""
    heads, dim, size = 2, 128, 64
    cache = _filled(device, [3000, 130], size, heads, dim, codes, torch.bfloat16)
    slots, plan = cache.slots([0, 1], [2900, 30], [100, 100]), cache.plan([0, 1], [100, 100], heads=4)
    cos, sin, sections = oracle.tables(128, dim // 2)
    positions = rotary.TokenRows(rk.RopeTable(cos, sin, sections), (torch.arange(200)[:, None] % 100).expand(200, 3).int().contiguous().to(device))
    g = torch.Generator().manual_seed(2)
    k, v, q = (torch.randn((200, h, dim), generator=g).bfloat16().to(device) for h in (heads, heads, 4))

    def step():
        cache.store(0, slots, k, v, positions=positions)
        return (*cache.read(0, slots), cache.attend(0, q, plan))

    expected = step()
    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        other = step()
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, expected))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outs = step()
    for replay in range(3):
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(10 + replay)))
        graph.replay()
        torch.cuda.synchronize(device)
        found = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(found, step()))


def test_refusals_on_the_device(device):
    cache = _filled(device, [40], 16, 2, 64, torch.int8, torch.bfloat16)
    places = cache.places([0], [3], [20])
    with pytest.raises(ConfigurationError, match="places"):
        cache.store(0, places, *(torch.zeros(20, 2, 64, dtype=torch.bfloat16, device=device) for _ in range(2)))
    out = torch.empty(2, 20, 2, 64, dtype=torch.bfloat16, device=device)
    with pytest.raises(ConfigurationError, match="overlaps"):
        cache.read(0, places, out=(out[0], out[0]))
    with pytest.raises(ConfigurationError):
        cache.read(0, places, out=(out[0], out[1].float()))
    with pytest.raises(ConfigurationError, match="codes"):
        cache.plan([0], [1], heads=2)._check(cache.keys[0], cache.values[0])
    before = [t.clone() for t in cache.read(0, places)]
    assert all(torch.equal(a, b) for a, b in zip(cache.read(0, places, out=tuple(out)), before))


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("exponent", [-108, -104, -90, -60, 60, 110])
@pytest.mark.parametrize("group", [2, 33])
def test_small_weights_of_small_and_large_values(device, codes, exponent, group):
    """Values far from 1, and a key of value 0 that takes nearly all of the weight: what the others add is of their weights'
    precision, about 2^-17 of the largest, whatever their scales (group 2: the form of single tokens)."""
    dtype, dim, size, lengths = torch.bfloat16, 64, 16, [300, 70]
    cache = _empty(device, 30, size, 1, dim, codes, dtype)
    cache.load_tables([(list(range(19)), 300), ([25, 20, 28, 22, 21], 70)])
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn((sum(lengths), 1, dim), generator=g) for _ in range(2))
    v *= 2.0 ** exponent
    for at in (7, 300 + 40):
        k[at], v[at] = 12.0, 0.0
    cache.store(0, cache.slots([0, 1], [0, 0], lengths), *(x.to(dtype).to(device) for x in (k, v)))
    q = torch.full((2, group, dim), 0.125) + 0.01 * torch.randn((2, group, dim), generator=g)
    q = q.to(dtype).to(device)
    assert cache.plan([0], [1], heads=group)._single == (group == 2)
    out = _check(cache, lengths, [1, 1], q)
    assert (out != 0).any(dim=2).all()


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,size", [(144, 64), (256, 64), (256, 16)])
def test_long_split_histories_of_wide_heads(device, codes, dtype, dim, size):
    """Parts of few tiles, joined: heads above 128 channels are cut as the others are."""
    lengths = [9000, 70]
    cache = _filled(device, lengths, size, 2, dim, codes, dtype)
    q = torch.randn((2, 6, dim), generator=torch.Generator().manual_seed(3)).to(dtype).to(device)
    native = _native(cache)
    plan = cache.plan([0, 1], [1, 1], heads=6)
    assert plan._single and plan._n_merges == 4  # also of the two tiles of 70 keys
    out, lse = cache.attend(0, q, plan, return_lse=True)
    for sequence, length in enumerate(lengths):
        k, v = (history.history(x[0], "BTHD", cache.pages_of(sequence), length) for x in (native.keys, native.values))
        for head in range(6):
            want, bound, logs, log_bound = history.attend(q[sequence:sequence + 1, head].double().cpu(), k[:, head // 3], v[:, head // 3],
                                                          np.ones((1, length), dtype=bool), dtype)
            assert oracle.worst(out[sequence:sequence + 1, head], want, bound) <= 0
            assert oracle.worst(lse[sequence:sequence + 1, head], logs, log_bound) <= 0
