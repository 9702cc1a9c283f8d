"""``attention.attend`` on the GPU against its plain form in 64 bits."""

import math

import numpy as np
import pytest
import torch

from reelcache_amd import attention, paged_cache, rotary
from reelcache_amd import restore_kernels as rk
from reelcache_amd.errors import ConfigurationError, StateError

import operator_oracle as oracle

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _cache(device, lengths, size, heads, dim, dtype, layout="BTHD", layers=1, seed=0, spare=2):
    """A cache with scattered pages; every row that no sequence has is NaN."""
    counts = [-(-n // size) for n in lengths]
    pages = sum(counts) + spare
    g = torch.Generator().manual_seed(seed)
    rows = (size, heads) if layout == "BTHD" else (heads, size)
    pools = [torch.randn((layers, pages, *rows, dim), generator=g).to(dtype).to(device) for _ in range(2)]
    order = np.random.default_rng(seed).permutation(pages).tolist()
    cuts = np.cumsum([0, *counts])
    tables = [order[a:b] for a, b in zip(cuts[:-1], cuts[1:])]
    cache = paged_cache.PagedCache(*pools, layout=layout)
    cache.load_tables(list(zip(tables, lengths)))
    for pool in pools:
        pool = pool if layout == "BTHD" else pool.transpose(2, 3)
        for page in order[cuts[-1]:]:
            pool[:, page] = math.nan
        for table, n in zip(tables, lengths):
            if n % size:
                pool[:, table[-1], n % size:] = math.nan
    return cache


def _check(cache, q, out, lse, lengths, queries, layer=0, **mask):
    start = 0
    for sequence, (length, n) in enumerate(zip(lengths, queries)):
        rows = slice(start, start + n)
        want, bound, logs, log_bound = oracle.attend(q[rows], cache.keys[layer], cache.values[layer],
                                                     cache.pages_of(sequence), length, n, cache.page_tokens,
                                                     layout=cache.layout, **mask)
        assert oracle.worst(out[rows], want, bound) <= 0, (sequence, length, n)
        if lse is not None:
            assert oracle.worst(lse[rows], logs, log_bound) <= 0, (sequence, length, n)
        start += n


def _run(device, lengths, queries, size, kv_heads, group, dim, dtype, layout="BTHD", seed=0, **mask):
    cache = _cache(device, lengths, size, kv_heads, dim, dtype, layout, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn((sum(queries), kv_heads * group, dim), generator=g).to(dtype).to(device)
    plan = cache.plan(list(range(len(lengths))), queries, heads=kv_heads * group, **mask)
    out, lse = cache.attend(0, q, plan, return_lse=True)
    _check(cache, q, out, lse, lengths, queries, **mask)
    assert torch.equal(out, cache.attend(0, q, plan))  # and the same bits again
    return cache, q, plan, out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size,kv_heads,group,dim,layout", [
    (16, 2, 1, 64, "BTHD"), (64, 1, 4, 128, "BTHD"), (100, 2, 2, 80, "BHTD"), (7, 1, 3, 96, "BTHD"), (130, 3, 1, 128, "BHTD"),
    (16, 1, 2, 20, "BTHD"), (9, 2, 1, 200, "BTHD"), (16, 1, 1, 7, "BHTD"), (64, 1, 1, 8, "BTHD"), (33, 1, 2, 104, "BTHD"),
])
def test_single_tokens(device, dtype, size, kv_heads, group, dim, layout):
    """One token of sequences of one token to several tiles of keys."""
    lengths = [1, 2, 31, 64, 65, 129, 300]
    _run(device, lengths, [1] * len(lengths), size, kv_heads, group, dim, dtype, layout)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block", [None, 1, 40])
@pytest.mark.parametrize("size,kv_heads,group,dim,layout", [
    (16, 1, 1, 64, "BTHD"), (64, 1, 2, 128, "BTHD"), (100, 1, 1, 80, "BHTD"), (7, 1, 1, 128, "BTHD"), (16, 1, 1, 20, "BTHD"),
    (150, 1, 1, 96, "BTHD"),
])
def test_chunks(device, dtype, block, size, kv_heads, group, dim, layout):
    """Chunks alone, behind a history, and beside single tokens."""
    _run(device, [70, 133, 260, 90, 40], [70, 129, 75, 1, 33], size, kv_heads, group, dim, dtype, layout, block=block)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [128, 64, 20])
def test_windows(device, dtype, dim):
    for window, block in ((1, 1), (63, 1), (50, None), (130, 16), (1 << 30, None)):
        _run(device, [300, 20, 77], [140, 20, 1], 16, 1, 1, dim, dtype, window=window, block=block)
    _run(device, [300, 20, 77], [140, 20, 1], 96, 1, 1, dim, dtype, window=33, block=1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,size", [(128, 16), (128, 64), (64, 70), (20, 16)])
def test_rows_that_see_nothing(device, dtype, dim, size):
    """More queries than tokens under a causal mask, and an empty history: zeros and -inf."""
    for lengths, queries in (([5, 0, 130], [9, 3, 140]), ([0], [1]), ([0, 3], [40, 50])):
        cache, q, plan, out = _run(device, lengths, queries, size, 1, 2, dim, dtype, block=1)
        assert not out[:max(0, queries[0] - lengths[0])].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,size", [(128, 16), (64, 64), (128, 100), (20, 8)])
def test_dropped_pages(device, dtype, dim, size):
    """Pages that were dropped are not seen, whatever they hold now; a query may see only such pages."""
    lengths, queries = [8 * size + 3, 3 * size], [size + 3, 1]
    cache = _cache(device, lengths, size, 1, dim, dtype)
    dropped = cache.pages_of(0)[2:5] + cache.pages_of(1)[:2]
    cache.drop(0, 2, 3)
    cache.drop(1, 0, 2)
    for pool in (cache.keys, cache.values):
        pool[:, dropped] = math.inf
    q = torch.randn((sum(queries), 2, dim), generator=torch.Generator().manual_seed(3)).to(dtype).to(device)
    for mask in ({}, {"block": 1}, {"window": size}):
        plan = cache.plan([0, 1], queries, heads=2, **mask)
        out, lse = cache.attend(0, q, plan, return_lse=True)
        _check(cache, q, out, lse, lengths, queries, **mask)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,size", [(128, 16), (64, 64), (96, 150), (20, 8)])
def test_hidden_rows_may_hold_anything(device, dtype, dim, size):
    """Infinities and NaN in keys and values of tokens that a causal mask hides from earlier queries: those
    queries are exact, the later ones get what arithmetic gives."""
    lengths, queries = [210, 20], [150, 20]
    cache = _cache(device, lengths, size, 1, dim, dtype)
    q = torch.randn((170, 1, dim), generator=torch.Generator().manual_seed(3)).to(dtype).to(device)
    bad = 150  # place of the first bad token of sequence 0; its query is row 90
    pages = cache.pages_of(0)
    plain = cache.values[0].clone(), cache.keys[0].clone()
    for at, value, which in ((bad, math.nan, "values"), (bad + 3, math.inf, "values"), (bad + 40, math.nan, "keys"),
                             (bad + 41, -math.inf, "keys")):
        getattr(cache, which)[0, pages[at // size], at % size, 0, at % dim] = value
    plan = cache.plan([0, 1], queries, heads=1, block=1)
    out = cache.attend(0, q, plan)
    want, bound, _, _ = oracle.attend(q[:90], plain[1], plain[0], pages, 210, 150, size, block=1)
    assert oracle.worst(out[:90], want[:90], bound[:90]) <= 0
    assert out[90:93, 0, bad % dim].isnan().all() and out[131:150].isnan().any(dim=2).all()
    other = torch.arange(dim, device=device) != bad % dim
    assert out[90:93, 0, other].isfinite().all() and (out[93:130, 0, (bad + 3) % dim] == math.inf).all()
    want, bound, _, _ = oracle.attend(q[150:], cache.keys[0], cache.values[0], cache.pages_of(1), 20, 20, size, block=1)
    assert oracle.worst(out[150:], want, bound) <= 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_and_sharp_scores(device, dtype):
    """Scores far apart (one key takes all), all equal, and growing along the keys, so that the running
    reference moves in every tile."""
    size, dim, n = 64, 64, 700
    cache = _cache(device, [n], size, 1, dim, dtype)
    pages = torch.tensor(cache.pages_of(0), device=device)
    ramp = torch.linspace(-1, 1, len(pages) * size, device=device).view(-1, size)
    q = torch.ones((200, 1, dim), device=device).to(dtype)
    for scale in (1.0, 20.0):
        cache.keys[0, pages, :, 0] = (ramp[..., None] * 3).expand(-1, -1, dim).to(dtype)
        for queries in (200, 1):
            for block in (None, 1):
                plan = cache.plan([0], [queries], heads=1, block=block, scale=scale)
                out, lse = cache.attend(0, q[:queries], plan, return_lse=True)
                _check(cache, q[:queries], out, lse, [n], [queries], block=block, scale=scale)
    cache.keys[0, pages] = 0
    plan = cache.plan([0], [200], heads=1)
    _check(cache, q, *cache.attend(0, q, plan, return_lse=True), [n], [200])


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_histories_split(device, dtype):
    """Keys split over many workgroups: single tokens and a short chunk over a long history."""
    _run(device, [9000, 5, 4100], [1, 1, 1], 64, 1, 2, 128, dtype)
    _run(device, [6000], [40], 16, 1, 1, 64, dtype, block=1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [128, 72, 20, 200])
@pytest.mark.parametrize("lengths,rows,least", [([20000], 8, 64), ([20000, 9000], 16, 9), ([2500] * 10, 80, 9)])
def test_rows_of_many_parts(device, dtype, dim, lengths, rows, least):
    """Few rows in very many parts, and more rows in several, of every head size."""
    _, _, plan, _ = _run(device, lengths, [1] * len(lengths), 64, 1, 8, dim, dtype)
    merges = plan.buffer[plan._merges:plan._merges + 8 * plan._n_merges].view(-1, 8)
    assert merges[:, 2].sum() == rows and merges[:, 5].max() >= least


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [128, 72, 256, 136])
def test_chunks_in_several_parts(device, dtype, dim):
    """Whole blocks of rows in two to eight parts, beside single tokens in more."""
    _, _, plan, _ = _run(device, [620, 2400], [250, 1], 64, 4, 1, dim, dtype, block=50)
    merges = plan.buffer[plan._merges:plan._merges + 8 * plan._n_merges].view(-1, 8)
    assert plan._n_many < plan._n_merges and merges[:, 2].max() == 128 and merges[plan._n_many:, 5].max() <= 8


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block", [None, 1])
@pytest.mark.parametrize("size,kv_heads,group,dim,layout", [
    (64, 1, 1, 256, "BTHD"), (16, 2, 2, 192, "BHTD"), (7, 1, 1, 136, "BTHD"), (100, 1, 3, 200, "BTHD"), (9, 1, 1, 248, "BTHD"),
    (16, 1, 1, 252, "BTHD"), (64, 1, 2, 250, "BTHD"),
])
def test_wide_heads(device, dtype, block, size, kv_heads, group, dim, layout):
    """Heads of more than 128 channels: single tokens, chunks, and histories in several parts."""
    _run(device, [70, 133, 260, 90, 1500, 1], [70, 129, 75, 1, 33, 1], size, kv_heads, group, dim, dtype, layout, block=block)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,size", [(256, 16), (192, 64), (160, 100)])
def test_hidden_rows_of_wide_heads_may_hold_anything(device, dtype, dim, size):
    """Infinite and NaN values behind a mask, in a dropped page and behind the last token."""
    lengths, queries = [5 * size + 3], [2 * size]
    cache = _cache(device, lengths, size, 1, dim, dtype)
    pages = cache.pages_of(0)
    q = torch.randn((2 * size, 2, dim), generator=torch.Generator().manual_seed(3)).to(dtype).to(device)
    cache.drop(0, 1, 1)
    for pool in (cache.keys, cache.values):
        pool[:, pages[1]] = math.inf
        pool[:, pages[5], 1] = -math.inf  # a token that only the last rows see under the causal mask
        pool[:, pages[5], 2] = math.nan   # and one that only the last row sees
    plan = cache.plan([0], queries, heads=2, block=1)
    out = cache.attend(0, q, plan)
    want, bound, _, _ = oracle.attend(q[:-2], cache.keys[0], cache.values[0], cache.pages_of(0), lengths[0] - 2,
                                      queries[0] - 2, size, block=1)
    assert oracle.worst(out[:-2], want, bound) <= 0
    assert torch.isnan(out[-1]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [128, 20])
def test_strides_outputs_and_rows_behind(device, dtype, dim):
    lengths, queries = [90, 33], [60, 1]
    cache = _cache(device, lengths, 16, 2, dim, dtype, layers=2)
    plan = cache.plan([0, 1], queries, heads=4)
    wide = torch.randn((70, 5, 2 * dim), generator=torch.Generator().manual_seed(2)).to(dtype).to(device)
    q = wide[:, 1:, dim:]  # strided, with rows behind the plan's
    out, lse = cache.attend(1, q, plan, return_lse=True)
    assert out.shape == q.shape and not out[61:].any() and (lse[61:] == -math.inf).all()
    _check(cache, q, out, lse, lengths, queries, layer=1)
    spread = wide[..., ::2][:, 1:, :]
    _check(cache, spread, cache.attend(1, spread, plan), None, lengths, queries, layer=1)
    for target in (torch.full((70, 4, dim), 7.0, dtype=dtype, device=device),
                   torch.full((70, 6, dim + 8), 7.0, dtype=dtype, device=device)[:, 1:5, 8:],
                   torch.full((70, 4, dim + 1), 7.0, dtype=dtype, device=device)[:, :, 1:],
                   torch.full((70, 4, dim, 2), 7.0, dtype=dtype, device=device)[..., 1]):
        assert cache.attend(1, q, plan, out=target) is target
        assert torch.equal(target[:61], out[:61]) and (target[61:] == 7).all()
    same = q.contiguous()
    assert cache.attend(1, same, plan, out=same) is same and torch.equal(same[:61], out[:61])
    odd = torch.empty(70 * 4 * dim + 1, dtype=dtype, device=device)[1:].view(70, 4, dim).copy_(q)
    assert torch.equal(cache.attend(1, odd, plan), out)


def test_pools_with_gaps_and_native_caches(device):
    """Pools whose rows have room between them, unaligned pools (general form), and a native cache tensor
    as a pool of one page that ends inside a tile."""
    g = torch.Generator().manual_seed(0)
    wide = [torch.randn((1, 6, 16, 3, 72), generator=g).bfloat16().to(device) for _ in range(2)]
    q = torch.randn((40, 4, 64), generator=g).bfloat16().to(device)
    for cut in (8, 3):
        cache = paged_cache.PagedCache(*(p[:, :, :, 1:, cut:cut + 64] for p in wide))
        cache.load_tables([([4, 0, 5], 45)])
        plan = cache.plan([0], [40], heads=4, block=1)
        _check(cache, q, cache.attend(0, q, plan), None, [45], [40], block=1)
    for layout, shape in (("BTHD", (1, 275, 2, 64)), ("BHTD", (1, 2, 275, 64))):
        native = [torch.randn(shape, generator=g).bfloat16().to(device) for _ in range(2)]
        cache = paged_cache.PagedCache(*(p[None] for p in native), layout=layout)
        cache.load_tables([([0], 270)])
        plan = cache.plan([0], [40], heads=4)
        _check(cache, q, cache.attend(0, q, plan), None, [270], [40])


def test_parts_of_a_history_join_by_their_sums(device):
    """Results over two caches joined by the returned logarithms equal attention over both."""
    dim, n = 64, 150
    cache = _cache(device, [n], 10, 1, dim, torch.float32)
    q = torch.randn((50, 1, dim), generator=torch.Generator().manual_seed(2)).to(device)
    pages = cache.pages_of(0)
    whole, logs = cache.attend(0, q, cache.plan([0], [50], heads=1), return_lse=True)
    parts = []
    for part in (pages[:7], pages[7:]):
        half = paged_cache.PagedCache(cache.keys, cache.values)
        half.load_tables([(part, 10 * len(part))])
        parts.append(half.attend(0, q, half.plan([0], [50], heads=1), return_lse=True))
    (a, la), (b, lb) = [(o.double(), x.double()) for o, x in parts]
    total = torch.logaddexp(la, lb)
    joined = a * (la - total).exp()[..., None] + b * (lb - total).exp()[..., None]
    _, bound, _, log_bound = oracle.attend(q, cache.keys[0], cache.values[0], pages, n, 50, 10)
    assert oracle.worst(whole, joined.cpu(), 4 * bound) <= 0 and oracle.worst(logs, total.cpu(), 4 * log_bound) <= 0


def test_refusals(device):
    cache = _cache(device, [20, 9], 8, 2, 64, torch.bfloat16)
    plan = cache.plan([0, 1], [4, 1], heads=4)
    q = torch.zeros((5, 4, 64), dtype=torch.bfloat16, device=device)
    for bad in (q[:4], q[:, :2], q[..., :32], q.float(), q.cpu(), q[0]):
        with pytest.raises(ConfigurationError):
            cache.attend(0, bad, plan)
    for out in (q.float(), torch.zeros((6, 4, 64), dtype=torch.bfloat16, device=device), q[:, :1].expand(5, 4, 64)):
        with pytest.raises(ConfigurationError):
            cache.attend(0, q, plan, out=out)
    long = torch.zeros((6, 4, 64), dtype=torch.bfloat16, device=device)
    with pytest.raises(ConfigurationError, match="overlap"):
        cache.attend(0, long[:5], plan, out=long[1:])
    with pytest.raises(ConfigurationError):
        attention.attend(q, cache.keys[0], cache.values[0], None)
    with pytest.raises(ConfigurationError):
        cache.attend(1, q, plan)
    assert cache.attend(0, q[:0], cache.plan([], [], heads=4)).shape == (0, 4, 64)
    cache.free(1)
    with pytest.raises(StateError):
        cache.attend(0, q, plan)


def test_streams_and_captured_replays(device):
    """Two captured calls that share a plan, replayed in turn with eager work between, and a call on
    another stream."""
    cache = _cache(device, [3000, 130], 64, 2, 128, torch.bfloat16, layers=2)
    cache.keys.nan_to_num_(0.0), cache.values.nan_to_num_(0.0)
    plan = cache.plan([0, 1], [1, 100], heads=4)
    q = torch.randn((101, 4, 128), generator=torch.Generator().manual_seed(2)).bfloat16().to(device)
    expected = cache.attend(0, q, plan)
    stream = torch.cuda.Stream(device)
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        other = cache.attend(0, q, plan)
    stream.synchronize()
    assert torch.equal(other, expected)
    graphs, outs = [], []
    for layer in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(cache.attend(layer, q, plan))
        graphs.append(graph)
    for replay in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(10 + replay)))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize(device)
        for layer in range(2):
            assert torch.equal(outs[layer], cache.attend(layer, q, plan))
    first, second = torch.cuda.Stream(device), torch.cuda.Stream(device)
    torch.cuda.synchronize(device)
    for graph, side in zip(graphs, (first, second)):  # both at once
        with torch.cuda.stream(side):
            graph.replay()
    torch.cuda.synchronize(device)
    for layer in range(2):
        assert torch.equal(outs[layer], cache.attend(layer, q, plan))


def test_a_step_of_two_layers(device):
    """The operators as an engine uses them: history restored into pages, the new chunk's queries and keys
    rotated, keys and values stored, attention, then a fork that goes on alone."""
    grid, heads, dim, size = (1, 6, 7), 2, 64, 16
    n = 42
    cos, sin, sections = oracle.tables(32, dim // 2)
    table = rk.RopeTable(cos, sin, sections)
    cache = paged_cache.PagedCache(*(torch.zeros(2, 16, size, heads, dim, dtype=torch.bfloat16, device=device) for _ in range(2)))
    g = torch.Generator().manual_seed(0)
    raw = [[torch.randn((3 * n, heads, dim), generator=g).bfloat16().to(device) for _ in range(2)] for _ in range(2)]
    a = cache.new()
    cache.extend([a], [n])
    for layer, (k, v) in enumerate(raw):
        jobs = [rk.ReconstructionJob(rk.DenseSource(x[:n].reshape(n, -1)), cache.view(layer, target, a, 0, n), grid, rope=rope)
                for x, target, rope in zip((k, v), "kv", (rk.RopePositions(table, 0), None))]
        rk.reconstruct(jobs).release()
    b = None
    for chunk in (1, 2):
        sequence = a if chunk == 1 else b
        slots, positions = cache.extend([sequence], [n]), rk.RopePositions(table, chunk)
        plan = cache.plan([sequence], [n], heads=2 * heads)
        rows = slice(chunk * n, (chunk + 1) * n)
        for layer, (k, v) in enumerate(raw):
            q = torch.randn((n, 2 * heads, dim), generator=g).bfloat16().to(device)
            turned = rotary.rotate(q, positions, grid=grid, layout="THD")
            cache.store(layer, slots, k[rows], v[rows], positions=positions, grid=grid)
            out = cache.attend(layer, turned, plan)
            places = torch.cat([oracle.grid_rows((i, 0, 0), grid) for i in range(chunk + 1)])
            angles = oracle.token_angles(cos, sin, sections, places)
            keys = oracle.rotate(k[:rows.stop], *(x[:, None] for x in angles))[0].bfloat16()
            want, bound, _, _ = oracle.attend(turned, keys[None], v[None, :rows.stop], [0], rows.stop, n, rows.stop)
            # The stored keys may round the other way where the plain rotation lies at a border: one step of
            # each key, through the score (both keys of a pair of scores) into the weights.
            shift = 2 * dim ** -0.5 * 2 * oracle.U[torch.bfloat16] * float((keys.abs().amax(0).float().amax(0) * turned.cpu().abs().float().amax((0, 1))).sum())
            assert oracle.worst(out, want, bound + shift * float(v.abs().max())) <= 0
        if chunk == 1:
            b = cache.fork(a)
    assert cache.pages_of(a)[:5] == cache.pages_of(b)[:5] and cache.pages_of(a)[5] != cache.pages_of(b)[5]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [54, 60, 63])
@pytest.mark.parametrize("layout", ["BTHD", "BHTD"])
def test_pages_just_below_a_tile(device, dtype, size, layout):
    """Single tokens, chunks and a dropped page in pages of a few tokens less than a tile."""
    _run(device, [1, size, size + 1, 300], [1, 1, 1, 1], size, 2, 2, 64, dtype, layout)
    _run(device, [133, 260, 40], [129, 75, 33], size, 1, 2, 128, dtype, layout, block=1)
    lengths, queries = [5 * size + 3], [size]
    cache = _cache(device, lengths, size, 1, 64, dtype, layout)
    dropped = cache.pages_of(0)[2]
    cache.drop(0, 2, 1)
    for pool in (cache.keys, cache.values):
        pool[:, dropped] = math.inf
    q = torch.randn((size, 2, 64), generator=torch.Generator().manual_seed(3)).to(dtype).to(device)
    plan = cache.plan([0], queries, heads=2, block=1)
    _check(cache, q, *cache.attend(0, q, plan, return_lse=True), lengths, queries, block=1)


FAR = [(128, 64, 700, 150), (64, 16, 300, 1), (96, 100, 400, 33), (200, 64, 300, 40), (20, 16, 200, 3), (128, 64, 9000, 2)]


def _uniform_keys(cache, n, numbers, dtype, device):
    """Keys that hold one number in all their channels; the values of the tokens, float64 on the CPU."""
    place = torch.arange(n)
    pages, rows = torch.tensor(cache.pages_of(0))[place // cache.page_tokens].to(device), (place % cache.page_tokens).to(device)
    cache.keys[0, pages, rows, 0] = numbers[:, None].expand(-1, cache.head_dim).to(dtype).to(device)
    return cache.values[0, pages, rows, 0].double().cpu()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,size,n,queries", FAR)
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_far_out(device, dtype, dim, size, n, queries, sign):
    """Scores of 10^8 and more: the keys that share the largest one share the row; the others, more than 10^6 below it,
    have no weight, whether they come before or after."""
    cache = _cache(device, [n], size, 1, dim, dtype)
    q = torch.full((queries, 2, dim), 8192.0, device=device).to(dtype)
    generator = torch.Generator().manual_seed(5)
    for largest in (4096.0, 8192.0, 32768.0):
        # Steps of a sixteenth, which every type holds: the products and their sums are exact in fp32 too.
        numbers = sign * largest * (1 - sign * torch.randint(1, 8, (n,), generator=generator).double() / 16)
        top = torch.randint(0, n, (3,), generator=generator).unique()
        numbers[top] = sign * largest
        seen = _uniform_keys(cache, n, numbers, dtype, device)[top]
        for scale in (dim ** -0.5, 1.0):
            out, lse = cache.attend(0, q, cache.plan([0], [queries], heads=2, scale=scale), return_lse=True)
            # One weight for all of them: rounded to the type alike (its sum is not), summed and divided in fp32.
            want, size_of = seen.mean(0), seen.abs().mean(0)
            bound = 1.01 * size_of * (oracle.U[dtype] + 8 * oracle.F32) + 1.01 * oracle.U[dtype] * want.abs() + oracle.TINY[dtype]
            assert oracle.worst(out, want.expand(queries, 2, dim), bound.expand(queries, 2, dim)) <= 0, (largest, scale)
            # The scale with log2 e, the product and the way back round once each.
            logs = torch.full((queries, 2), sign * largest * dim * 8192.0 * scale + math.log(len(top)), dtype=torch.float64)
            assert oracle.worst(lse, logs, 8 * oracle.F32 * (1 + logs.abs())) <= 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,size,n,queries", FAR)
@pytest.mark.parametrize("first", [False, True])
def test_scores_far_below_others(device, dtype, dim, size, n, queries, first):
    """Scores of -10^8 and less beside ordinary ones, before or behind them: only those have weights."""
    cache = _cache(device, [n], size, 1, dim, dtype)
    q = torch.full((queries, 2, dim), 8192.0, device=device).to(dtype)
    kept = torch.arange(20) if first else torch.arange(n - 20, n)
    numbers = torch.full((n,), -8192.0, dtype=torch.float64)
    numbers[kept] = torch.linspace(-2.0 ** -14, 2.0 ** -14, 20, dtype=torch.float64)
    values = _uniform_keys(cache, n, numbers, dtype, device)
    out, lse = cache.attend(0, q, cache.plan([0], [queries], heads=2), return_lse=True)
    score = numbers[kept].to(dtype).double() * dim * 8192.0 * dim ** -0.5
    weight, seen = torch.softmax(score, 0), values[kept]
    # Each score: dim products and sums, the scaling, the shift by the largest; then the exponential and the sums.
    off = (dim + 8) * oracle.F32 * float(score.abs().max()) + 4 * oracle.F32
    bound = 1.01 * (weight @ seen.abs()) * (oracle.U[dtype] + 2 * off + 64 * oracle.F32) + 1.01 * oracle.U[dtype] * (weight @ seen).abs() + oracle.TINY[dtype]
    if dtype == torch.float16:
        bound = bound + seen.abs().sum(0) * 2.0 ** -31
    assert oracle.worst(out, (weight @ seen).expand(queries, 2, dim), bound.expand(queries, 2, dim)) <= 0
    logs = torch.full((queries, 2), float(torch.logsumexp(score, 0)), dtype=torch.float64)
    assert oracle.worst(lse, logs, 1.01 * off + 64 * oracle.F32 * (1 + logs.abs())) <= 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,size", [(128, 16), (64, 64), (96, 100), (200, 64), (20, 8)])
@pytest.mark.parametrize("parts", ["one", "few", "many"])
def test_scores_of_minus_infinity(device, dtype, dim, size, parts):
    """A query all of whose scores are -inf has no softmax (NaN, and a log of -inf); one that sees nothing has zeros, and
    one that sees a single finite score has that key's value."""
    n, queries = {"one": (90, 100), "few": (2400, 2500), "many": (20000, 3)}[parts]
    block = 1 if parts != "many" else None
    cache = _cache(device, [n, 2 * size, 5], size, 1, dim, dtype)
    cache.keys[..., 0] = -math.inf  # of every token, those behind the sequences too
    lone = cache.pages_of(1)[1], size - 1  # the last key of sequence 1
    cache.keys[0, lone[0], lone[1], 0] = 0.5
    q = torch.rand((queries + 3, 2, dim), generator=torch.Generator().manual_seed(1)).add_(0.5).to(dtype).to(device)
    counts = [queries, 2, 1]
    out, lse = cache.attend(0, q, cache.plan([0, 1, 2], counts, heads=2, block=block), return_lse=True)
    hidden = max(0, queries - n) if block else 0
    assert not out[:hidden].any() and out[hidden:queries].isnan().all() and (lse[:queries] == -math.inf).all()
    value = cache.values[0, lone[0], lone[1], 0].double().cpu()
    bound = (oracle.U[dtype] * 2.02 + 8 * oracle.F32) * value.abs() + oracle.TINY[dtype] + (2.0 ** -31 if dtype == torch.float16 else 0.0)
    sighted = slice(queries + 1, queries + 2) if block else slice(queries, queries + 2)
    assert oracle.worst(out[sighted], value.expand_as(out[sighted]), bound.expand_as(out[sighted])) <= 0
    if block:
        assert out[queries].isnan().all()
    assert out[queries + 2].isnan().all() and lse[queries + 2].tolist() == [-math.inf] * 2
    # Behind dropped pages: nothing is seen at all, or only what is left.
    cache.drop(1, 0, 1)
    out, lse = cache.attend(0, q[:1], cache.plan([1], [1], heads=2, window=size + 1), return_lse=True)
    assert oracle.worst(out, value.expand_as(out), bound.expand_as(out)) <= 0
    cache.keys[0, lone[0], lone[1], 0] = -math.inf
    out = cache.attend(0, q[:2], cache.plan([1], [2], heads=2))
    assert out.isnan().all()
    out, lse = cache.attend(0, q[:size + 2], cache.plan([1], [size + 2], heads=2, block=1), return_lse=True) if queries > size else (None, None)
    if out is not None:  # the first two stand in the dropped page
        assert not out[:2].any() and out[2:].isnan().all() and (lse == -math.inf).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,group", [(7, 1), (33, 3), (129, 1)])
def test_odd_heads_in_odd_parts(device, dtype, dim, group):
    """Partial rows of an odd number of words, and an odd number of them."""
    for n in (3000, 3200, 3400):
        _, _, plan, _ = _run(device, [n], [1], 16, 1, group, dim, dtype)
        assert plan._n_merges


@pytest.mark.parametrize("layout", ["BTHD", "BHTD"])
@pytest.mark.parametrize("dim,size", [(128, 256), (100, 250)])
def test_pools_past_32_bits(device, layout, dim, size):
    """Pages that lie more than 2^32 elements into their pools: copies, stores and attention, tiled and general."""
    heads, dtype = 8, torch.bfloat16
    pages = (1 << 32) // (size * heads * dim) + 40
    cache = paged_cache.PagedCache.allocate(pages, size, heads, dim, device=device, layout=layout)
    assert (pages - 40) * cache.keys.stride(1) * 2 > 1 << 32
    last = list(range(pages - 12, pages - 4))
    for pool in (cache.keys, cache.values):
        assert pool[0, last[0]].data_ptr() - pool.data_ptr() > 1 << 33
    n = 6 * size + 41
    cache.load_tables([(last[:7], n - 30), ([*range(pages - 13)], (pages - 13) * size)])  # the lower pages are taken
    generator = torch.Generator(device).manual_seed(1)
    for pool in (cache.keys, cache.values):
        pool[0, pages - 13:] = torch.randn(pool[0, pages - 13:].shape, generator=generator, device=device).to(dtype)
    child = cache.fork(0)
    slots = cache.extend([child], [30])  # copies the begun page
    assert cache.pages_of(child)[-1] != last[6] and min(cache.pages_of(child)) > pages - 14
    k, v = (torch.randn((30, heads, dim), generator=generator, device=device).to(dtype) for _ in range(2))
    cache.store(0, slots, k, v)
    tokens = [torch.cat([(pool[0, page] if layout == "BTHD" else pool[0, page].transpose(0, 1)) for page in cache.pages_of(child)])[:n]
              for pool in (cache.keys, cache.values)]
    assert torch.equal(tokens[0][-30:], k) and torch.equal(tokens[1][-30:], v)
    begun = (n - 30) % size
    for pool in (cache.keys, cache.values):
        old, new = (pool[0, page] if layout == "BTHD" else pool[0, page].transpose(0, 1) for page in (last[6], cache.pages_of(child)[6]))
        assert torch.equal(old[:begun], new[:begun])
    q = torch.randn((30, heads, dim), generator=generator, device=device).to(dtype)
    out, lse = cache.attend(0, q, cache.plan([child], [30], heads=heads, block=1), return_lse=True)
    want, bound, logs, log_bound = oracle.attend(q, tokens[0][None], tokens[1][None], [0], n, 30, n, block=1)
    assert oracle.worst(out, want, bound) <= 0 and oracle.worst(lse, logs, log_bound) <= 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,size", [(128, 16), (64, 64), (200, 100), (20, 16)])
@pytest.mark.parametrize("level", [8192.0, -8192.0])
def test_scores_far_out_under_masks(device, dtype, dim, size, level):
    """Equal scores of +-10^9 weigh as equal scores of 0 do, whatever a row sees of them: under masks, with a dropped
    page, beside rows that see nothing, in one part and in several, and beside a sequence of ordinary scores."""
    lengths, queries = [5 * size + 3, 70, 4000], [2 * size, 90, 3]
    cache = _cache(device, lengths, size, 1, dim, dtype)
    cache.drop(0, 1, 1)
    q = torch.full((sum(queries), 2, dim), 8192.0, device=device).to(dtype)
    q[2 * size:2 * size + 90] = torch.randn((90, 2, dim), generator=torch.Generator().manual_seed(1)).to(dtype).to(device)
    ordinary = cache.keys[0, cache.pages_of(1)].clone()
    for mask in ({}, {"block": 1}, {"block": 7, "window": 3 * size // 2}):
        cache.keys.fill_(level)
        cache.keys[0, cache.pages_of(1)] = ordinary
        out = cache.attend(0, q, cache.plan([0, 1, 2], queries, heads=2, **mask))
        cache.keys.fill_(0.0)
        cache.keys[0, cache.pages_of(1)] = ordinary
        _check(cache, q, out, None, lengths, queries, **mask)
