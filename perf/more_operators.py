"""The operators of long histories, as measurable cases: keys and values in 8 bits, and attention to chosen blocks.

A history that outgrows the memory for its pages is kept in 8-bit codes, and one that outgrows the time for its
attention is attended to where a cheap score finds it worth while.  ``kind`` names the call:

* ``store8`` -- ``QuantizedCache.store`` of new tokens (keys rotated, a scale for each token and head) and
  ``QuantizedCache.read`` of them, which returns the values that the codes stand for;
* ``read8`` -- ``QuantizedCache.read`` of whole histories;
* ``attend8`` -- ``QuantizedCache.attend``: new tokens (one, a chunk, or prompts) attend to 8-bit pages;
* ``index`` -- ``BlockIndex.update``: the mean key of each block that new tokens touched;
* ``sparse`` -- ``BlockIndex.select`` and ``BlockIndex.attend``: the blocks of each run of queries by the product of
  their sum with the blocks' mean keys, and the attention to those.

``run`` computes them in their plain form (blocks are scored in 64 bits, so that every order of the sums gives the same
choice), or with ``own`` by the framework's calls.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LEAST = 2.0 ** -126  # smallest scale

CACHE = {"heads": 12, "kv_heads": 12, "head_dim": 128, "page_tokens": 1560, "layout": "BTHD", "dtype": "bf16"}
STORE = {**CACHE, "kind": "store8", "batch": 1, "frames": 3, "height": 30, "width": 52, "history": 28080, "rope": True,
         "codes": "int8"}
READ = {**CACHE, "kind": "read8", "batch": 1, "longest": 32760, "shortest": 32760, "codes": "e4m3"}
ATTEND = {**CACHE, "kind": "attend8", "batch": 1, "queries": 4680, "shortest_query": 4680, "longest": 32760,
          "shortest": 32760, "block": 0, "window": 0, "codes": "e4m3"}
INDEX = {**CACHE, "kind": "index", "batch": 1, "new": 4680, "longest": 32760, "shortest": 32760, "block_tokens": 120,
         "codes": ""}
SPARSE = {**ATTEND, "kind": "sparse", "codes": "", "block_tokens": 120, "query_block": 120, "top": 24, "first": 1,
          "recent": 1}


def listed():
    return [
        # One token of 32 sequences into their 16-token pages: the smallest store.
        dict(STORE, name="store8_tokens", batch=32, frames=1, height=1, width=1, heads=8, kv_heads=8, page_tokens=16,
             history=4000, dtype="fp16"),
        # The clean keys and values of a CausVid chunk into pages of one latent frame.
        dict(STORE, name="store8_chunk"),
        # A seven-chunk history read back for a reader of native tensors.
        dict(READ, name="read8_history"),
        # Single tokens over short histories: the smallest attention call.
        dict(ATTEND, name="attend8_tokens_short", batch=8, queries=1, shortest_query=1, longest=1000, shortest=37,
             heads=32, kv_heads=8, page_tokens=16, codes="int8"),
        # Single tokens over long histories, four query heads to a key head.
        dict(ATTEND, name="attend8_tokens_long", batch=4, queries=1, shortest_query=1, longest=65536, shortest=20000,
             heads=32, kv_heads=8, page_tokens=64, codes="int8"),
        # A CausVid chunk over its seven-chunk history (itself the last).
        dict(ATTEND, name="attend8_chunk"),
        # Prompts and tokens together: odd lengths, causal, small pages, heads of 80 channels.
        dict(ATTEND, name="attend8_ragged", batch=6, queries=777, shortest_query=1, longest=5003, shortest=211,
             heads=20, kv_heads=5, head_dim=80, page_tokens=16, block=1, dtype="fp16", codes="int8"),
        # The blocks of a CausVid chunk after its store.
        dict(INDEX, name="index_chunk"),
        # The block of each of 32 sequences that its newest token touched.
        dict(INDEX, name="index_tokens", batch=32, new=1, heads=8, kv_heads=8, page_tokens=64, longest=4000, shortest=300,
             block_tokens=64),
        # Single tokens over long histories, of which each key head takes 31 blocks of 64.
        dict(SPARSE, name="sparse_tokens", batch=4, queries=1, shortest_query=1, longest=65536, shortest=20000, heads=32,
             kv_heads=8, page_tokens=64, block_tokens=64, query_block=1, top=28, recent=2),
        # A CausVid chunk over its history, a tenth of the blocks for every 120 queries.
        dict(SPARSE, name="sparse_chunk"),
        # Prompts over 8-bit pages, causal, with grouped heads.
        dict(SPARSE, name="sparse_prompts", batch=4, queries=1500, shortest_query=33, longest=12000, shortest=1700, heads=20,
             kv_heads=5, head_dim=80, page_tokens=64, block_tokens=32, query_block=32, top=30, recent=2, block=1,
             dtype="fp16", codes="int8"),
    ]


def _span(rng, low, high):
    """An integer of [low, high], even over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _drawn_queries(rng, case):
    """Tokens, a chunk or ragged prompts with their masks, at no more scores than the largest listed case has."""
    form = rng.choice(["token", "token", "chunk", "ragged"])
    if form == "token":
        case.update(batch=_span(rng, 1, 32), queries=1, shortest_query=1, longest=_span(rng, 64, 40000), block=0, window=0)
        case["shortest"] = _span(rng, 1, case["longest"])
    elif form == "chunk":
        queries = _span(rng, 200, 4680)
        case.update(batch=1, queries=queries, shortest_query=queries, block=rng.choice([0, 0, 1, -(-queries // 3)]),
                    window=rng.choice([0, 0, 0, _span(rng, 100, 20000)]))
        most = 4680 * 32760 * 12 * 128 // (queries * case["heads"] * case["head_dim"])
        case["longest"] = case["shortest"] = max(queries, min(queries + _span(rng, 1, 28000), most))
    else:
        case.update(batch=rng.randint(2, 8), queries=_span(rng, 20, 1500), longest=_span(rng, 1500, 12000),
                    block=rng.choice([0, 1, 1]), window=0)
        case.update(shortest_query=_span(rng, 1, case["queries"]), shortest=_span(rng, case["queries"], case["longest"]))
    return case


def draw(rng):
    kind = rng.choice(["store8", "read8", "attend8", "attend8", "attend8", "index", "sparse", "sparse", "sparse"])
    kv_heads = rng.choice([1, 2, 5, 8, 12])
    case = {"kv_heads": kv_heads, "heads": kv_heads * rng.choice([1, 1, 2, 4]), "head_dim": rng.choice([64, 80, 96, 128, 128]),
            "layout": rng.choice(["BTHD", "BTHD", "BHTD"]), "dtype": rng.choice(["bf16", "bf16", "fp16"]),
            "codes": rng.choice(["int8", "int8", "e4m3"]), "page_tokens": rng.choice([16, 64, 256, 390, 1560])}
    if kind == "store8":
        return dict(STORE, **case, batch=rng.randint(1, 4), frames=rng.randint(1, 3), height=_span(rng, 1, 30),
                    width=_span(rng, 1, 52), history=_span(rng, 1, 30000), rope=rng.random() < 0.7)
    if kind == "read8":
        case = dict(READ, **case, batch=rng.randint(1, 6), longest=_span(rng, 10, 32760))
        return dict(case, shortest=_span(rng, 1, case["longest"]))
    if kind == "attend8":
        return _drawn_queries(rng, dict(ATTEND, **case))
    if rng.random() < 0.7:
        case.update(codes="", dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    case["page_tokens"] = page = rng.choice([64, 128, 256, 390, 1560])
    case["block_tokens"] = rng.choice([n for n in (16, 32, 64, 65, 78, 120, 128, 156) if page % n == 0])
    if kind == "index":
        case = dict(INDEX, **case, batch=rng.randint(1, 8), new=_span(rng, 1, 4680))
        case["longest"] = case["new"] + _span(rng, 1, 20000)
        return dict(case, shortest=_span(rng, case["new"], case["longest"]))
    case = _drawn_queries(rng, dict(SPARSE, **case))
    case.update(query_block=1 if case["queries"] == 1 else rng.choice([16, 32, 64, 100, 128]), top=_span(rng, 1, 40),
                first=rng.randint(0, 2), recent=rng.randint(0, 3))
    if case["dtype"] == "fp32" and case["queries"] > 1:
        case["longest"] = min(case["longest"], max(case["queries"], 9000))
        case["shortest"] = min(case["shortest"], case["longest"])
    # The plain form gathers every run's blocks: at most 2 GB.
    case["top"] = max(1, min(case["top"], (1 << 29) // (case["batch"] * -(-case["queries"] // case["query_block"]) * case["kv_heads"]
                                                        * case["block_tokens"] * case["head_dim"]) - 8))
    return case


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------


def _tokens(case):
    return case["frames"] * case["height"] * case["width"]


def _spread(low, high, count):
    """``count`` integers from ``high`` down to ``low``, even over the logarithm."""
    if count == 1:
        return [high]
    return [round(high * (low / high) ** (i / (count - 1))) for i in range(count)]


def _lengths(case):
    """(queries, keys) of each sequence."""
    keys = _spread(case["shortest"], case["longest"], case["batch"])
    queries = [case["new"]] * case["batch"] if case["kind"] == "index" else _spread(case["shortest_query"], case["queries"], case["batch"])
    return queries, [max(a, b) for a, b in zip(queries, keys)]


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(shape, dtype, g):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32).to(dtype)


def _angles(rows, rotated):
    """Wan-like tables in 64 bits: a third of the pairs (rounded down) for rows and columns each, the rest for
    frames; ``[rows, pairs]`` cosines, sines and the three pair counts."""
    pairs = rotated // 2
    spatial = pairs // 3
    sections = (pairs - 2 * spatial, spatial, spatial)
    frequencies = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64) / n) for n in sections if n])
    angles = torch.arange(rows, dtype=torch.float64)[:, None] * frequencies[None]
    return angles.cos().to(DEVICE), angles.sin().to(DEVICE), sections


def _grid_rows(case, first):
    """int32 [T, 3]: (frame, row, column) of each token of a chunk that begins at frame ``first``."""
    axes = torch.meshgrid(torch.arange(case["frames"]) + first, torch.arange(case["height"]), torch.arange(case["width"]),
                          indexing="ij")
    return torch.stack([axis.reshape(-1) for axis in axes], dim=1).to(torch.int32).to(DEVICE)


def _scattered(page_counts, seed):
    """Pages of each sequence, without order."""
    order = np.random.default_rng(seed).permutation(sum(page_counts)).tolist()
    cuts = np.cumsum([0, *page_counts])
    return [order[a:b] for a, b in zip(cuts[:-1], cuts[1:])]


def _table(tables):
    """int32 [sequences, most pages] on the device; -1 behind a sequence's last page."""
    width = max(len(t) for t in tables)
    return torch.tensor([t + [-1] * (width - len(t)) for t in tables], dtype=torch.int32, device=DEVICE)


def _encode(x, codes):
    """(codes, fp32 scales) of fp32 rows ``x[..., channels]``."""
    most = x.abs().amax(dim=-1)
    if codes == "int8":
        scale = (most / torch.full_like(most, 127.0)).clamp(min=LEAST)
        code = (x * (torch.ones_like(scale) / scale)[..., None]).round().clamp(-127, 127)
    else:
        mantissa, exponent = torch.frexp(most)
        exponent = torch.where(most > 0, exponent - 9 + (mantissa > 0.875), -126).clamp(min=-126)
        scale = torch.ldexp(torch.ones_like(most), exponent)
        code = torch.ldexp(x, -exponent[..., None])
    return code.to(CODES[codes]), scale


def _decode(code, scale, dtype):
    """The values that codes stand for, of the cache's type."""
    return (code.float() * scale[..., None]).to(dtype)


def _pool(case, pages, g):
    """fp32 ``[pages, page_tokens, heads, channels]`` with channels of several sizes, neighbours alike."""
    shape = (pages, case["page_tokens"], case["kv_heads"], case["head_dim"])
    x = torch.randn(shape, generator=g, device=DEVICE)
    x += torch.randn((pages, -(-shape[1] // 32), *shape[2:]), generator=g, device=DEVICE).repeat_interleave(32, dim=1)[:, :shape[1]]
    return x.mul_(0.4 + 0.8 * torch.rand(shape[3], generator=g, device=DEVICE))


def _pools(case, pages, g, state):
    """The K and V pools of one layer, native or in codes with their scales ``[pages, heads, page_tokens]``."""
    for name in ("keys", "values"):
        x = _pool(case, pages, g).to(DTYPES[case["dtype"]])
        if case["codes"]:
            x, scale = _encode(x.float(), case["codes"])
            state[name + "_scale"] = scale.transpose(1, 2).contiguous()
        state[name] = x.transpose(1, 2).contiguous() if case["layout"] == "BHTD" else x


def _cache(case, state, tables, lengths):
    """The framework's cache over a state's pools."""
    from reelcache_amd import paged_cache, quantized_cache

    pools = [state["keys"][None], state["values"][None]]
    if case["codes"]:
        cache = quantized_cache.QuantizedCache(*pools, state["keys_scale"][None], state["values_scale"][None],
                                               dtype=DTYPES[case["dtype"]], layout=case["layout"])
    else:
        cache = paged_cache.PagedCache(*pools, layout=case["layout"])
    cache.load_tables(list(zip(tables, lengths)))
    return cache


def _prepare_store(case, seed):
    g, dtype, new, size, history = _generator(seed), DTYPES[case["dtype"]], _tokens(case), case["page_tokens"], case["history"]
    counts = [-(-(history + new) // size)] * case["batch"]
    tables = _scattered(counts, seed)
    shape = (case["batch"] * new, case["kv_heads"], case["head_dim"])
    state = {"case": case, "k": _normal(shape, dtype, g), "v": _normal(shape, dtype, g), "table": _table(tables)}
    _pools(case, sum(counts), g, state)
    state["cos"], state["sin"], state["sections"] = _angles(64, case["head_dim"])
    state["rows"] = _grid_rows(case, seed % 18).repeat(case["batch"], 1)
    state["at"] = torch.arange(history, history + new, device=DEVICE)
    if own:
        from reelcache_amd import restore_kernels, rotary

        cache = state["cache"] = _cache(case, state, tables, [history + new] * case["batch"])
        state["slots"] = cache.slots(list(range(case["batch"])), [history] * case["batch"], [new] * case["batch"])
        if case["rope"]:
            table = restore_kernels.RopeTable(state["cos"], state["sin"], state["sections"])
            state["positions"] = rotary.TokenRows(table, state["rows"])
    return state


def _row_places(lengths):
    """[tokens] sequence and place of each token of histories one behind the other."""
    sequence = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths))
    place = torch.cat([torch.arange(n) for n in lengths])
    return sequence.to(DEVICE), place.to(DEVICE)


def _prepare_read(case, seed):
    g, size = _generator(seed), case["page_tokens"]
    lengths = _spread(case["shortest"], case["longest"], case["batch"])
    counts = [-(-n // size) for n in lengths]
    tables = _scattered(counts, seed)
    state = {"case": case, "table": _table(tables)}
    _pools(case, sum(counts), g, state)
    state["sequence"], state["place"] = _row_places(lengths)
    if own:
        cache = state["cache"] = _cache(case, state, tables, lengths)
        state["places"] = cache.places(list(range(case["batch"])), [0] * case["batch"], lengths)
    return state


def _prepare_index(case, seed):
    g, size = _generator(seed), case["page_tokens"]
    new, lengths = _lengths(case)
    counts = [-(-n // size) for n in lengths]
    tables = _scattered(counts, seed)
    state = {"case": case, "table": _table(tables)}
    _pools(case, sum(counts), g, state)
    shape = (sum(counts), size // case["block_tokens"], case["kv_heads"], case["head_dim"])
    state["means"] = _normal(shape, DTYPES[case["dtype"]], g)
    # The blocks of the pool that the new tokens lie in.
    touched = [table[at // size] * shape[1] + at % size // case["block_tokens"]
               for table, n, length in zip(tables, new, lengths)
               for at in range((length - n) // case["block_tokens"] * case["block_tokens"], length, case["block_tokens"])]
    state["touched"] = torch.tensor(touched, device=DEVICE)
    if own:
        from reelcache_amd import sparse_attention

        cache = state["cache"] = _cache(case, state, tables, lengths)
        state["index"] = sparse_attention.BlockIndex(cache, state["means"][None])
        state["slots"] = cache.slots(list(range(case["batch"])), [a - b for a, b in zip(lengths, new)], new)
    return state


def _runs(case):
    """int64 [runs, 8]: sequence, first query, queries, blocks [first, last) that any query of the run sees, blocks [first,
    last) that are full and that every query sees whole, and the block of the last query (-1: before the first key)."""
    rows, size = [], case["block_tokens"]
    for sequence, (n, length) in enumerate(zip(*_lengths(case))):
        begin = np.arange(0, n, case["query_block"], dtype=np.int64)
        end = np.minimum(begin + case["query_block"], n)
        seen = [_visible(case, length, length - n + i) for i in (begin, end - 1)]
        low, high = seen[0][0], np.maximum(seen[1][1], seen[0][0])
        inner_low, inner_high = seen[1][0], seen[0][1]
        some = high > low
        first, last = np.where(some, low // size, 0), np.where(some, -(-high // size), 0)
        rows.append(np.stack([np.full_like(begin, sequence), begin, end - begin, first, last, -(-inner_low // size),
                              inner_high // size, (length - n + end - 1) // size], axis=1))
    return np.concatenate(rows)


def _taken(case, runs):
    """(always, scored): truth values [runs, blocks] of the blocks that a run takes in any case, and that it scores."""
    block = np.arange(-(-case["longest"] // case["block_tokens"]))[None]
    first, last, low, high, at = (runs[:, i, None] for i in range(3, 8))
    seen = (block >= first) & (block < last)
    scored = seen & (block >= low) & (block < high) & (block >= case["first"])
    scored &= (block > at) | (block <= at - case["recent"])
    return seen & ~scored, scored


def _prepare_attend(case, seed):
    g, dtype, size = _generator(seed), DTYPES[case["dtype"]], case["page_tokens"]
    queries, keys = _lengths(case)
    counts = [-(-n // size) for n in keys]
    tables = _scattered(counts, seed)
    state = {"case": case, "q": _normal((sum(queries), case["heads"], case["head_dim"]), dtype, g), "table": _table(tables)}
    _pools(case, sum(counts), g, state)
    most = max(queries)
    starts = np.cumsum([0, *queries[:-1]])
    state["queries"], state["lengths"] = torch.tensor(queries, device=DEVICE), torch.tensor(keys, device=DEVICE)
    if case["kind"] == "attend8":
        places = np.arange(most)[None] + starts[:, None]
        state["places"] = torch.from_numpy(np.where(np.arange(most)[None] < np.array(queries)[:, None], places, -1)).to(DEVICE)
    else:
        runs = _runs(case)
        always, scored = _taken(case, runs)
        state["always"], state["scored"] = torch.from_numpy(always).to(DEVICE), torch.from_numpy(scored).to(DEVICE)
        state["width"] = int((always.sum(1) + np.minimum(case["top"], scored.sum(1))).max())
        at = np.arange(case["query_block"])[None]
        places = np.where(at < runs[:, 2:3], starts[runs[:, 0]][:, None] + runs[:, 1:2] + at, -1)
        state["places"] = torch.from_numpy(places).to(DEVICE)  # rows of q of each run, -1 behind its last
        state["sequence"], state["first"] = torch.from_numpy(runs[:, 0].copy()).to(DEVICE), torch.from_numpy(runs[:, 1].copy()).to(DEVICE)
        pool = _native(state, "keys").double()
        state["means"] = pool.unflatten(1, (-1, case["block_tokens"])).mean(dim=2).to(dtype)
    if own:
        cache = state["cache"] = _cache(case, state, tables, keys)
        masks = {"block": case["block"] or None, "window": case["window"] or None}
        if case["kind"] == "attend8":
            state["plan"] = cache.plan(list(range(case["batch"])), queries, heads=case["heads"], **masks)
        else:
            from reelcache_amd import sparse_attention

            state["index"] = sparse_attention.BlockIndex(cache, state["means"][None])
            state["plan"] = state["index"].plan(list(range(case["batch"])), queries, heads=case["heads"], top=case["top"],
                                                query_block=case["query_block"], first=case["first"], recent=case["recent"],
                                                **masks)
    return state


def prepare(case, seed):
    if case["kind"] == "store8":
        return _prepare_store(case, seed)
    if case["kind"] == "read8":
        return _prepare_read(case, seed)
    if case["kind"] == "index":
        return _prepare_index(case, seed)
    return _prepare_attend(case, seed)


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------


def _token_rows(x, case):
    """A pool as ``[pages, page_tokens, heads, ...]``."""
    return x.transpose(1, 2) if case["layout"] == "BHTD" else x


def _native(state, name):
    """A pool's values ``[pages, page_tokens, heads, channels]``, of the cache's type."""
    case = state["case"]
    pool = _token_rows(state[name], case)
    return _decode(pool, state[name + "_scale"].transpose(1, 2), DTYPES[case["dtype"]]) if case["codes"] else pool


def _rows_read(state, name, page, row):
    """The values of the rows (page, row) of a pool in codes: ``[rows, heads, channels]``."""
    case = state["case"]
    return _decode(_token_rows(state[name], case)[page, row], state[name + "_scale"].transpose(1, 2)[page, row],
                   DTYPES[case["dtype"]])


def _rotated(x, cos, sin):
    """fp32 ``x[..., D]`` with its interleaved pairs rotated."""
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)


def _run_store(state):
    case = state["case"]
    if own:
        cache, slots = state["cache"], state["slots"]
        cache.store(0, slots, state["k"], state["v"], positions=state.get("positions"))
        return cache.read(0, slots)
    k, v = state["k"].float(), state["v"].float()
    if case["rope"]:
        column = torch.arange(state["cos"].shape[1], device=DEVICE)
        t, h, _ = state["sections"]
        at = state["rows"].long()[:, (column >= t).long() + (column >= t + h).long()]  # each pair's table row
        k = _rotated(k, state["cos"][at, column].float()[:, None], state["sin"][at, column].float()[:, None])
    page, row = state["at"] // case["page_tokens"], (state["at"] % case["page_tokens"]).repeat(case["batch"])
    page = state["table"].long()[:, page].reshape(-1)
    for name, x in (("keys", k), ("values", v)):
        code, scale = _encode(x, case["codes"])
        # (8-bit floats are moved as bytes: not every torch indexes them)
        _token_rows(state[name], case).view(torch.uint8)[page, row] = code.view(torch.uint8)
        state[name + "_scale"].transpose(1, 2)[page, row] = scale
    return tuple(_rows_read(state, name, page, row) for name in ("keys", "values"))


def _run_read(state):
    if own:
        return state["cache"].read(0, state["places"])
    size = state["case"]["page_tokens"]
    page, row = state["table"].long()[state["sequence"], state["place"] // size], state["place"] % size
    return tuple(_rows_read(state, name, page, row) for name in ("keys", "values"))


def _run_index(state):
    case = state["case"]
    if own:
        state["index"].update(0, state["slots"])
        return state["means"]
    rows = state["touched"][:, None] * case["block_tokens"] + torch.arange(case["block_tokens"], device=DEVICE)
    page, row = rows // case["page_tokens"], rows % case["page_tokens"]
    keys = _token_rows(state["keys"], case)[page, row]
    if case["codes"]:
        keys = _decode(keys, state["keys_scale"].transpose(1, 2)[page, row], DTYPES[case["dtype"]])
    state["means"].flatten(0, 1)[state["touched"]] = keys.double().mean(dim=1).to(state["means"].dtype)
    return state["means"]


def _hidden(case, place, key, length):
    """Whether a query at ``place`` does not see ``key`` (both broadcast)."""
    hidden = (key >= length) | (key < 0) | torch.zeros_like(place, dtype=torch.bool)
    if case["block"]:
        hidden = hidden | (key >= (place // case["block"] + 1) * case["block"])
    if case["window"]:
        hidden = hidden | (key <= place - case["window"])
    return hidden


def _attention(q, keys, values, hidden):
    """fp32 attention ``[..., rows, D]`` over ``[..., keys, D]``; rows that see nothing give zeros."""
    scores = torch.matmul(q * q.shape[-1] ** -0.5, keys.transpose(-1, -2).contiguous())
    scores.masked_fill_(hidden, -math.inf)
    scores.sub_(scores.amax(dim=-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = scores.sum(dim=-1, keepdim=True)
    return torch.matmul(scores, values.contiguous()) / total.masked_fill(total == 0, 1.0)


def _run_attend(state):
    case, q = state["case"], state["q"]
    if own:
        return state["cache"].attend(0, q, state["plan"])
    heads, kv_heads, dim, longest = case["heads"], case["kv_heads"], case["head_dim"], case["longest"]
    table, places = state["table"].long().clamp(min=0), state["places"]
    batch, most = places.shape
    # [sequence, key head, token, channel] in fp32; behind a sequence's pages: page 0, which the mask hides.
    keys, values = (_native(state, name)[table].reshape(batch, -1, kv_heads, dim)[:, :longest].permute(0, 2, 1, 3).float()
                    for name in ("keys", "values"))
    grouped = q[places.clamp(min=0)].float().reshape(batch, most, kv_heads, heads // kv_heads, dim)
    grouped = grouped.permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, -1, dim)
    place = (state["lengths"] - state["queries"])[:, None] + torch.arange(most, device=DEVICE)  # of each query
    hidden = _hidden(case, place[..., None], torch.arange(keys.shape[2], device=DEVICE), state["lengths"][:, None, None])
    hidden = hidden[:, None, None].expand(-1, 1, heads // kv_heads, -1, -1).reshape(batch, 1, -1, keys.shape[2])
    out = _attention(grouped, keys, values, hidden).reshape(batch, kv_heads, heads // kv_heads, most, dim)
    return out.permute(0, 3, 1, 2, 4).reshape(batch, most, heads, dim)[places >= 0].to(q.dtype)


def _run_select(state):
    """int32 [runs, key heads, width]: the blocks of each run in ascending order, -1 behind the last."""
    case, places = state["case"], state["places"]
    group, size, per_page = case["heads"] // case["kv_heads"], case["block_tokens"], case["page_tokens"] // case["block_tokens"]
    pooled = torch.where((places >= 0)[..., None, None], state["q"][places.clamp(min=0)].double(), 0.0).sum(dim=1)
    pooled = pooled.unflatten(1, (-1, group)).sum(dim=2)  # [runs, key heads, channels]
    block = torch.arange(state["scored"].shape[1], device=DEVICE)
    page = state["table"].long()[:, (block * size // case["page_tokens"]).clamp(max=state["table"].shape[1] - 1)].clamp(min=0)
    means = state["means"][page, block % per_page].double().permute(0, 2, 3, 1).contiguous()  # [sequences, heads, channels, blocks]
    scores = torch.matmul(pooled[:, :, None], means[state["sequence"]].contiguous())[:, :, 0]
    scored = state["scored"][:, None]
    order = torch.where(scored, scores, -math.inf).sort(dim=-1, descending=True, stable=True)[1]
    rank = torch.empty_like(order).scatter_(-1, order, block.expand_as(order).contiguous())
    taken = (scored & (rank < case["top"])) | state["always"][:, None]
    found = torch.where(taken, block, block.numel()).sort(dim=-1)[0][..., :state["width"]]
    return torch.where(found == block.numel(), -1, found).to(torch.int32)


def _run_sparse(state):
    case, q = state["case"], state["q"]
    if own:
        blocks = state["index"].select(0, q, state["plan"])
        return blocks, state["index"].attend(0, q, state["plan"], blocks=blocks)
    blocks, places = _run_select(state), state["places"]
    heads, kv_heads, dim, size = case["heads"], case["kv_heads"], case["head_dim"], case["page_tokens"]
    runs, most = places.shape
    key = blocks.long()[..., None] * case["block_tokens"] + torch.arange(case["block_tokens"], device=DEVICE)
    key = torch.where(blocks[..., None] < 0, -1, key).flatten(2)  # [runs, key heads, keys]
    at = key.clamp(min=0).minimum(state["lengths"][state["sequence"]][:, None, None] - 1)
    page = state["table"].long()[state["sequence"][:, None, None], at // size]
    head = torch.arange(kv_heads, device=DEVICE)[:, None]
    found = []
    for name in ("keys", "values"):
        rows = _token_rows(state[name], case)[page, at % size, head]
        if case["codes"]:
            rows = _decode(rows, state[name + "_scale"][page, head, at % size], DTYPES[case["dtype"]])
        found.append(rows.float())
    grouped = q[places.clamp(min=0)].float().reshape(runs, most, kv_heads, heads // kv_heads, dim)
    grouped = grouped.permute(0, 2, 3, 1, 4).reshape(runs, kv_heads, -1, dim)
    place = (state["lengths"] - state["queries"])[state["sequence"]] + state["first"]
    place = place[:, None] + torch.arange(most, device=DEVICE)
    hidden = _hidden(case, place[:, None, :, None], key[:, :, None], state["lengths"][state["sequence"]][:, None, None, None])
    hidden = hidden[:, :, None].expand(-1, -1, heads // kv_heads, -1, -1).reshape(runs, kv_heads, -1, key.shape[2])
    out = _attention(grouped, *found, hidden).reshape(runs, kv_heads, heads // kv_heads, most, dim)
    return blocks, out.permute(0, 3, 1, 2, 4).reshape(runs, most, heads, dim)[places >= 0].to(q.dtype)


def run(state):
    kind = state["case"]["kind"]
    if kind == "store8":
        return _run_store(state)
    if kind == "read8":
        return _run_read(state)
    if kind == "index":
        return _run_index(state)
    return _run_attend(state) if kind == "attend8" else _run_sparse(state)


# ---------------------------------------------------------------------------------------------
# Bytes and operations, and values in 64 bits
# ---------------------------------------------------------------------------------------------


def _visible(case, length, place):
    """Keys [first, last) that the queries at ``place`` (an array) see of a sequence."""
    last = np.full_like(place, length)
    if case["block"]:
        last = np.minimum(last, np.maximum(place // case["block"] + 1, 0) * case["block"])
    first = np.clip(place - case["window"] + 1, 0, length) if case["window"] else np.zeros_like(place)
    return first, last


def work(case):
    size, dim, kind = SIZES[case["dtype"]], case["head_dim"], case["kind"]
    row = dim + 4 if case["codes"] else dim * size  # bytes of a head's row in the cache
    if kind == "store8":
        rows = 2 * case["batch"] * _tokens(case) * case["kv_heads"]
        # Read, written as codes, read again, returned as values.
        return {"bytes": rows * (2 * dim * size + 2 * row) + case["batch"] * _tokens(case) * 16, "flops": rows * 4 * dim}
    if kind == "read8":
        rows = 2 * sum(_spread(case["shortest"], case["longest"], case["batch"])) * case["kv_heads"]
        return {"bytes": rows * (row + dim * size), "flops": rows * dim}
    queries, keys = _lengths(case)
    if kind == "index":
        blocks = sum(-(-a // case["block_tokens"]) - (a - b) // case["block_tokens"] for a, b in zip(keys, queries))
        rows = blocks * case["kv_heads"]
        return {"bytes": rows * (case["block_tokens"] * row + dim * size), "flops": rows * case["block_tokens"] * dim}
    rows = 2 * sum(queries) * case["heads"]
    if kind == "attend8":
        pairs = reach = 0
        for n, length in zip(queries, keys):
            first, last = _visible(case, length, np.arange(length - n, length, dtype=np.int64))
            pairs += int(np.maximum(last - first, 0).sum())
            reach += max(0, int(last.max() - first.min()))
        return {"bytes": rows * dim * size + 2 * reach * case["kv_heads"] * row, "flops": 4 * pairs * case["heads"] * dim}
    runs = _runs(case)
    always, scored = _taken(case, runs)
    taken = always.sum(1) + np.minimum(case["top"], scored.sum(1))
    # Means and taken blocks are read at least once for a sequence and head; a run's queries see a taken block in half or
    # whole, which counts as whole.
    sequence = runs[:, 0]
    means = sum(int(scored[sequence == s].any(axis=0).sum()) for s in range(case["batch"]))
    fetched = sum(min(int(taken[sequence == s].sum()), -(-keys[s] // case["block_tokens"])) for s in range(case["batch"]))
    scores = int(scored.sum()) * case["kv_heads"]
    return {"bytes": rows * dim * size + means * case["kv_heads"] * dim * size
            + 2 * fetched * case["kv_heads"] * case["block_tokens"] * row,
            "flops": 4 * int((taken * runs[:, 2]).sum()) * case["block_tokens"] * case["heads"] * dim + 2 * scores * dim}


def _values(state, name):
    """A pool's values in 64 bits ``[pages, page_tokens, heads, channels]``: codes times scales, rounded to the type."""
    case, pool = state["case"], state[name].float().double()
    if case["codes"]:
        scale = state[name + "_scale"].double()
        pool = pool * (scale if case["layout"] == "BHTD" else scale.permute(0, 2, 1))[..., None]
        pool = pool.to(DTYPES[case["dtype"]]).double()
    return pool.permute(0, 2, 1, 3) if case["layout"] == "BHTD" else pool


def _history(state, values, sequence, length):
    pages = state["table"][sequence, :-(-length // state["case"]["page_tokens"])].long()
    return values[pages].flatten(0, 1)[:length]


def _stood_for(x, codes):
    """What rows of 64-bit values are read back as."""
    most = x.abs().amax(dim=-1, keepdim=True)
    if codes == "int8":
        step = (most / 127).clamp(min=LEAST)
        return torch.round(x / step) * step
    unit = torch.exp2(torch.ceil(torch.log2(most / 448)).clamp(min=-126))
    y = x / unit
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * unit


def _exact_store(case, state):
    k, v = state["k"].double(), state["v"].double()
    if case["rope"]:
        t, h, _ = state["sections"]
        turn, at = torch.complex(state["cos"], state["sin"]), state["rows"].long()
        turn = torch.cat([turn[at[:, 0], :t], turn[at[:, 1], t:t + h], turn[at[:, 2], t + h:]], dim=-1)[:, None]
        k = torch.view_as_real(torch.view_as_complex(k.unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)
    return _stood_for(k, case["codes"]), _stood_for(v, case["codes"])


def _exact_heads(q, keys, values, seen):
    """Attention in 64 bits of ``q[n, D]`` over ``[m, D]`` under a mask."""
    scores = torch.where(seen, q @ keys.T / math.sqrt(q.shape[1]), -math.inf)
    return torch.nan_to_num(torch.softmax(scores, dim=1), nan=0.0) @ values


def _exact_attend(case, state):
    queries, lengths = _lengths(case)
    out, group = torch.empty(state["q"].shape, dtype=torch.float64, device=DEVICE), case["heads"] // case["kv_heads"]
    keys, values = _values(state, "keys"), _values(state, "values")
    start = 0
    for sequence, (n, length) in enumerate(zip(queries, lengths)):
        k, v = _history(state, keys, sequence, length), _history(state, values, sequence, length)
        first, last = (torch.from_numpy(x).to(DEVICE) for x in _visible(case, length, np.arange(length - n, length)))
        key = torch.arange(length, device=DEVICE)
        seen = (key >= first[:, None]) & (key < last[:, None])
        for head in range(case["heads"]):
            out[start:start + n, head] = _exact_heads(state["q"][start:start + n, head].double(), k[:, head // group],
                                                      v[:, head // group], seen)
        start += n
    return out


def _exact_sparse(case, state):
    queries, lengths = _lengths(case)
    starts, group, size = np.cumsum([0, *queries[:-1]]), case["heads"] // case["kv_heads"], case["block_tokens"]
    out = torch.empty(state["q"].shape, dtype=torch.float64, device=DEVICE)
    keys, values = _values(state, "keys"), _values(state, "values")
    per_page, means = case["page_tokens"] // size, state["means"].double().flatten(0, 1)
    runs = _runs(case)
    if len(runs) * case["kv_heads"] > 4000:
        return None
    always, scored = _taken(case, runs)
    for run_, forced, choice in zip(runs, always, scored):
        sequence, begin, n = (int(x) for x in run_[:3])
        length = lengths[sequence]
        at = int(starts[sequence]) + begin
        place = length - queries[sequence] + begin + np.arange(n)
        first, last = (torch.from_numpy(x).to(DEVICE) for x in _visible(case, length, place))
        k, v = _history(state, keys, sequence, length), _history(state, values, sequence, length)
        candidates = torch.from_numpy(np.flatnonzero(choice)).to(DEVICE)
        mean = means[state["table"][sequence].long()[candidates // per_page] * per_page + candidates % per_page]
        for head in range(case["kv_heads"]):
            q = state["q"][at:at + n, head * group:(head + 1) * group].double()
            score = (mean[:, head] * q.sum(dim=(0, 1))).sum(dim=1)
            best = candidates[torch.argsort(score, descending=True, stable=True)[:case["top"]]]
            blocks = torch.cat([best, torch.from_numpy(np.flatnonzero(forced)).to(DEVICE)])
            key = (blocks[:, None] * size + torch.arange(size, device=DEVICE)).flatten()
            key = key[key < length]
            seen = (key >= first[:, None]) & (key < last[:, None])
            for member in range(group):
                out[at:at + n, head * group + member] = _exact_heads(q[:, member], k[key, head], v[key, head], seen)
    return None, out


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "store8":
        return _exact_store(case, state)
    if case["kind"] == "read8":
        lengths = _spread(case["shortest"], case["longest"], case["batch"])
        return tuple(torch.cat([_history(state, _values(state, name), s, n) for s, n in enumerate(lengths)])
                     for name in ("keys", "values"))
    if case["kind"] == "index":
        means, sums = state["means"].double(), _values(state, "keys").unflatten(1, (-1, case["block_tokens"])).sum(dim=2)
        means.flatten(0, 1)[state["touched"]] = sums.flatten(0, 1)[state["touched"]] / case["block_tokens"]
        return means
    return _exact_attend(case, state) if case["kind"] == "attend8" else _exact_sparse(case, state)
