"""The operators around an attention cache, as measurable cases.

A restored history is of use once an engine attends to it.  A case names one of the calls that an
engine makes of a cache on the way there; ``kind`` says which:

* ``rotate`` -- ``rotary.rotate`` of queries and keys by positions of several axes (frame, row, column),
  and with ``grad`` the gradients of both;
* ``store`` -- ``PagedCache.store``: the keys of new tokens rotated and written with their values into
  the slots of their pages;
* ``fork`` -- ``PagedCache.fork`` and ``extend``: sequences that share a history go on apart, so the
  pages they have begun are copied in every layer;
* ``compact`` -- ``PagedCache.compact``: pages in use move down to the lowest ones;
* ``attend`` -- ``attention.attend``: new tokens (one, or a chunk) attend to their sequence's pages.

``run`` computes them in their plain form in 32 bits, or with ``own`` by the framework's calls.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}

ROTATE = {"kind": "rotate", "batch": 1, "frames": 3, "height": 30, "width": 52, "heads": 12, "kv_heads": 12,
          "head_dim": 128, "rotated": 128, "layout": "BTHD", "pairing": "interleaved", "positions": "grid",
          "grad": False, "dtype": "bf16"}
STORE = {"kind": "store", "batch": 1, "frames": 3, "height": 30, "width": 52, "heads": 12, "head_dim": 128,
         "page_tokens": 1560, "history": 28080, "rope": True, "dtype": "bf16"}
PAGES = {"layers": 30, "heads": 12, "head_dim": 128, "page_tokens": 256, "pages": 40, "dtype": "bf16"}
ATTEND = {"kind": "attend", "batch": 1, "queries": 4680, "shortest_query": 4680, "longest": 32760, "shortest": 32760,
          "heads": 12, "kv_heads": 12, "head_dim": 128, "page_tokens": 1560, "layout": "BTHD", "block": 0,
          "window": 0, "dtype": "bf16"}


def listed():
    return [
        # Queries and keys of one token of sixteen sequences, each at a place of its own.
        dict(ROTATE, name="rotate_tokens", batch=16, frames=1, height=1, width=1, heads=32, kv_heads=8,
             positions="tokens"),
        # A CausVid chunk of three latent frames, on the grid the restore rotates by.
        dict(ROTATE, name="rotate_chunk"),
        # A training step over LongCat-shaped heads, [B, H, T, D]: rotation and both gradients.
        dict(ROTATE, name="rotate_train", batch=2, heads=32, kv_heads=32, layout="BHTD", pairing="half",
             positions="tokens", grad=True, dtype="fp32"),
        # One token of 32 sequences into their 16-token pages.
        dict(STORE, name="store_tokens", batch=32, frames=1, height=1, width=1, heads=8, page_tokens=16, history=4000,
             dtype="fp16"),
        # The clean keys and values of a CausVid chunk into pages of one latent frame.
        dict(STORE, name="store_chunk"),
        # Eight continuations of one history, each with a page of its own begun in 30 layers.
        dict(PAGES, name="fork_history", kind="fork", forks=8, tokens=2400, added=100),
        # A cache of 30 layers after sequences ended: the rest moves down.
        dict(PAGES, name="compact_layers", kind="compact", moved=12),
        # Single tokens over short histories: the smallest attention call.
        dict(ATTEND, name="attend_token_short", batch=8, queries=1, shortest_query=1, longest=1000, shortest=37,
             heads=32, kv_heads=8, page_tokens=16),
        # Single tokens over long histories, four query heads to a key head.
        dict(ATTEND, name="attend_token_long", batch=4, queries=1, shortest_query=1, longest=65536, shortest=20000,
             heads=32, kv_heads=8, page_tokens=64),
        # A CausVid chunk over its seven-chunk history (itself the last), pages of one latent frame.
        dict(ATTEND, name="attend_chunk"),
        # A LongCat-shaped chunk over eight chunks, pages of [H, T, D].
        dict(ATTEND, name="attend_wide_chunk", heads=32, kv_heads=32, longest=37440, shortest=37440, layout="BHTD"),
        # Prompts and tokens together: odd lengths, causal, small pages, heads of 80 channels.
        dict(ATTEND, name="attend_ragged", batch=6, queries=777, shortest_query=1, longest=5003, shortest=211,
             heads=20, kv_heads=5, head_dim=80, page_tokens=16, block=1, dtype="fp16"),
    ]


def _span(rng, low, high):
    """An integer of [low, high], even over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["rotate", "rotate", "store", "fork", "compact", "attend", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    head_dim = rng.choice([64, 80, 96, 128, 128])
    if kind == "rotate":
        kv_heads = rng.choice([2, 5, 8, 12])
        return dict(ROTATE, batch=rng.randint(1, 4), frames=rng.randint(1, 4), height=_span(rng, 1, 30),
                    width=_span(rng, 1, 52), heads=kv_heads * rng.choice([1, 1, 2, 4]), kv_heads=kv_heads,
                    head_dim=head_dim, rotated=rng.choice([head_dim, head_dim, head_dim // 2]),
                    layout=rng.choice(["BTHD", "BHTD"]), pairing=rng.choice(["interleaved", "half"]),
                    positions=rng.choice(["grid", "tokens"]), grad=rng.random() < 0.4, dtype=dtype)
    if kind == "store":
        return dict(STORE, batch=rng.randint(1, 4), frames=rng.randint(1, 3), height=_span(rng, 1, 30),
                    width=_span(rng, 1, 52), heads=_span(rng, 1, 32), head_dim=head_dim,
                    page_tokens=rng.choice([16, 64, 256, 390, 1560]), history=_span(rng, 1, 30000),
                    rope=rng.random() < 0.7, dtype=dtype)
    if kind == "fork":
        page_tokens = rng.choice([16, 64, 100, 256])
        pages = rng.randint(24, 48)
        return dict(PAGES, kind="fork", layers=rng.randint(1, 30), heads=_span(rng, 2, 16), head_dim=head_dim,
                    page_tokens=page_tokens, pages=pages, forks=rng.randint(1, 8),
                    tokens=rng.randint(1, (pages - 16) * page_tokens), added=rng.randint(1, page_tokens), dtype=dtype)
    if kind == "compact":
        pages = rng.randint(24, 48)
        return dict(PAGES, kind="compact", layers=rng.randint(1, 30), heads=_span(rng, 2, 16), head_dim=head_dim,
                    page_tokens=rng.choice([16, 64, 100, 256]), pages=pages, moved=rng.randint(1, pages // 3), dtype=dtype)
    kv_heads = rng.choice([1, 2, 5, 8, 12])
    case = dict(ATTEND, kv_heads=kv_heads, heads=kv_heads * rng.choice([1, 1, 2, 4]), head_dim=head_dim,
                page_tokens=rng.choice([16, 64, 256, 390, 1560]), layout=rng.choice(["BTHD", "BTHD", "BHTD"]), dtype=dtype)
    form = rng.choice(["token", "token", "chunk", "ragged"])
    if form == "token":
        case.update(batch=_span(rng, 1, 32), queries=1, shortest_query=1, longest=_span(rng, 64, 40000))
        case["shortest"] = _span(rng, 1, case["longest"])
    elif form == "chunk":
        queries = _span(rng, 200, 4680)
        case.update(queries=queries, shortest_query=queries, longest=queries + _span(rng, 1, 28000))
        case["shortest"] = case["longest"]
        case["block"] = rng.choice([0, 0, 1, -(-queries // 3)])
        case["window"] = rng.choice([0, 0, 0, _span(rng, 100, 20000)])
    else:
        case.update(batch=rng.randint(2, 8), queries=_span(rng, 20, 1500), longest=_span(rng, 1500, 12000),
                    block=rng.choice([0, 1, 1]))
        case.update(shortest_query=_span(rng, 1, case["queries"]), shortest=_span(rng, case["queries"], case["longest"]))
    if form == "chunk":  # no more scores than the largest listed case has
        case["longest"] = case["shortest"] = max(queries, min(case["longest"], 4680 * 37440 * 32 // (queries * case["heads"])))
    if dtype == "fp32" and form != "token":
        case["longest"] = min(case["longest"], max(case["queries"], 9000))
        case["shortest"] = min(case["shortest"], case["longest"])
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
    """(queries, keys) of each sequence of an attention case."""
    queries = _spread(case["shortest_query"], case["queries"], case["batch"])
    keys = _spread(case["shortest"], case["longest"], case["batch"])
    return queries, [max(a, b) for a, b in zip(queries, keys)]


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(shape, dtype, g, scale=1.0):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32).mul_(scale).to(dtype)


def _angles(rows, rotated):
    """Wan-like tables in 64 bits: a third of the pairs (rounded down) for rows and columns each, the
    rest for frames; ``[rows, pairs]`` cosines, sines and the three pair counts."""
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


def _shape(case, heads):
    tokens = _tokens(case)
    return ((case["batch"], tokens, heads, case["head_dim"]) if case["layout"] == "BTHD"
            else (case["batch"], heads, tokens, case["head_dim"]))


def _pool_shape(case, pages):
    rows = (case["page_tokens"], case["kv_heads"] if "kv_heads" in case else case["heads"])
    return (pages, *(rows if case.get("layout", "BTHD") == "BTHD" else rows[::-1]), case["head_dim"])


def _prepare_rotate(case, seed):
    g, dtype = _generator(seed), DTYPES[case["dtype"]]
    state = {"case": case, "q": _normal(_shape(case, case["heads"]), dtype, g),
             "k": _normal(_shape(case, case["kv_heads"]), dtype, g)}
    first = seed % 18
    state["cos"], state["sin"], state["sections"] = _angles(max(64, first + case["frames"]), case["rotated"])
    state["first"] = first
    rows = _grid_rows(case, first)
    if case["positions"] == "tokens":
        shift = torch.randint(0, 8, (case["batch"], 1, 3), generator=g, device=DEVICE, dtype=torch.int32)
        state["rows"] = (rows[None] + shift).contiguous()
    else:
        state["rows"] = rows[None].expand(case["batch"], -1, -1)
    if case["grad"]:
        state["q"].requires_grad_(True), state["k"].requires_grad_(True)
        state["dq"] = _normal(state["q"].shape, dtype, g)
        state["dk"] = _normal(state["k"].shape, dtype, g)
    if own:
        from reelcache_amd import restore_kernels, rotary

        table = restore_kernels.RopeTable(state["cos"], state["sin"], state["sections"])
        state["positions"] = (rotary.TokenRows(table, state["rows"]) if case["positions"] == "tokens"
                              else restore_kernels.RopePositions(table, (first, 0, 0)))
        state["grid"] = (case["frames"], case["height"], case["width"])
    return state


def _scattered(page_counts, pages, seed):
    """Pages of each sequence, drawn without order from ``pages``."""
    order = np.random.default_rng(seed).permutation(pages).tolist()
    cuts = np.cumsum([0, *page_counts])
    return [order[a:b] for a, b in zip(cuts[:-1], cuts[1:])]


def _table(tables):
    """int32 [sequences, most pages] on the device; -1 behind a sequence's last page."""
    width = max(len(t) for t in tables)
    return torch.tensor([t + [-1] * (width - len(t)) for t in tables], dtype=torch.int32, device=DEVICE)


def _prepare_store(case, seed):
    g, dtype, new, size = _generator(seed), DTYPES[case["dtype"]], _tokens(case), case["page_tokens"]
    history = case["history"]
    counts = [-(-(history + new) // size)] * case["batch"]
    tables = _scattered(counts, sum(counts), seed)
    shape = (case["batch"] * new, case["heads"], case["head_dim"])
    state = {"case": case, "k": _normal(shape, dtype, g), "v": _normal(shape, dtype, g),
             "keys": _normal(_pool_shape(case, sum(counts)), dtype, g),
             "values": _normal(_pool_shape(case, sum(counts)), dtype, g), "table": _table(tables)}
    state["cos"], state["sin"], state["sections"] = _angles(64, case["head_dim"])
    state["rows"] = _grid_rows(case, seed % 18).repeat(case["batch"], 1)
    state["at"] = torch.arange(history, history + new, device=DEVICE)
    if own:
        from reelcache_amd import paged_cache, restore_kernels, rotary

        cache = paged_cache.PagedCache(state["keys"][None], state["values"][None])
        cache.load_tables([(pages, history + new) for pages in tables])
        state["cache"] = cache
        state["slots"] = cache.slots(list(range(case["batch"])), [history] * case["batch"], [new] * case["batch"])
        if case["rope"]:
            table = restore_kernels.RopeTable(state["cos"], state["sin"], state["sections"])
            state["positions"] = rotary.TokenRows(table, state["rows"])
    return state


def _prepare_pages(case, seed):
    g, dtype = _generator(seed), DTYPES[case["dtype"]]
    shape = (case["layers"], *_pool_shape(case, case["pages"]))
    state = {"case": case, "keys": torch.empty(shape, dtype=dtype, device=DEVICE),
             "values": torch.empty(shape, dtype=dtype, device=DEVICE)}
    state["keys"].normal_(generator=g), state["values"].normal_(generator=g)
    pages, size = case["pages"], case["page_tokens"]
    if case["kind"] == "fork":
        used = -(-case["tokens"] // size)
        state["tables"] = [(_scattered([used], pages, seed)[0], case["tokens"])]
    else:
        # Pages in use: all but ``moved`` holes among the lowest, and ``moved`` of the highest.
        free = case["moved"]
        low = np.random.default_rng(seed).permutation(pages - free)
        keep = sorted(low[free:].tolist())
        tables = [list(range(pages - free, pages)), keep]
        state["tables"] = [(table, len(table) * size) for table in tables if table]
    if own:
        from reelcache_amd import paged_cache

        state["cache"] = paged_cache.PagedCache(state["keys"], state["values"])
    return state


def _prepare_attend(case, seed):
    g, dtype, size = _generator(seed), DTYPES[case["dtype"]], case["page_tokens"]
    queries, keys = _lengths(case)
    counts = [-(-n // size) for n in keys]
    tables = _scattered(counts, sum(counts), seed)
    state = {"case": case, "q": _normal((sum(queries), case["heads"], case["head_dim"]), dtype, g),
             "keys": _normal(_pool_shape(case, sum(counts)), dtype, g),
             "values": _normal(_pool_shape(case, sum(counts)), dtype, g), "table": _table(tables)}
    most = max(queries)
    places = [[i if j < n else -1 for j, i in enumerate(range(a, a + most))]
              for a, n in zip(np.cumsum([0, *queries[:-1]]).tolist(), queries)]
    state["places"] = torch.tensor(places, device=DEVICE)  # row of q at [sequence, query], -1 behind the last
    state["queries"] = torch.tensor(queries, device=DEVICE)
    state["lengths"] = torch.tensor(keys, device=DEVICE)
    if own:
        from reelcache_amd import paged_cache

        cache = paged_cache.PagedCache(state["keys"][None], state["values"][None], layout=case["layout"])
        cache.load_tables(list(zip(tables, keys)))
        state["cache"] = cache
        state["plan"] = cache.plan(list(range(case["batch"])), queries, heads=case["heads"], block=case["block"] or None,
                                   window=case["window"] or None)
    return state


def prepare(case, seed):
    if case["kind"] == "rotate":
        return _prepare_rotate(case, seed)
    if case["kind"] == "store":
        return _prepare_store(case, seed)
    if case["kind"] == "attend":
        return _prepare_attend(case, seed)
    return _prepare_pages(case, seed)


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------


def _token_angles(cos, sin, sections, rows):
    """fp32 cosines and sines ``[..., pairs]`` of tokens at ``rows[..., 3]``."""
    column = torch.arange(cos.shape[1], device=cos.device)
    axis = (column >= sections[0]).long() + (column >= sections[0] + sections[1]).long()
    at = rows.long()[..., axis]  # each pair's table row
    return cos[at, column].float(), sin[at, column].float()


def _rotated(x, cos, sin, pairing):
    """``x[..., D]`` in fp32 with its first ``2 * pairs`` channels rotated; cos and sin broadcast."""
    pairs = cos.shape[-1]
    x = x.float()
    if pairing == "interleaved":
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
    c, d = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((c, d), dim=-1).flatten(-2) if pairing == "interleaved" else torch.cat((c, d), dim=-1)
    return torch.cat((turned, x[..., 2 * pairs:]), dim=-1)


def _run_rotate(state):
    case = state["case"]
    q, k = state["q"], state["k"]
    if own:
        from reelcache_amd import rotary

        out = rotary.rotate((q, k), state["positions"], grid=state["grid"] if case["positions"] == "grid" else None,
                            layout=case["layout"], pairing=case["pairing"])
        if not case["grad"]:
            return out
        return (*(t.detach() for t in out), *torch.autograd.grad(out, (q, k), (state["dq"], state["dk"])))
    cos, sin = _token_angles(state["cos"], state["sin"], state["sections"], state["rows"])
    axis = 2 if case["layout"] == "BTHD" else 1
    cos, sin = cos.unsqueeze(axis), sin.unsqueeze(axis)
    with torch.no_grad():
        out = [_rotated(x, cos, sin, case["pairing"]).to(x.dtype) for x in (q, k)]
        if case["grad"]:  # a rotation's transpose is the rotation back
            out += [_rotated(x, cos, -sin, case["pairing"]).to(x.dtype) for x in (state["dq"], state["dk"])]
    return tuple(out)


def _run_store(state):
    case = state["case"]
    if own:
        state["cache"].store(0, state["slots"], state["k"], state["v"], positions=state.get("positions"))
        return state["keys"], state["values"]
    k = state["k"].float()
    if case["rope"]:
        cos, sin = _token_angles(state["cos"], state["sin"], state["sections"], state["rows"])
        k = _rotated(k, cos[:, None], sin[:, None], "interleaved")
    page, row = state["at"] // case["page_tokens"], state["at"] % case["page_tokens"]
    page = state["table"].long()[:, page].reshape(-1)
    row = row.repeat(case["batch"])
    state["keys"][page, row] = k.to(state["keys"].dtype)
    state["values"][page, row] = state["v"]
    return state["keys"], state["values"]


def _lowest_free(tables, pages, count):
    """The ``count`` lowest pages that no table holds."""
    free = np.setdiff1d(np.arange(pages), np.concatenate([np.asarray(t) for t, _ in tables]))
    return free[:count]


def _run_fork(state):
    case, tables = state["case"], state["tables"]
    forks, size = case["forks"], case["page_tokens"]
    if own:
        cache = state["cache"]
        cache.load_tables(tables)
        children = [cache.fork(0) for _ in range(forks)]
        cache.extend(children, [case["added"]] * forks)
        return state["keys"], state["values"], cache.page_table(children)
    (parent, tokens), = tables
    begun = tokens % size  # tokens of the last page when it is not full: that page is copied
    after = -(-(tokens + case["added"]) // size)
    kept = len(parent) - (1 if begun else 0)
    fresh = _lowest_free(tables, case["pages"], forks * (after - kept)).reshape(forks, after - kept)
    if begun:
        to = torch.from_numpy(fresh[:, 0].copy()).to(DEVICE)
        state["keys"][:, to, :begun] = state["keys"][:, parent[-1:], :begun]
        state["values"][:, to, :begun] = state["values"][:, parent[-1:], :begun]
    table = np.concatenate([np.tile(np.asarray(parent[:kept], dtype=np.int64), (forks, 1)), fresh], axis=1)
    return state["keys"], state["values"], torch.from_numpy(table.astype(np.int32)).to(DEVICE)


def _run_compact(state):
    case, tables = state["case"], state["tables"]
    if own:
        cache = state["cache"]
        cache.load_tables(tables)
        cache.compact()
        return state["keys"], state["values"], cache.page_table(list(range(len(tables))))
    used = np.unique(np.concatenate([np.asarray(t) for t, _ in tables]))
    source = used[used >= used.size]
    target = np.setdiff1d(np.arange(used.size), used)
    src, dst = torch.from_numpy(source).to(DEVICE), torch.from_numpy(target).to(DEVICE)
    state["keys"][:, dst] = state["keys"][:, src]
    state["values"][:, dst] = state["values"][:, src]
    moved = np.arange(-1, case["pages"])  # new page of each page; -1 stays -1 at the end
    moved = np.append(moved[1:], -1)
    moved[source] = target
    width = max(len(t) for t, _ in tables)
    table = np.asarray([list(t) + [-1] * (width - len(t)) for t, _ in tables])
    return state["keys"], state["values"], torch.from_numpy(moved[table].astype(np.int32)).to(DEVICE)


def _run_attend(state):
    case = state["case"]
    q = state["q"]
    if own:
        return state["cache"].attend(0, q, state["plan"])
    size, heads, kv_heads, dim = case["page_tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    table, places = state["table"].long(), state["places"]
    batch, most = places.shape
    keys, values = state["keys"], state["values"]
    if case["layout"] == "BHTD":
        keys, values = keys.transpose(1, 2), values.transpose(1, 2)
    longest = case["longest"]
    # [sequence, key head, token, channel] in fp32; a page of -1 reads page 0, which the mask hides.
    keys = keys[table.clamp(min=0)].reshape(batch, -1, kv_heads, dim)[:, :longest].permute(0, 2, 1, 3).float()
    values = values[table.clamp(min=0)].reshape(batch, -1, kv_heads, dim)[:, :longest].permute(0, 2, 1, 3).float()
    longest = keys.shape[2]
    grouped = q[places.clamp(min=0)].float().reshape(batch, most, kv_heads, heads // kv_heads, dim)
    grouped = grouped.permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, -1, dim)
    scores = torch.matmul(grouped * dim ** -0.5, keys.transpose(2, 3).contiguous())
    scores = scores.reshape(batch, kv_heads, heads // kv_heads, most, longest)
    place = (state["lengths"] - state["queries"])[:, None] + torch.arange(most, device=DEVICE)  # of each query
    key = torch.arange(longest, device=DEVICE)
    hidden = (key >= state["lengths"][:, None])[:, None, :]
    if case["block"]:
        hidden = hidden | (key >= ((place // case["block"] + 1) * case["block"])[..., None])
    if case["window"]:
        hidden = hidden | (key <= (place - case["window"])[..., None])
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    scores.sub_(scores.amax(dim=-1, keepdim=True)).exp_()
    total = scores.sum(dim=-1, keepdim=True)
    out = torch.matmul(scores.reshape(batch, kv_heads, -1, longest), values.contiguous())
    out = out.reshape(batch, kv_heads, heads // kv_heads, most, dim) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, most, heads, dim)
    return out[places >= 0].to(q.dtype)


def run(state):
    kind = state["case"]["kind"]
    if kind == "rotate":
        return _run_rotate(state)
    if kind == "store":
        return _run_store(state)
    if kind == "fork":
        return _run_fork(state)
    if kind == "compact":
        return _run_compact(state)
    return _run_attend(state)


# ---------------------------------------------------------------------------------------------
# Bytes and operations, and values in 64 bits
# ---------------------------------------------------------------------------------------------


def _visible(case, queries, keys):
    """(query, key) pairs that one sequence's mask shows, and the keys that any of its queries sees."""
    place = np.arange(keys - queries, keys, dtype=np.int64)
    end = np.minimum(keys, (place // case["block"] + 1) * case["block"]) if case["block"] else np.full_like(place, keys)
    begin = np.maximum(0, place - case["window"] + 1) if case["window"] else np.zeros_like(place)
    return int(np.maximum(end - begin, 0).sum()), int(end.max() - begin.min())


def work(case):
    size, kind = SIZES[case["dtype"]], case["kind"]
    if kind == "rotate":
        values = case["batch"] * _tokens(case) * (case["heads"] + case["kv_heads"])
        times = 2 if case["grad"] else 1
        rows = case["batch"] * _tokens(case) * 12 if case["positions"] == "tokens" else 0
        table = 64 * case["rotated"] * 4
        return {"bytes": times * (2 * values * case["head_dim"] * size + rows + table),
                "flops": times * 3 * values * case["rotated"]}
    if kind == "store":
        tokens = case["batch"] * _tokens(case)
        values = tokens * case["heads"] * case["head_dim"]
        return {"bytes": 4 * values * size + tokens * (4 + (12 if case["rope"] else 0)),
                "flops": 3 * values if case["rope"] else 0}
    row = case["heads"] * case["head_dim"] * size
    if kind == "fork":
        begun = case["tokens"] % case["page_tokens"]
        # The shared page is read once, each fork's own written; a full last page is not copied.
        return {"bytes": max(2 * case["layers"] * begun * row * (1 + case["forks"]), 64 * case["forks"]), "flops": 0}
    if kind == "compact":
        return {"bytes": 2 * 2 * case["layers"] * case["moved"] * case["page_tokens"] * row, "flops": 0}
    queries, keys = _lengths(case)
    seen = [_visible(case, a, b) for a, b in zip(queries, keys)]
    rows = 2 * sum(queries) * case["heads"] + 2 * sum(n for _, n in seen) * case["kv_heads"]
    return {"bytes": rows * case["head_dim"] * size,
            "flops": 4 * sum(pairs for pairs, _ in seen) * case["heads"] * case["head_dim"]}


def _turned(x, state, rows, pairing, back=False):
    """``x[..., H, D]`` at ``rows[..., 3]`` in 64 bits: the pairs as complex numbers times unit ones."""
    t, h, _ = state["sections"]
    turn = torch.complex(state["cos"], state["sin"])
    parts = [turn[rows[..., 0].long(), :t], turn[rows[..., 1].long(), t:t + h], turn[rows[..., 2].long(), t + h:]]
    turn = torch.cat(parts, dim=-1).unsqueeze(-2)
    n = turn.shape[-1]
    x = x.double()
    head = x[..., :2 * n]
    number = (torch.view_as_complex(head.unflatten(-1, (n, 2)).contiguous()) if pairing == "interleaved"
              else torch.complex(head[..., :n].contiguous(), head[..., n:].contiguous()))
    number = number * (turn.conj() if back else turn)
    out = x.clone()
    if pairing == "interleaved":
        out[..., :2 * n] = torch.view_as_real(number).flatten(-2)
    else:
        out[..., :n], out[..., n:2 * n] = number.real, number.imag
    return out


def _exact_attend(case, state):
    queries, keys = _lengths(case)
    out = torch.empty(state["q"].shape, dtype=torch.float64, device=DEVICE)
    group = case["heads"] // case["kv_heads"]
    first = 0
    for sequence, (n, length) in enumerate(zip(queries, keys)):
        pages = state["table"][sequence, :-(-length // case["page_tokens"])].long()
        place = torch.arange(length - n, length, device=DEVICE)
        last = torch.full_like(place, length)
        if case["block"]:
            last = torch.minimum(last, place - place % case["block"] + case["block"])
        begin = place - case["window"] + 1 if case["window"] else torch.zeros_like(place)
        key = torch.arange(length, device=DEVICE)
        shown = (key[None] >= begin[:, None]) & (key[None] < last[:, None])
        for head in range(case["kv_heads"]):
            k, v = ((pool[pages][:, :, head] if case["layout"] == "BTHD" else pool[pages][:, head])
                    .reshape(-1, case["head_dim"])[:length].double() for pool in (state["keys"], state["values"]))
            for member in range(head * group, (head + 1) * group):
                scores = state["q"][first:first + n, member].double() @ k.T / math.sqrt(case["head_dim"])
                weights = torch.softmax(torch.where(shown, scores, torch.full_like(scores, -math.inf)), dim=1)
                out[first:first + n, member] = weights @ v
        first += n
    return out


def exact(case, seed):
    if case["kind"] in ("fork", "compact"):
        return None  # pages are copied, nothing is computed
    state = prepare(case, seed)
    if case["kind"] == "attend":
        return _exact_attend(case, state)
    if case["kind"] == "store":
        rows = torch.cat([state["table"][i].long()[state["at"] // case["page_tokens"]] * case["page_tokens"]
                          + state["at"] % case["page_tokens"] for i in range(case["batch"])])
        keys, values = state["keys"].double(), state["values"].double()
        k = _turned(state["k"], state, state["rows"], "interleaved") if case["rope"] else state["k"].double()
        keys.flatten(0, 1)[rows] = k
        values.flatten(0, 1)[rows] = state["v"].double()
        return keys, values
    with torch.no_grad():
        given = [(state["q"], False), (state["k"], False)]
        given += [(state["dq"], True), (state["dk"], True)] if case["grad"] else []
        out = []
        for x, back in given:
            x = x if case["layout"] == "BTHD" else x.transpose(1, 2)
            x = _turned(x, state, state["rows"], case["pairing"], back)
            out.append((x if case["layout"] == "BTHD" else x.transpose(1, 2)).contiguous())
        return tuple(out)
