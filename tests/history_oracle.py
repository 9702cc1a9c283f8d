"""Plain forms of the operators of long histories: 8-bit codes, means of key blocks, their choice, attention to them.

Codes and scales are defined in fp32, so their plain form is exact; attention and means are in 64 bits with the error that
a kernel may have (``U``: half a step of a rounding, relative to the value)."""

import math

import numpy as np
import torch

from operator_oracle import F32, TINY, U

LEAST = 2.0 ** -126


def encode(x, codes, dtype=None):
    """(codes, fp32 scales) of fp32 rows ``x[..., channels]`` on the CPU, by the operations that define them; ``dtype``: the
    cache's (x's without it)."""
    dtype = dtype or x.dtype
    x = x.float().cpu()
    most = x.abs().amax(dim=-1)
    lost = ~torch.isfinite(x).all(dim=-1)
    if codes == torch.int8:
        scale = (most / torch.full_like(most, 127.0)).clamp(min=LEAST)
        code = (x * (torch.ones_like(scale) / scale)[..., None]).round().clamp(-127, 127)
    else:
        # The least e with most <= 448 * 2**e, in whole numbers.
        m, e = torch.frexp(most.double())
        e = torch.where(most > 0, e - 9 + (m > 0.875).int(), torch.full_like(e, -126)).clamp(min=-126)
        scale = torch.exp2(e.double()).float()
        limit = torch.where(256 * scale.double() > torch.finfo(dtype).max, 240.0, 448.0)[..., None]
        code = (x.double() / scale.double()[..., None]).clamp(-limit, limit).float()
    code = torch.where(lost[..., None], torch.zeros_like(code), code).to(codes)
    return code, torch.where(lost, torch.full_like(scale, math.nan), scale)


def decode(code, scale, dtype):
    """What codes stand for: the fp32 product, rounded to the type."""
    return (code.float() * scale[..., None]).to(dtype)


def rotated(x, cos, sin):
    """fp32 ``x[tokens, heads, D]`` (CPU) with its first interleaved pairs turned, each operation rounded once."""
    pairs = cos.shape[-1]
    x, cos, sin = x.float().cpu().clone(), cos.float()[:, None], sin.float()[:, None]
    a, b = x[..., 0:2 * pairs:2].clone(), x[..., 1:2 * pairs:2].clone()
    x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2] = a * cos - b * sin, a * sin + b * cos
    return x


def rows_of(pool, layout):
    """A layer's pool as [pages, page_tokens, heads, ...]."""
    return pool if layout == "BTHD" else pool.transpose(1, 2)


def history(pool, layout, pages, length):
    """[length, heads, ...] of a sequence in 64 bits on the CPU; rows in dropped pages are zeros."""
    rows = rows_of(pool, layout).double().cpu()
    found = torch.stack([rows[page] if page >= 0 else torch.zeros_like(rows[0]) for page in pages]) if pages else rows[:0]
    return found.flatten(0, 1)[:length]


def visible(length, place, block=None, window=None):
    """Truth values over the keys that a query at ``place`` sees, holes apart."""
    key = np.arange(length)
    seen = np.ones(length, dtype=bool)
    if block:
        seen &= key < (math.floor(place / block) + 1) * block
    if window:
        seen &= key > place - window
    return seen


def choice(q, keys_mean, pages, length, queries, size, page_tokens, *, top, query_block, first, recent, block=None, window=None):
    """[(first query, queries, [blocks of each key head])] of a sequence's runs: the rule, stated key by key.
    ``keys_mean(block, head)``: float64 mean; ``q``: float64 [n, heads, D]; key heads from ``keys_mean.heads``."""
    blocks = -(-length // size)
    held = [pages[j * size // page_tokens] >= 0 for j in range(blocks)]
    group = q.shape[1] // keys_mean.heads
    out = []
    for start in range(0, queries, query_block):
        n = min(query_block, queries - start)
        seen = np.array([visible(length, length - queries + start + i, block, window) for i in range(n)]).reshape(n, length)
        own = math.floor((length - queries + start + n - 1) / size)
        always, scored = [], []
        for j in range(blocks):
            part = seen[:, j * size:(j + 1) * size]
            if not part.any() or not held[j]:
                continue
            whole = part.shape[1] == size and part.all()
            kept = j < first or own - recent < j <= own
            (always if kept or not whole else scored).append(j)
        found = []
        for head in range(keys_mean.heads):
            pooled = q[start:start + n, head * group:(head + 1) * group].sum(dim=(0, 1))
            scores = [float((pooled * keys_mean(j, head)).sum()) for j in scored]
            rank = sorted(range(len(scored)), key=lambda i: (0 if math.isnan(scores[i]) else 1, -scores[i] if not math.isnan(scores[i]) else 0, scored[i]))
            found.append(sorted(always + [scored[i] for i in rank[:top]]))
        out.append((start, n, found))
    return out


def attend(q, k, v, seen, dtype, scale=None):
    """(out, bound, lse, lse bound) of rows ``q[n, D]`` over keys ``k[m, D]`` (64 bits) under ``seen[n, m]``."""
    n, dim = q.shape
    scale = dim ** -0.5 if scale is None else scale
    out, bound = torch.zeros(n, dim, dtype=torch.float64), torch.zeros(n, dim, dtype=torch.float64)
    lse, lse_bound = torch.full((n,), -math.inf, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    rounded = U[dtype] if dtype != torch.float32 else 0.0
    for i in range(n):
        at = torch.from_numpy(np.flatnonzero(seen[i]))
        if not len(at):
            continue
        key, value = k[at], v[at]
        score = key @ q[i] * scale
        weight = torch.softmax(score, dim=0)
        out[i] = weight @ value
        size = weight @ value.abs()
        # As in operator_oracle.attend: scores of fp32 products and sums, exponentials, sums over the keys, weights rounded
        # to the type for the matrix cores, the result once.
        off = float(((dim + 2) * F32 * scale * (key.abs() @ q[i].abs())).max()) + 4 * F32 * float(score.abs().max()) + 4 * F32
        sums = (len(at) + 32) * F32
        bound[i] = size * 1.01 * (rounded + 2 * off + 2 * sums) + 1.01 * U[dtype] * out[i].abs() + TINY[dtype]
        if dtype == torch.float16:
            bound[i] += value.abs().sum(dim=0) * 2.0 ** -31
        lse[i] = torch.logsumexp(score, dim=0)
        lse_bound[i] = 1.01 * (off + sums) + 8 * F32 * (1 + lse[i].abs())
    return out, bound, lse, lse_bound
