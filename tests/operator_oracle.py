"""Plain 64-bit forms of the cache operators, with the error that each kernel may have.

Half a step of a rounding is ``finfo(t).eps / 2`` relative to the value (``U`` below; fp32: 2**-24).
"""

import math

import numpy as np
import torch

F32 = 2.0 ** -24
U = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}
# Half a step of the subnormals, which are rounded absolutely.
TINY = {t: torch.finfo(t).tiny * torch.finfo(t).eps / 2 for t in U}


def tables(rows, pairs, base=10000.0):
    """(cos, sin, sections): float64 [rows, pairs] of a three-axis table with a third of the pairs for
    height and width each."""
    spatial = pairs // 3
    sections = (pairs - 2 * spatial, spatial, spatial)
    frequency = torch.cat([base ** (-torch.arange(n, dtype=torch.float64) / max(n, 1)) for n in sections])
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * frequency[None]
    return angle.cos(), angle.sin(), sections


def rotate(x, cos, sin, pairing="interleaved"):
    """(value, bound) of ``x[..., D]`` turned by float64 cos / sin ``[..., pairs]`` (broadcast)."""
    dtype, x = x.dtype, x.double().cpu()
    pairs = cos.shape[-1]
    if pairing == "interleaved":
        first, second = slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)
    else:
        first, second = slice(0, pairs), slice(pairs, 2 * pairs)
    a, b = x[..., first], x[..., second]
    value, size = x.clone(), torch.zeros_like(x)
    value[..., first], value[..., second] = a * cos - b * sin, a * sin + b * cos
    size[..., first], size[..., second] = (a * cos).abs() + (b * sin).abs(), (a * sin).abs() + (b * cos).abs()
    # Table entry, product and sum are each rounded once in fp32 (three half steps of the terms; 1.01 for
    # their second order), then the result once to its type.
    bound = 3.03 * F32 * size + 1.01 * U[dtype] * value.abs() + TINY[dtype]
    bound[..., 2 * pairs:] = 0
    return value, bound


def token_angles(cos, sin, sections, rows):
    """float64 [..., pairs] cos and sin of tokens at int rows [..., 3]."""
    axis = torch.tensor([0] * sections[0] + [1] * sections[1] + [2] * sections[2])
    at = rows.long()[..., axis]
    column = torch.arange(cos.shape[1])
    return cos[at, column], sin[at, column]


def grid_rows(first, grid):
    axes = torch.meshgrid(*(torch.arange(n) + f for f, n in zip(first, grid)), indexing="ij")
    return torch.stack([a.reshape(-1) for a in axes], dim=1).int()


def attend(q, keys, values, pages, length, queries, page_tokens, *, block=None, window=None, scale=None,
           layout="BTHD"):
    """(out, bound, lse, lse bound) of one sequence: ``q[n, heads, D]`` over pools ``[pages, T, H, D]``
    (or ``[pages, H, T, D]``); float64 on the CPU."""
    dtype = q.dtype
    q, keys, values = (x.double().cpu() for x in (q, keys, values))
    if layout == "BHTD":
        keys, values = keys.transpose(1, 2), values.transpose(1, 2)
    n, heads, dim = q.shape
    kv_heads = keys.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    out, bound = torch.zeros(n, heads, dim, dtype=torch.float64), torch.zeros(n, heads, dim, dtype=torch.float64)
    lse, lse_bound = torch.full((n, heads), -math.inf, dtype=torch.float64), torch.zeros(n, heads, dtype=torch.float64)
    key = np.arange(length)
    held = np.array([pages[j // page_tokens] >= 0 for j in key], dtype=bool) if length else np.zeros(0, bool)
    rounded = U[dtype] if dtype != torch.float32 else 0.0
    for i in range(n):
        place = length - queries + i
        seen = held.copy()
        if block:
            seen &= key < (math.floor(place / block) + 1) * block
        if window:
            seen &= key > place - window
        at = key[seen]
        if not len(at):
            continue
        page = torch.tensor([pages[j // page_tokens] for j in at])
        row = torch.tensor(at % page_tokens)
        for head in range(heads):
            member = head * kv_heads // heads
            k, v = keys[page, row, member], values[page, row, member]
            score = k @ q[i, head] * scale
            weight = torch.softmax(score, dim=0)
            out[i, head] = weight @ v
            size = weight @ v.abs()
            # A score: dim products and sums in fp32 and the scaling; then the exponent's argument and the
            # exponential (two half steps each, relative to the largest argument and to the value).
            off = float(((dim + 2) * F32 * scale * (k.abs() @ q[i, head].abs())).max())
            off += 4 * F32 * float(score.abs().max()) + 4 * F32
            sums = (len(at) + 32) * F32  # fp32 sums over the keys, their joining and the quotient
            # Weights and their sum carry `off` and `sums` each; weights are rounded to the type for the
            # matrix cores, and the result once.
            bound[i, head] = size * 1.01 * (rounded + 2 * off + 2 * sums) + 1.01 * U[dtype] * out[i, head].abs() + TINY[dtype]
            if dtype == torch.float16:  # weights below the smallest fp16 step (2**-24, scaled up by 2**7)
                bound[i, head] += v.abs().sum(dim=0) * 2.0 ** -31
            lse[i, head] = torch.logsumexp(score, dim=0)
            lse_bound[i, head] = 1.01 * (off + sums) + 8 * F32 * (1 + lse[i, head].abs())
    return out, bound, lse, lse_bound


def worst(value, expected, bound):
    """Largest excess of |value - expected| over the bound (nan where one is nan and the other is not)."""
    value = value.double().cpu()
    same = (value == expected) | (value.isnan() & expected.isnan())
    excess = torch.where(same, torch.zeros_like(bound), (value - expected).abs() - bound)
    return float(excess.max()) if excess.numel() else 0.0
