"""Rotation of queries and keys by positions of several axes (frame, height, width), with gradients.

The restore kernels rotate archived keys as they write them (reelcache/restore_kernels.py:1401-1444,
:1557-1585); an engine has to turn the queries and keys of its new tokens by the same tables before
they meet.  :func:`rotate` does that for any layout, for one tensor or for several in one launch
(``rch_rotary``).  Places come from the job model of the restore:

* :class:`~reelcache_amd.restore_model.RopePositions`: a chunk's first rows, with ``grid`` the token
  grid of a separable table (a dense table takes one row per token);
* :class:`TokenRows`: a place of its own for every token, for packed pictures and videos of several
  sizes, single tokens of several sequences, or text between them.

Arithmetic: fp32 products rounded apart and one rounding to the tensor's type, as the restore rounds.
The gradient is the rotation back of the output's gradient, by the same kernel.
"""

from __future__ import annotations

import contextlib
import ctypes
import weakref
from dataclasses import dataclass
from typing import Any

import torch

from . import _lib
from ._checks import count, in_memory, need, one_of, strided
from .errors import ConfigurationError, StateError, UnsupportedError
from .restore_model import _AXES, LAYOUTS, OUTPUT_DTYPES, Remembering, RopePositions, RopeTable

PAIRINGS = ("interleaved", "half")
#: Most tensors of one call.
MAX_TENSORS = 4

_DTYPE_CODES = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16, torch.float32: _lib.DT_F32}
_NULL = contextlib.nullcontext()


@dataclass(frozen=True, eq=False)
class TokenRows(Remembering):
    """A :class:`RopeTable` row for every token.

    ``rows``: an int32 tensor on the tokens' device, ``[T, 3]`` or ``[B, T, 3]`` of (frame, height,
    width) rows for a separable table, ``[T]`` or ``[B, T]`` for a dense one; any strides.  The values
    stay on the device: a token whose row lies outside its axis turns to NaN.
    """

    table: RopeTable
    rows: torch.Tensor

    def __post_init__(self):
        need(isinstance(self.table, RopeTable), "token rows require a RopeTable")
        rows = strided(self.rows, "token rows")
        need(rows.dtype == torch.int32, "token rows must be an int32 tensor")
        last = 1 if self.table.sections is None else 2
        need(rows.ndim in (last, last + 1), "token rows are [T, 3] or [B, T, 3] (separable table), [T] or [B, T] (dense)")
        need(self.table.sections is None or rows.shape[-1] == 3, "separable token rows are (t_row, h_row, w_row)")

    @property
    def tokens(self):
        return self.rows.shape[-1 if self.table.sections is None else -2]

    @property
    def batch(self):
        """Sequences that have rows of their own, or None when all share them."""
        return self.rows.shape[0] if self.rows.ndim == (2 if self.table.sections is None else 3) else None


def entered(device):
    """A context in which ``device`` (of a tensor that is there) is current; nothing to enter when it is already."""
    return _NULL if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


def capturing():
    """Whether the current stream captures a HIP graph."""
    return torch.cuda.is_current_stream_capturing()


def need_gpu(device, what):
    if device.type != "cuda":
        raise UnsupportedError(f"{what} runs on the GPU (HIP, gfx950); move the tensors to a cuda device")
    _lib.library()  # raises UnsupportedError with the reason when the library is unavailable


def raw_stream(device):
    """The current stream of ``device`` as an integer handle."""
    return torch._C._cuda_getCurrentRawStream(device.index)


# Streams that a table's device copy has been used on: its memory comes from the upload stream, so the
# allocator has to know them before the copy is dropped (once per copy and stream).
_TABLE_STREAMS: weakref.WeakKeyDictionary = weakref.WeakKeyDictionary()
# Device copies that captured calls read: their graphs read them on every replay, whatever becomes of the table, so
# they stay for the life of the process (as the staging of captured restores does).
_CAPTURED_TABLES: set = set()


def _table_pairs(table, device, stream):
    """Address of the table's (cos, sin) pairs on ``device``, valid for work enqueued next on the current
    stream (``stream``: its handle)."""
    entry = table._device_cache.get(device)
    if entry is None or entry.ready is not None or entry.stamp != table._stamp():
        entry = table._kernel_block(device, torch.cuda.current_stream(device))
    used = _TABLE_STREAMS.get(entry)
    if used is None:
        used = _TABLE_STREAMS[entry] = set()
    if stream not in used:
        entry.block.record_stream(torch.cuda.current_stream(device))
        used.add(stream)
    if torch._C._cuda_isCurrentStreamCapturing():
        _CAPTURED_TABLES.add(entry)
    return entry.pairs.data_ptr()


_PAIRS_AT = _lib.ROTARY_FIELDS.index("pairs_ptr")
_ROWS_AT = _lib.ROTARY_FIELDS.index("rows_ptr")
_SLOTS_AT = _lib.ROTARY_FIELDS.index("slots_ptr")
_WORDS = len(_lib.ROTARY_FIELDS)


def position_fields(positions, grid, tokens, batch, head_dim, device):
    """The place fields of ``rch_rotary_job`` (pairs_ptr .. rows_axis_stride; the addresses are left 0) and
    the pair count."""
    if positions is None:
        return 0, (0,) * 16
    need(isinstance(positions, (RopePositions, TokenRows)), "positions must be RopePositions or TokenRows")
    table = positions.table
    need(table.head_dim <= head_dim, "the table rotates more channels than a head has")
    limits = (table.rows, 0, 0) if table.sections is None else table.section_rows
    axes, sections = (1, (0, 0)) if table.sections is None else (3, table.sections[:2])
    if isinstance(positions, TokenRows):
        need(grid is None, "token rows take no grid")
        rows = positions.rows
        need(rows.device == device, "token rows must be on the tensors' device")
        need(positions.tokens == tokens and positions.batch in (None, batch), "token rows do not match the tokens")
        strides = rows.stride() if axes == 3 else (*rows.stride(), 0)
        place = (0, 0, 0, 0, 0, 0, strides[0] if len(strides) == 3 else 0, strides[-2], strides[-1])
    elif axes == 1:
        need(grid is None, "a dense table takes no grid")
        need(positions.rows + tokens <= table.rows, "the tokens run past the RoPE table")
        place = (positions.rows, 0, 0, 0, 0, 0, 0, 0, 0)
    else:
        need(grid is not None and len(grid) == 3, "a separable table needs the (frames, height, width) grid of the tokens")
        for value in grid:
            count(value, "grid extent", minimum=1)
        need(grid[0] * grid[1] * grid[2] == tokens, "the grid does not hold the tokens")
        for first, extent, limit, pairs in zip(positions.rows, grid, limits, table.sections):
            need(pairs == 0 or first + extent <= limit, "the grid runs past the RoPE table")
        place = (*positions.rows, grid[1], grid[2], 0, 0, 0, 0)
    return table.pairs, (0, axes, *sections, *limits, *place)


class Launch:
    """A checked ``rch_rotary`` launch of one geometry: everything but the addresses."""

    __slots__ = ("array", "dtype", "image", "jobs", "pairing")

    def __init__(self, jobs, dtype, pairing):
        self.jobs, self.dtype = len(jobs), _DTYPE_CODES[dtype]
        self.pairing = _lib.PAIRS_HALF if pairing == "half" else _lib.PAIRS_INTERLEAVED
        flat = [value for job in jobs for value in job]
        self.array = ctypes.c_int64 * len(flat)
        self.image = bytes(self.array(*flat))

    def __call__(self, addresses, pairs, rows, slots, stream):
        """Launches with the (source, destination) addresses of the jobs and those of the table (for the
        jobs that turn), the token rows and the slots; 0 where there are none."""
        fields = self.array.from_buffer_copy(self.image)
        at = 0
        for source, target, turns in addresses:
            fields[at], fields[at + 1] = source, target
            if turns:
                fields[at + _PAIRS_AT], fields[at + _ROWS_AT] = pairs, rows
            fields[at + _SLOTS_AT] = slots
            at += _WORDS
        _lib.check(_lib.function("rch_rotary")(fields, self.jobs, self.dtype, self.pairing, stream))


def addresses_of(positions, device, stream):
    """(table pairs, token rows) addresses of a launch's positions."""
    if positions is None:
        return 0, 0
    return (_table_pairs(positions.table, device, stream),
            positions.rows.data_ptr() if isinstance(positions, TokenRows) else 0)


#: Geometries of calls that one position object remembers.
_MOST_KNOWN = 64


def known_calls(holder):
    """The launches prepared for an object's earlier calls, by their geometry."""
    known = holder.__dict__.get("_known_calls")
    if known is None or len(known) >= _MOST_KNOWN:
        known = holder.__dict__["_known_calls"] = {}
    return known


def _geometry(x, layout):
    """((batch, tokens, heads, head_dim), element strides of the same) of a tensor."""
    shape, stride, axes = x.shape, x.stride(), _AXES[layout]
    sizes = tuple(1 if axis is None else shape[axis] for axis in axes)
    return sizes, tuple(0 if axis is None else stride[axis] for axis in axes)


def _check(x, layout, name):
    in_memory(x, name)
    if x.ndim != (3 if layout == "THD" else 4):
        raise ConfigurationError(f"{name}: {layout} has the wrong number of dimensions")
    if x.dtype not in OUTPUT_DTYPES:
        raise ConfigurationError(f"{name} must be bfloat16, float16 or float32")


def changed(x):
    """Tells autograd that a kernel has written into a caller's tensor."""
    if not x.is_inference():
        torch.autograd.graph.increment_version(x)


def _span(x):
    """Byte range [first, last) that a strided tensor touches."""
    if x.numel() == 0:
        return 0, 0
    reach = sum((size - 1) * stride for size, stride in zip(x.shape, x.stride()))
    return x.data_ptr(), x.data_ptr() + (reach + 1) * x.element_size()


def _prepare(tensors, outs, positions, grid, layout, pairing, inverse):
    """The :class:`Launch` of tensors into outputs (both with unit channel stride), or None when there is
    nothing to do."""
    device = tensors[0].device
    jobs, places = [], {}
    for x, out in zip(tensors, outs):
        (batch, tokens, heads, head_dim), strides = _geometry(x, layout)
        to = _geometry(out, layout)[1]
        key = (tokens, batch, head_dim)
        if key not in places:  # queries and keys of a call share them
            places[key] = position_fields(positions, grid, tokens, batch, head_dim, device)
        pairs, place = places[key]
        jobs.append((0, 0, batch, tokens, heads, head_dim, pairs, *strides[:3], *to[:3], *place, 0, 0, 0, int(inverse), 0))
    if all(0 in job[2:6] for job in jobs):
        return None
    # A tensor without elements rides along as no work.
    return Launch([job if job[4] and job[5] else (0, 0, 0, 0, 1, 8, 0, *job[7:]) for job in jobs],
                  tensors[0].dtype, pairing)


def _run(launch, tensors, outs, positions):
    if launch is not None:
        device = tensors[0].device
        stream = raw_stream(device)
        launch([(x.data_ptr(), out.data_ptr(), True) for x, out in zip(tensors, outs)],
               *addresses_of(positions, device, stream), 0, stream)


def _rotate(tensors, positions, grid, layout, pairing, inverse):
    """The rotation of checked tensors into new ones."""
    with entered(tensors[0].device):
        known = known_calls(positions)
        key = (layout, pairing, inverse, grid, *[(x.shape, x.stride(), x.dtype, x.device) for x in tensors])
        call = known.get(key)
        if call is None:
            plain = all(x.stride(-1) == 1 or x.shape[-1] == 1 for x in tensors)
            if not plain:
                tensors = [x if x.stride(-1) == 1 else x.contiguous() for x in tensors]
            # As the input lies in memory, unless that takes the channels apart (overlapping rows).
            outs = tuple(torch.empty_like(x) for x in tensors)
            form = torch.preserve_format
            if any(out.stride(-1) != 1 and out.shape[-1] > 1 for out in outs):
                form = torch.contiguous_format
                outs = tuple(torch.empty_like(x, memory_format=form) for x in tensors)
            call = _prepare(tensors, outs, positions, grid, layout, pairing, inverse), form
            if plain:
                known[key] = call
        else:
            outs = tuple([torch.empty_like(x, memory_format=call[1]) for x in tensors])
        _run(call[0], tensors, outs, positions)
    return outs


def _rotate_into(tensors, outs, positions, grid, layout, pairing, inverse):
    """The rotation of checked tensors into given ones."""
    with entered(tensors[0].device):
        sources = [x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous() for x in tensors]
        targets = [o if o.stride(-1) == 1 or o.shape[-1] == 1 else torch.empty(o.shape, dtype=o.dtype, device=o.device)
                   for o in outs]
        _run(_prepare(sources, targets, positions, grid, layout, pairing, inverse), sources, targets, positions)
        for out, target in zip(outs, targets):
            if target is not out:
                out.copy_(target)
            else:
                changed(out)


def _table_state(table, device):
    """What a table's angles on ``device`` go by: its stamp, and the device copy where the stamp counts no
    updates (inference tensors, whose owner drops the copy)."""
    return table._stamp(), table._device_cache.get(device) if table._inference else None


class _Rotation(torch.autograd.Function):
    """The rotation as a differentiable function of its tensors; linear, so the backward pass is the
    rotation back (differentiable itself, as it goes through :func:`rotate`)."""

    @staticmethod
    def forward(ctx, positions, grid, layout, pairing, inverse, *tensors):
        ctx.arguments = (positions, grid, layout, pairing, inverse)
        ctx.set_materialize_grads(False)
        if isinstance(positions, TokenRows):
            ctx.save_for_backward(positions.rows)  # rows changed in place before the backward pass are refused
        outs = _rotate(tensors, positions, grid, layout, pairing, inverse)
        ctx.table = _table_state(positions.table, tensors[0].device)  # a table changed before the backward pass is refused
        if not all(ctx.needs_input_grad[5:]):  # a rotated tensor requires a gradient where its input does
            ctx.mark_non_differentiable(*[out for out, wanted in zip(outs, ctx.needs_input_grad[5:]) if not wanted])
        return outs

    @staticmethod
    def backward(ctx, *grads):
        positions, grid, layout, pairing, inverse = ctx.arguments
        wanted = [i for i, g in enumerate(grads) if g is not None and ctx.needs_input_grad[5 + i]]
        out = [None] * len(grads)
        if not wanted:
            return (None, None, None, None, None, *out)
        given = tuple([grads[i] for i in wanted])
        if isinstance(positions, TokenRows):
            ctx.saved_tensors  # noqa: B018  (checks the rows' version)
        if _table_state(positions.table, given[0].device) != ctx.table:
            raise StateError("the RoPE table was changed between a rotation and its backward pass")
        if torch.is_grad_enabled():  # a graph of the gradients is asked for
            turned = rotate(given, positions, grid=grid, layout=layout, pairing=pairing, inverse=not inverse)
        else:
            turned = _rotate(given, positions, grid, layout, pairing, not inverse)
        for i, g in zip(wanted, turned):
            out[i] = g
        return (None, None, None, None, None, *out)


def rotate(tensors: Any, positions, *, grid=None, layout="BTHD", pairing="interleaved", inverse=False, out=None):
    """Rotate one tensor, or a tuple of up to four in one launch (queries and keys), by ``positions``.

    ``tensors``: bfloat16, float16 or float32 of one dtype and device in ``layout`` (``"BTHD"``,
    ``"THD"`` or ``"BHTD"``), any strides; head counts may differ (interleaved pairs need an even
    ``head_dim``).  The first ``positions.table.head_dim``
    channels of a head turn and the rest are copied.  ``pairing``: channels ``(2j, 2j + 1)`` turn
    together (``"interleaved"``, as the restored caches have them) or ``(j, n + j)`` of the first ``2n``
    (``"half"``).  ``inverse`` turns back.  ``out``: a tensor (or a tuple) of the same shapes to write
    into, which may be the input itself; without it the outputs are new tensors.

    Runs on the current stream of the tensors' device.  Differentiable in the tensors (in
    reverse mode; not with ``out``); a table or token rows changed in place before the backward pass are
    refused there.  A captured call keeps the angles that the table had then.  Returns a tensor, or a tuple for a tuple.
    """
    single = isinstance(tensors, torch.Tensor)
    tensors = (tensors,) if single else tuple(tensors)
    if not 1 <= len(tensors) <= MAX_TENSORS:
        raise ConfigurationError(f"one call rotates 1 to {MAX_TENSORS} tensors")
    one_of(layout, LAYOUTS, "layout")
    one_of(pairing, PAIRINGS, "pairing")
    if not isinstance(positions, (RopePositions, TokenRows)):
        raise ConfigurationError("positions must be RopePositions or TokenRows")
    first = tensors[0]
    for x in tensors:
        _check(x, layout, "a rotated tensor")
        if x.dtype != first.dtype or x.device != first.device:
            raise ConfigurationError("the tensors of one call share dtype and device")
    need_gpu(first.device, "the rotation")
    grid = None if grid is None else tuple(grid)
    if out is None:
        if torch.is_grad_enabled() and any([x.requires_grad for x in tensors]):
            results = _Rotation.apply(positions, grid, layout, pairing, inverse, *tensors)
        else:
            results = _rotate(tensors, positions, grid, layout, pairing, inverse)
        return results[0] if single else results
    outs = (out,) if isinstance(out, torch.Tensor) else tuple(out)
    need(len(outs) == len(tensors), "out must have one tensor for each input")
    if torch.is_grad_enabled() and any(x.requires_grad for x in (*tensors, *outs)):
        raise ConfigurationError("out= is not differentiable; rotate without it, or under torch.no_grad()")
    spans = [_span(x) for x in tensors]
    for i, (x, o) in enumerate(zip(tensors, outs)):
        _check(o, layout, "out")
        need(o.shape == x.shape and o.dtype == x.dtype and o.device == x.device, "out must match its input")
        need(all(stride != 0 or size <= 1 for size, stride in zip(o.shape, o.stride())),
             "out with broadcast (zero) strides aliases itself")
        low, high = _span(o)
        for j, (a, b) in enumerate(spans):
            same = i == j and o.data_ptr() == x.data_ptr() and o.stride() == x.stride()
            need(same or high <= a or b <= low, "out overlaps an input without being it")
        for other in outs[:i]:
            a, b = _span(other)
            need(high <= a or b <= low, "the outputs overlap")
    _rotate_into(tensors, outs, positions, grid, layout, pairing, inverse)
    return out


__all__ = ["MAX_TENSORS", "PAIRINGS", "TokenRows", "rotate"]
