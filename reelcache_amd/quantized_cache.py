"""A KV cache whose pages hold 8-bit codes: half the memory of 16-bit pages, and half the bytes that attention reads.

:class:`QuantizedCache` is a :class:`~reelcache_amd.paged_cache.PagedCache` (sequences fork, extend, drop, compact, page
tables and plans are the same) over pools of codes with an fp32 scale for every token and head.  ``store`` rotates and
quantises new tokens as it writes them (``rch_codes_store``), ``read`` gives back the values that the codes stand for
(``rch_codes_read``), and ``attend`` attends to those values as it reads the codes.  The archives' quantiser
(reelcache/_hevc.py:400-540) scales each rank column of a chunk; here a row has to stand alone, since it is written once,
token by token, and shared, copied and dropped with its page.

Formats, for the largest magnitude ``m`` of a token's head:

* ``torch.int8``: scale ``max(m / 127, 2**-126)``, codes ``rint(x / scale)`` in -127 .. 127 (off by half a step of m / 127);
* ``torch.float8_e4m3fn``: scale ``2**e``, the least that holds ``m <= 448 * scale``, codes ``x / scale`` rounded to nearest
  even (off by ``2**-4`` of each value: better for rows with few large channels, and cheaper to read); within +-240 where
  256 times the scale is more than the cache's ``dtype`` holds.  Of a scale that a caller wrote, the power of two counts.

A code ``c`` stands for ``c * scale``, rounded to the cache's ``dtype``.  A token's head that holds an infinity or a NaN
stands for NaN in all its channels.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._checks import count, in_memory, need, one_of
from .errors import ConfigurationError, UnsupportedError
from .paged_cache import _LAYOUTS, PagedCache, _apart, _reach
from .rotary import _DTYPE_CODES, _span, changed, entered, known_calls, need_gpu, position_fields, raw_stream

#: Types of the pools, and of the values that their codes stand for.
CODE_DTYPES = (torch.int8, torch.float8_e4m3fn)
VALUE_DTYPES = (torch.bfloat16, torch.float16)

_FORMATS = {torch.int8: _lib.CODES_INT8, torch.float8_e4m3fn: _lib.CODES_E4M3}
_Image = ctypes.c_int64 * len(_lib.CODES_FIELDS)
_CODES_AT, _SCALES_AT, _SLOTS_AT, _PAIRS_AT, _ROWS_AT = (
    _lib.CODES_FIELDS.index(name) for name in ("k_codes_ptr", "k_scales_ptr", "slots_ptr", "pairs_ptr", "rows_ptr"))


class QuantizedCache(PagedCache):
    """K and V pools of every layer in 8-bit codes, and the pages of each sequence.

    ``keys``, ``values``: pools as :class:`PagedCache` takes them, of one of :data:`CODE_DTYPES`.  ``key_scales``,
    ``value_scales``: fp32 ``[layers, pages, heads, page_tokens]``, whatever the layout, with unit stride over the tokens.
    ``dtype``: what the codes stand for, and what tokens and queries come in (:data:`VALUE_DTYPES`).
    Attention is tiled for the matrix cores where ``head_dim`` is a multiple of 16 (16-bit pools: of 8).
    """

    _POOL_DTYPES, _POOL_TYPES = CODE_DTYPES, "int8 or float8_e4m3fn"

    def __init__(self, keys, values, key_scales, value_scales, *, dtype=torch.bfloat16, layout="BTHD"):
        super().__init__(keys, values, layout=layout)
        one_of(dtype, VALUE_DTYPES, "the dtype of a quantised cache")
        if self.head_dim > _lib.CODES_MAX_DIM:
            raise UnsupportedError(f"a quantised cache takes at most {_lib.CODES_MAX_DIM} channels to a head")
        shape = (self.layers, self.pages, self.heads, self.page_tokens)
        for scales, name in ((key_scales, "key_scales"), (value_scales, "value_scales")):
            in_memory(scales, name)
            need(scales.shape == shape and scales.dtype == torch.float32 and scales.device == self.device,
                 f"{name} must be fp32 [layers, pages, heads, page_tokens] on the pools' device")
            need(scales.stride(3) == 1 or self.page_tokens == 1, f"{name} must have unit stride over the tokens")
            need(_apart(scales), f"{name} must keep its elements apart")
            need(not scales.requires_grad, f"{name} must not require gradients")
        need(key_scales.data_ptr() != value_scales.data_ptr(), "keys and values need scales of their own")
        self.key_scales, self.value_scales, self.dtype = key_scales, value_scales, dtype
        self.codes = _FORMATS[keys.dtype]
        self._scale_reach = _reach(key_scales), _reach(value_scales)
        self._scale_bytes = 4 * key_scales.stride(0), 4 * value_scales.stride(0)
        self._geometry += (dtype, key_scales.stride()[1:], value_scales.stride()[1:])
        self._counted += tuple(scales for scales in (key_scales, value_scales) if not scales.is_inference())
        self._moving = tuple(scales.unsqueeze(4) for scales in (key_scales, value_scales))  # as pools of one channel
        for scales in self._moving:
            self._take_along(scales, (1, 3, 2))

    @classmethod
    def allocate(cls, pages, page_tokens, heads, head_dim, *, codes=torch.int8, layers=1, dtype=torch.bfloat16, device="cuda",
                 layout="BTHD"):
        """A cache over new, uninitialised pools of ``codes``."""
        one_of(layout, _LAYOUTS, "pool layout")
        one_of(codes, CODE_DTYPES, "codes")
        for value, name in ((pages, "pages"), (page_tokens, "page_tokens"), (heads, "heads"), (head_dim, "head_dim"),
                            (layers, "layers")):
            count(value, name, minimum=1)
        rows = (page_tokens, heads) if layout == "BTHD" else (heads, page_tokens)
        keys, values = (torch.empty((layers, pages, *rows, head_dim), dtype=codes, device=device) for _ in range(2))
        scales = [torch.empty((layers, pages, heads, page_tokens), dtype=torch.float32, device=device) for _ in range(2)]
        return cls(keys, values, *scales, dtype=dtype, layout=layout)

    # -----------------------------------------------------------------------------------------

    def _pools(self):
        return self.keys, self.values, self.key_scales, self.value_scales

    def _scales(self, layer):
        k_bytes, v_bytes = self._scale_bytes
        return self.key_scales.data_ptr() + layer * k_bytes, self.value_scales.data_ptr() + layer * v_bytes

    def _scale_strides(self):
        return tuple(scales.stride(axis) for scales in (self.key_scales, self.value_scales) for axis in (1, 2))

    def view(self, layer, target, sequence, start, tokens):
        """Refused: a restore writes values of the cache's dtype.  Restore into a tensor of its own and ``store`` that."""
        raise UnsupportedError("a restore cannot write codes; restore into a tensor and store it")

    def _fields(self, dense, tokens, turned=(0, (0,) * 16)):
        """The ``rch_codes`` image of a call: everything but the addresses."""
        page, token, head = self._axes
        k, v = self.keys.stride(), self.values.stride()
        fields = (0, 0, dense[0].stride(0), dense[0].stride(1), dense[1].stride(0), dense[1].stride(1), 0, 0, k[page], k[token],
                  k[head], v[page], v[token], v[head], 0, 0, *self._scale_strides(), tokens, self.heads, self.head_dim,
                  self.pages, self.page_tokens, 0, self.codes, turned[0], *turned[1])
        return bytes(_Image(*fields))

    def _addressed(self, image, layer, dense, slots):
        """A call's fields with its addresses, but those of the positions."""
        fields = _Image.from_buffer_copy(image)
        k_bytes, v_bytes = self._layer_bytes
        fields[0], fields[1] = dense
        fields[_CODES_AT], fields[_CODES_AT + 1] = self.keys.data_ptr() + layer * k_bytes, self.values.data_ptr() + layer * v_bytes
        fields[_SCALES_AT], fields[_SCALES_AT + 1] = self._scales(layer)
        fields[_SLOTS_AT] = slots
        return fields

    def _store_launch(self, sources, positions, grid, tokens):
        return tuple(map(_reach, sources)), self._fields(sources, tokens, position_fields(positions, grid, tokens, 1, self.head_dim, self.device))

    def _launch_store(self, launch, layer, sources, pools, turned, slots, stream):
        (k_reach, v_reach), image = launch
        k, v = sources
        for scales, room in zip((self.key_scales.data_ptr(), self.value_scales.data_ptr()), self._scale_reach):
            if (k < scales + room and scales < k + k_reach) or (v < scales + room and scales < v + v_reach):
                raise ConfigurationError("what a store reads overlaps the scales that it writes")
        fields = self._addressed(image, layer, sources, slots)
        fields[_PAIRS_AT], fields[_ROWS_AT] = turned
        _lib.check(_lib.function("rch_codes_store")(fields, _DTYPE_CODES[self.dtype], stream))

    def read(self, layer, places, *, out=None):
        """The keys and values of tokens, as their codes stand for them: two tensors ``[tokens, heads, head_dim]`` of the
        cache's dtype.

        ``places``: :class:`~reelcache_amd.paged_cache.Places` (or ``Slots``) of this cache.  ``out``: two tensors of that
        shape to write into, any strides.  Runs on the current stream; not differentiable.  Returns ``out``.
        """
        if type(layer) is not int or not 0 <= layer < self.layers:
            raise ConfigurationError("there is no such layer")
        self._current(places)
        shape = (places.tokens, self.heads, self.head_dim)
        given = out is not None
        if given:
            out = tuple(out)
            self._check_out(out, shape)
        need_gpu(self.device, "a paged cache")
        with entered(self.device):
            if given:
                targets = [x if x.stride(2) == 1 or self.head_dim == 1 else torch.empty(shape, dtype=x.dtype, device=x.device)
                           for x in out]
            else:
                targets = out = (torch.empty(shape, dtype=self.dtype, device=self.device),
                                 torch.empty(shape, dtype=self.dtype, device=self.device))
            if places.tokens == 0:
                return out
            keys, values = targets
            known = known_calls(places)
            key = ("read", keys.stride(), values.stride())
            image = known.get(key)
            if image is None:
                image = known[key] = self._fields(targets, places.tokens)
            stream = raw_stream(self.device)
            fields = self._addressed(image, layer, (keys.data_ptr(), values.data_ptr()), places.index.data_ptr())
            _lib.check(_lib.function("rch_codes_read")(fields, _DTYPE_CODES[self.dtype], stream))
            if stream != places.stream:  # the allocator learns of a stream that the index was not made on
                places.index.record_stream(torch.cuda.current_stream(self.device))
            if given:
                for x, target in zip(out, targets):
                    if target is not x:
                        x.copy_(target)
                    else:
                        changed(x)
        return out

    def _check_out(self, out, shape):
        need(len(out) == 2, "out must be the tensors of the keys and of the values")
        for x, name in zip(out, ("out of the keys", "out of the values")):
            in_memory(x, name)
            need(x.shape == shape and x.dtype == self.dtype and x.device == self.device,
                 f"{name} must be [tokens, heads, head_dim] of the cache's dtype and device")
            need(not x.requires_grad, f"{name} must not require gradients")
            need(_apart(x), f"{name} must keep its elements apart")
        spans = [_span(x) for x in (*out, *self._pools())]
        for i, (low, high) in enumerate(spans[:2]):
            need(all(high <= a or b <= low for a, b in spans[i + 1:]), "out overlaps the other one, or a pool")


__all__ = ["CODE_DTYPES", "QuantizedCache", "VALUE_DTYPES"]
