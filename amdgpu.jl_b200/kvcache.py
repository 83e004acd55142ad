"""Key/value cache in 8 bits, in pages: tokens are quantised as they are written, contexts are read back.

Whole rows scattered and gathered by index, beside the element-wise ``getindex`` and compaction of
src/kernels/indexing.jl:8-36 of the reference.  Slots and pages are 1-based like every index of this
package; slot s is place (s-1) mod page_size of page (s-1) div page_size + 1.
"""
from __future__ import annotations

from ._lib import check, lib
from .array import ROCArray, on_stream
from .quantization import Quantized8, copy_on
from .rotary import RotaryPlan
from .runtime import Stream, current_stream


class QuantizedCache:
    """Keys and values as :class:`Quantized8` of dims (head size, heads, page size, pages).  They may
    be views with any strides above the first dimension; head sizes may differ."""

    __slots__ = ("keys", "values")

    def __init__(self, keys: Quantized8, values: Quantized8):
        if len(keys.dims) != 4 or len(values.dims) != 4 or keys.dims[1:] != values.dims[1:]:
            raise ValueError("a cache is (head size, heads, page size, pages), alike for keys and values but for the head size")
        if keys.format != values.format:
            raise ValueError("keys and values of a cache have one format")
        self.keys, self.values = keys, values

    @property
    def page_size(self) -> int: return self.keys.dims[2]
    @property
    def pages(self) -> int: return self.keys.dims[3]
    @property
    def slots(self) -> int: return self.page_size * self.pages
    @property
    def format(self) -> str: return self.keys.format

    def _arrays(self):
        return self.keys.codes, self.keys.scales, self.values.codes, self.values.scales


def quantized_cache(head_dim: int, heads: int, page_size: int, pages: int, format: str = "int8", *,
                    value_dim: int | None = None, stream: Stream | None = None) -> QuantizedCache:
    """An empty cache (zeros)."""
    st = stream or current_stream()
    sides = []
    for d in (head_dim, head_dim if value_dim is None else value_dim):
        q = Quantized8((d, heads, page_size, pages), format, st)
        q.codes.fill_(0, st)
        q.scales.fill_(0, st)
        sides.append(q)
    return QuantizedCache(*sides)


def _neighbours(A: ROCArray, st: Stream) -> ROCArray:
    return A if A._strides is None or A._strides[:1] == (1,) or A.dims[:1] == (1,) else copy_on(A, st)


def cache_write_(cache: QuantizedCache, K: ROCArray, V: ROCArray, slots: ROCArray, *, rotary: RotaryPlan | None = None,
                 positions: ROCArray | None = None, stream: Stream | None = None) -> QuantizedCache:
    """Writes the tokens of `K` and `V`, (head size, heads, tokens), to their `slots` (Int32 or Int64,
    one per token).  Slot 0 leaves a token out (a padded batch); of several tokens with one slot the
    last is kept; a slot outside the cache is not written and surfaces as an error at the next
    synchronisation.  With `rotary` the keys are turned to their `positions` on the way.  More than
    2048 tokens take 4 bytes per slot of the cache as workspace, which the stream keeps."""
    if (rotary is None) != (positions is None):
        raise ValueError("cache write: a rotary plan and positions belong together")
    st = stream or current_stream()
    K, V = _neighbours(K, st), _neighbours(V, st)
    kq, ks, vq, vs = cache._arrays()
    table = None if rotary is None else rotary.table
    layout, factor = (0, 1.0) if rotary is None else (rotary._layout, rotary.factor)
    check(lib.b200_cache_write(st.handle, *on_stream(st, kq, ks, vq, vs, K, V, slots, positions, table), layout, factor))
    return cache


def cache_read_(K: ROCArray, V: ROCArray, cache: QuantizedCache, pages: ROCArray, lengths: ROCArray,
                stream: Stream | None = None):
    """Reads contexts back into `K` and `V`, (head size, heads, places, sequences): place l of sequence
    b out of page ``pages[l div page_size, b]``, for ``lengths[b]`` places; the places behind are left
    as they were.  A length past the places or the page table, or a page outside the cache, surfaces
    as an error at the next synchronisation; what is in range is read."""
    st = stream or current_stream()
    kq, ks, vq, vs = cache._arrays()
    check(lib.b200_cache_read(st.handle, *on_stream(st, K, V, kq, ks, vq, vs, pages, lengths)))
    return K, V
