"""Rotary positions: pairs of a head's elements turned by angles that grow with the position.

Element-wise over views of the projection's result, where the reference's user writes strided
broadcasts with tables of sines and cosines (src/broadcast.jl:3-30).  A plan holds the pairs'
frequencies in 2^-64 turns per position, rounded once; position times frequency wraps exactly, so an
angle is off by at most 2^-65 turns per position from the frequency's own and no table of angles is
read.
"""
from __future__ import annotations

import functools
import math

import numpy as np

from ._lib import check, lib
from .array import ROCArray, on_stream
from .quantization import copy_on
from .runtime import Stream, current_stream

_LAYOUTS = {"half": 0, "interleaved": 1}
_SCALINGS = ("none", "linear", "ntk", "yarn")


def rotary_frequencies(rot: int, base: float = 10000.0, scaling: str = "none", stretch: float = 1.0,
                       original_length: int | None = None, beta_fast: float = 32.0, beta_slow: float = 1.0):
    """Angles per position (radians) of the rot/2 pairs, and the factor on cosine and sine.

    "none": base^(-2i/rot).  "linear": those over `stretch` (positions interpolated).  "ntk": base
    times stretch^(rot/(rot-2)).  "yarn" (Peng et al. 2023): pairs that turn more than `beta_fast`
    times over `original_length` positions keep their frequency, those below `beta_slow` are
    interpolated, those between are mixed in proportion; factor 0.1 ln(stretch) + 1.  (Some models
    mix by the pair's index between two rounded bounds instead: they pass their own frequencies to
    :class:`RotaryPlan`.)"""
    if rot < 0 or rot % 2:
        raise ValueError("rotary: an even number of elements is turned")
    if scaling not in _SCALINGS:
        raise ValueError(f"rotary: scaling must be one of {_SCALINGS}, not {scaling!r}")
    if not (base > 0 and stretch > 0):
        raise ValueError("rotary: base and stretch must be positive")
    base, stretch = float(base), float(stretch)
    if scaling == "ntk" and rot > 2:
        base *= stretch ** (rot / (rot - 2.0))
    f = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if scaling == "linear":
        return [x / stretch for x in f], 1.0
    if scaling == "yarn":
        if not original_length or original_length < 1 or not beta_fast > beta_slow:
            raise ValueError("rotary: yarn needs the original length and beta_fast > beta_slow")
        keep = [min(1.0, max(0.0, (original_length * x / (2.0 * math.pi) - beta_slow) / (beta_fast - beta_slow))) for x in f]
        return [x * k + x / stretch * (1.0 - k) for x, k in zip(f, keep)], 0.1 * math.log(stretch) + 1.0
    return f, 1.0


_PI_BITS = 1280       # a binary64 is below 2^1024: 64 bits of a turn stay right, and 190 more


@functools.cache
def _two_pi() -> int:
    """2 pi 2^_PI_BITS to a few units, by Machin's formula pi/4 = 4 arctan(1/5) - arctan(1/239)."""
    one = 1 << (_PI_BITS + 32)

    def arctan(n):
        term = total = one // n
        k = 1
        while term:
            term //= -n * n
            k += 2
            total += term // k
        return total
    return (8 * (4 * arctan(5) - arctan(239))) >> 32


def _turns(x: float) -> int:
    """Angle per position in 2^-64 turns, modulo a turn.  In integers: a binary64 quotient would leave a
    fast pair 53 of the 64 bits, and the position multiplies what it is off by."""
    n, d = x.as_integer_ratio()
    n, d = n << (_PI_BITS + 65), d * _two_pi()
    return (n // d + 1) // 2 % (1 << 64)


class RotaryPlan:
    """What :func:`rotary_` and the cache's write keep between calls: the device table (UInt64, one
    entry per pair), the layout of the pairs and the factor on cosine and sine."""

    __slots__ = ("table", "layout", "factor", "_layout")

    def __init__(self, frequencies, layout: str = "half", factor: float = 1.0, stream: Stream | None = None):
        if layout not in _LAYOUTS:
            raise ValueError(f"rotary: layout must be one of {sorted(_LAYOUTS)}, not {layout!r}")
        frequencies = [float(x) for x in frequencies]
        if not all(map(math.isfinite, frequencies)) or not math.isfinite(factor):
            raise ValueError("rotary: frequencies and factor must be finite")
        turns = [_turns(x) for x in frequencies]
        self.table = ROCArray.from_host(np.array(turns, dtype=np.uint64), stream)
        self.layout, self._layout, self.factor = layout, _LAYOUTS[layout], float(factor)

    @property
    def rot(self) -> int:
        """Elements turned at the front of a head."""
        return 2 * self.table.size


def rotary_plan(rot: int, *, base: float = 10000.0, layout: str = "half", scaling: str = "none", stretch: float = 1.0,
                original_length: int | None = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
                stream: Stream | None = None) -> RotaryPlan:
    f, factor = rotary_frequencies(rot, base, scaling, stretch, original_length, beta_fast, beta_slow)
    return RotaryPlan(f, layout, factor, stream)


def rotary_(Y: ROCArray, X: ROCArray, positions: ROCArray, plan: RotaryPlan, *, adjoint: bool = False,
            stream: Stream | None = None) -> ROCArray:
    """Turns the first ``plan.rot`` elements of every head of `X`, (head size, heads, tokens) or
    (head size, heads, tokens, batch), to its token's position; the others are copied.  `positions`
    (Int32 or Int64): (tokens,) or (tokens, batch).  `adjoint` turns back: the gradient.  `Y` may be
    `X`.  Any strides above the first dimension, so slices of a fused projection need no copy."""
    if Y.dims != X.dims or Y.dtype != X.dtype:
        raise ValueError("rotary: source and destination must have the same size and element type")
    st = stream or current_stream()
    Xr = X if X._strides is None or X._strides[:1] == (1,) or X.dims[:1] == (1,) else copy_on(X, st)
    check(lib.b200_rotary(st.handle, *on_stream(st, Y, Xr, positions, plan.table), plan._layout, plan.factor, 1 if adjoint else 0))
    return Y
