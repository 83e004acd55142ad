"""Arrays kept in 8 bits: codes and one scale byte per block of 32 neighbours.

``quantize!`` / ``dequantize!`` stand beside the element conversions of a broadcast
(src/broadcast.jl:3-30 of the reference, ``convert.(T, x)``).  A block's scale is the smallest power
of two (2^-127 at least) that brings its largest magnitude to 127 ("int8": Int8 codes) or to 448
("e4m3": bytes of the 1-4-3 float, held as UInt8); a code is the value over the scale, rounded to
nearest even, so the rounding is the only loss: half a code of the block's scale for int8, 2^-4 of
the value for e4m3 (codes below 2^-6: 2^-10 of the scale).  A block with an infinity or a NaN reads
back as NaN.
"""
from __future__ import annotations

import numpy as np

from ._lib import check, lib
from .array import ROCArray, check_device, copyto_, on_stream
from .runtime import Stream, current_stream

BLOCK = 32
_FORMATS = {"int8": np.dtype(np.int8), "e4m3": np.dtype(np.uint8)}


def is_rows(A: ROCArray, lead: int) -> bool:
    """The first `lead` dimensions are dense and the others collapse to one (not negative) stride."""
    if A._strides is None:
        return True
    d, rows, ld = 1, 1, 0
    for k, (n, s) in enumerate(zip(A.dims, A._strides)):
        if k < lead:
            if n > 1 and s != d:
                return False
            d *= n
        elif n != 1:
            if rows == 1:
                ld = s
            elif s != ld * rows:
                return False
            rows *= n
    return ld >= 0


def rows_in(A: ROCArray | None, lead: int, st: Stream) -> ROCArray | None:
    """`A`, or a dense copy where its strides are not those of rows."""
    return A if A is None or is_rows(A, lead) else copy_on(A, st)


def copy_on(A: ROCArray, st: Stream) -> ROCArray:
    """A dense copy made by a kernel, so of an array of the stream's own device only."""
    check_device(st, A)
    return A.copy(st)


def rows_out(A: ROCArray | None, lead: int, st: Stream) -> ROCArray | None:
    """`A`, or a dense stand-in that :func:`rows_back` copies into it."""
    if A is None or is_rows(A, lead):
        return A
    check_device(st, A)                     # the operator itself sees the stand-in only
    return A.similar(stream=st)


def rows_back(A: ROCArray | None, stand_in: ROCArray | None, st: Stream) -> None:
    if stand_in is not A:
        copyto_(A, stand_in, st)


class Quantized8:
    """An array in 8 bits: ``codes`` of its dims (Int8, or UInt8 for e4m3) and ``scales`` (UInt8),
    whose first dimension counts the blocks of 32."""

    __slots__ = ("codes", "scales")

    def __init__(self, dims, format: str = "int8", stream: Stream | None = None):
        if format not in _FORMATS:
            raise ValueError(f"format must be one of {sorted(_FORMATS)}, not {format!r}")
        dims = (int(dims),) if isinstance(dims, (int, np.integer)) else tuple(int(d) for d in dims)
        if not dims:
            raise ValueError("an array kept in 8 bits has at least one dimension")
        st = stream or current_stream()
        self.codes = ROCArray(_FORMATS[format], dims, stream=st)
        self.scales = ROCArray(np.uint8, (-(-dims[0] // BLOCK),) + dims[1:], stream=st)

    @classmethod
    def wrap(cls, codes: ROCArray, scales: ROCArray) -> "Quantized8":
        """Codes and scales that exist already, views of larger arrays for instance."""
        if codes.dtype not in _FORMATS.values() or scales.dtype != np.uint8:
            raise ValueError("codes are Int8 or UInt8 (e4m3), scales UInt8")
        if codes.ndim < 1 or scales.dims != (-(-codes.dims[0] // BLOCK),) + codes.dims[1:]:
            raise ValueError(f"the scales need one byte per {BLOCK} elements of the first dimension")
        q = cls.__new__(cls)
        q.codes, q.scales = codes, scales
        return q

    @property
    def dims(self): return self.codes.dims
    shape = dims
    @property
    def format(self) -> str: return "int8" if self.codes.dtype == np.int8 else "e4m3"
    @property
    def nbytes(self) -> int: return self.codes.nbytes + self.scales.nbytes

    def __repr__(self):
        return f"Quantized8{{{self.format}}}{self.dims}"


def quantize_(q: Quantized8, X: ROCArray, stream: Stream | None = None) -> Quantized8:
    """Rows of `X` (Float16, BFloat16 or Float32) to 8 bits."""
    st = stream or current_stream()
    Xr = rows_in(X, 1, st)
    check(lib.b200_quantize(st.handle, *on_stream(st, q.codes, q.scales, Xr)))
    return q


def quantize(X: ROCArray, format: str = "int8", stream: Stream | None = None) -> Quantized8:
    st = stream or current_stream()
    return quantize_(Quantized8(X.dims, format, st), X, st)


def dequantize_(X: ROCArray, q: Quantized8, stream: Stream | None = None) -> ROCArray:
    """What the codes stand for, rounded to `X`'s type; values past its range become its largest."""
    st = stream or current_stream()
    Xr = rows_out(X, 1, st)
    check(lib.b200_dequantize(st.handle, *on_stream(st, Xr, q.codes, q.scales)))
    rows_back(X, Xr, st)
    return X


def dequantize(q: Quantized8, dtype=np.float32, stream: Stream | None = None) -> ROCArray:
    st = stream or current_stream()
    return dequantize_(ROCArray(dtype, q.dims, stream=st), q, st)
