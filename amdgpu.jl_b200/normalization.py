"""Layer norm along the leading dimensions, and its gradient.

One pass over the rows each, where the reference's user writes a chain of ``mapreduce`` with
``dims`` and broadcasts (src/kernels/mapreduce.jl:86-173, src/broadcast.jl:3-30).  The rows that the
gradient needs are the source itself, or a checkpoint: the normalised rows in 8 bits
(:class:`Quantized8`), written by the forward pass.
"""
from __future__ import annotations

import numpy as np

from ._lib import check, lib
from .array import ROCArray, on_stream
from .quantization import Quantized8, rows_back, rows_in, rows_out
from .runtime import Stream, current_stream


def _lead(X, lead, *params) -> int:
    for p in params:
        if p is not None:
            n = len(p.dims)
            if lead is not None and lead != n:
                raise ValueError("layernorm: `lead` and the parameters differ in dimensions")
            lead = n
            if p.dims != X.dims[:n]:
                raise ValueError(f"layernorm: parameters of size {p.dims} for rows of size {X.dims[:n]}")
    if lead is None:
        lead = 1
    if not 1 <= lead <= len(X.dims):
        raise ValueError("layernorm: `lead` counts the normalised dimensions, 1 to ndims")
    return lead


def layernorm_(Y: ROCArray, X: ROCArray, gamma: ROCArray | None = None, beta: ROCArray | None = None, *, eps: float = 1e-5,
               lead: int | None = None, mean: ROCArray | None = None, rstd: ROCArray | None = None,
               checkpoint: Quantized8 | None = None, stream: Stream | None = None) -> ROCArray:
    """``Y = (X - m) r gamma + beta`` with m the mean and r the reciprocal root of the variance plus
    `eps` of every row.  A row is the first `lead` dimensions (those of `gamma` or `beta` where
    given, else 1).  `mean` and `rstd` (Float32, one per row) and `checkpoint` (``(X - m) r`` in 8
    bits) are filled in for :func:`layernorm_backward_`.  `Y` may be `X`."""
    if Y.dims != X.dims or Y.dtype != X.dtype:
        raise ValueError("layernorm: source and destination must have the same size and element type")
    lead = _lead(X, lead, gamma, beta)
    if checkpoint is not None and checkpoint.dims != X.dims:
        raise ValueError("layernorm: the checkpoint must have the source's size")
    st = stream or current_stream()
    Xr = rows_in(X, lead, st)
    Yr = Xr if Y is X and Xr is X else rows_out(Y, lead, st)
    q, s = (None, None) if checkpoint is None else (checkpoint.codes, checkpoint.scales)
    y, x, g, b, *kept = on_stream(st, Yr, Xr, gamma, beta, mean, rstd, q, s)
    check(lib.b200_layernorm(st.handle, y, x, lead, g, b, eps, *kept))
    if Yr is not Y:
        rows_back(Y, Yr, st)
    return Y


def layernorm(X: ROCArray, gamma: ROCArray | None = None, beta: ROCArray | None = None, *, eps: float = 1e-5,
              lead: int | None = None, stream: Stream | None = None) -> ROCArray:
    st = stream or current_stream()
    return layernorm_(X.similar(stream=st), X, gamma, beta, eps=eps, lead=lead, stream=st)


def layernorm_backward_(dX: ROCArray | None, dY: ROCArray, X: "ROCArray | Quantized8", gamma: ROCArray | None = None, *,
                        rstd: ROCArray, mean: ROCArray | None = None, dgamma: ROCArray | None = None,
                        dbeta: ROCArray | None = None, lead: int | None = None, stream: Stream | None = None) -> ROCArray | None:
    """The gradient of :func:`layernorm_` at `X` (with `mean` and `rstd` of the forward pass) or at
    the forward pass's checkpoint (with `rstd`).  Writes those of `dX`, `dgamma`, `dbeta` that are
    given; `dX` may be `dY` or `X`."""
    kept = isinstance(X, Quantized8)
    if X.dims != dY.dims or (not kept and X.dtype != dY.dtype):
        raise ValueError("layernorm gradient: dY must have the source's size and element type")
    if dX is not None and (dX.dims != dY.dims or dX.dtype != dY.dtype):
        raise ValueError("layernorm gradient: dX must have dY's size and element type")
    if not kept and mean is None:
        raise ValueError("layernorm gradient: the mean of the rows is needed beside the source")
    lead = _lead(dY, lead, gamma, dgamma, dbeta)
    st = stream or current_stream()
    dYr, Xr = rows_in(dY, lead, st), X if kept else rows_in(X, lead, st)
    dXr = rows_out(dX, lead, st)
    x, q, s = (None, X.codes, X.scales) if kept else (Xr, None, None)
    dx, dg, db, dy, *rest = on_stream(st, dXr, dgamma, dbeta, dYr, x, q, s, gamma, mean, rstd)
    check(lib.b200_layernorm_backward(st.handle, dx, dg, db, dy, lead, *rest))
    if dXr is not dX:
        rows_back(dX, dXr, st)
    return dX


def layernorm_backward(dY: ROCArray, X: "ROCArray | Quantized8", gamma: ROCArray | None = None, *, rstd: ROCArray,
                       mean: ROCArray | None = None, lead: int | None = None, stream: Stream | None = None):
    """``(dX, dgamma, dbeta)`` in new arrays; the last two in `gamma`'s type (Float32 without one)."""
    st = stream or current_stream()
    lead = _lead(dY, lead, gamma)
    dX = dY.similar(stream=st)
    ptype = np.dtype(np.float32) if gamma is None else gamma.dtype
    dgamma, dbeta = (ROCArray(ptype, dY.dims[:lead], stream=st) for _ in range(2))
    layernorm_backward_(dX, dY, X, gamma, rstd=rstd, mean=mean, dgamma=dgamma, dbeta=dbeta, lead=lead, stream=st)
    return dX, dgamma, dbeta
