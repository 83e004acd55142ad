"""silu and gelu, plain or with a gate, and their gradients from inputs kept as they are or in 8 bits.

``y .= f.(a)`` / ``y .= f.(a) .* b`` as one broadcast would compute them (src/broadcast.jl:3-30 of the
reference), with the codes of `a` and `b` (:class:`Quantized8`) written in the same pass where the
gradient is to take them instead of the arrays.  gelu is the tanh form.
"""
from __future__ import annotations

from ._lib import check, lib
from .array import ROCArray, on_stream
from .quantization import Quantized8, rows_back, rows_in, rows_out
from .runtime import Stream, current_stream

_ACTS = {"silu": 0, "gelu": 1}


def _act(f) -> int:
    if f not in _ACTS:
        raise ValueError(f"activation must be one of {sorted(_ACTS)}, not {f!r}")
    return _ACTS[f]


def _same(what, A, *others):
    for o in others:
        if o is not None and (o.dims != A.dims or (isinstance(o, ROCArray) and o.dtype != A.dtype)):
            raise ValueError(f"{what}: the operands must have the same size and element type")


def activation_(f: str, Y: ROCArray, A: ROCArray, gate: ROCArray | None = None, *, checkpoint: Quantized8 | None = None,
                gate_checkpoint: Quantized8 | None = None, stream: Stream | None = None) -> ROCArray:
    """``Y = f(A)``, or ``f(A) gate``; `checkpoint` and `gate_checkpoint` receive `A` and `gate` in 8
    bits for :func:`activation_backward_`.  `Y` may be `A` or `gate`."""
    act = _act(f)
    _same("activation", A, Y, gate, checkpoint, gate_checkpoint)
    st = stream or current_stream()
    Ar, Br, Yr = rows_in(A, 1, st), rows_in(gate, 1, st), rows_out(Y, 1, st)
    qa, sa = (None, None) if checkpoint is None else (checkpoint.codes, checkpoint.scales)
    qb, sb = (None, None) if gate_checkpoint is None else (gate_checkpoint.codes, gate_checkpoint.scales)
    check(lib.b200_activation(st.handle, act, *on_stream(st, Yr, Ar, Br, qa, sa, qb, sb)))
    if Yr is not Y:
        rows_back(Y, Yr, st)
    return Y


def activation(f: str, A: ROCArray, gate: ROCArray | None = None, stream: Stream | None = None) -> ROCArray:
    st = stream or current_stream()
    return activation_(f, A.similar(stream=st), A, gate, stream=st)


def activation_backward_(f: str, dA: ROCArray, dY: ROCArray, A: "ROCArray | Quantized8",
                         gate: "ROCArray | Quantized8 | None" = None, *, dgate: ROCArray | None = None,
                         stream: Stream | None = None) -> ROCArray:
    """``dA = dY f'(A)`` (times the gate) and ``dgate = dY f(A)``; `A` and `gate` both arrays or both
    checkpoints.  Destinations may be `dY` or the inputs."""
    act = _act(f)
    _same("activation gradient", dY, dA, A, gate, dgate)
    if (gate is None) != (dgate is None):
        raise ValueError("activation gradient: gate and dgate belong together")
    kept = isinstance(A, Quantized8)
    if gate is not None and isinstance(gate, Quantized8) != kept:
        raise ValueError("activation gradient: the gate must come in the form of the input, array or checkpoint")
    st = stream or current_stream()
    dYr, dAr, dBr = rows_in(dY, 1, st), rows_out(dA, 1, st), rows_out(dgate, 1, st)
    a = b = qa = sa = qb = sb = None
    if kept:
        qa, sa = A.codes, A.scales
        if gate is not None:
            qb, sb = gate.codes, gate.scales
    else:
        a, b = rows_in(A, 1, st), rows_in(gate, 1, st)
    check(lib.b200_activation_backward(st.handle, act, *on_stream(st, dAr, dBr, dYr, a, b, qa, sa, qb, sb)))
    rows_back(dA, dAr, st)
    rows_back(dgate, dBr, st)
    return dA
