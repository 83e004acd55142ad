"""Rotary positions against binary64: layouts, part of the head, stretched contexts, far positions."""
import numpy as np
import pytest

import row_reference as ref
from helpers import Guarded, bits_equal

pytestmark = pytest.mark.gpu

# head size, turned elements, heads, tokens
SHAPES = [(2, 2, 1, 1), (6, 4, 3, 5), (8, 8, 1, 3), (10, 10, 2, 7), (16, 16, 4, 9), (64, 64, 8, 33), (64, 32, 2, 100), (80, 26, 5, 11),
          (96, 64, 16, 48), (128, 128, 40, 17), (128, 0, 2, 3), (192, 64, 1, 1000), (256, 256, 1, 1), (576, 64, 3, 4)]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", list(ref.TYPES))
def test_against_the_formula(gpu, dtype, layout):
    t = ref.TYPES[dtype]
    for k, (d, rot, heads, n) in enumerate(SHAPES):
        rng = np.random.default_rng(k)
        x = rng.standard_normal((d, heads, n)).astype(t)
        scaling = ("none", "linear", "ntk", "yarn")[k % 4]
        kw = dict(scaling=scaling, stretch=4.0, original_length=2048)
        freq, factor = gpu.rotary.rotary_frequencies(rot, **kw) if rot else ([], 1.0)
        plan = gpu.rotary_plan(rot, layout=layout, **kw) if rot else gpu.RotaryPlan([], layout)
        pos = rng.integers(0, 100_000, n).astype(np.int32 if k % 2 else np.int64)
        pos[0] = 0
        X, P = gpu.ROCArray.from_host(x), gpu.ROCArray.from_host(pos)
        for adjoint in (False, True):
            Y = Guarded(gpu, t, (d, heads, n))
            gpu.rotary_(Y.array, X, P, plan, adjoint=adjoint)
            want = ref.turn(x, pos, freq, factor, layout, adjoint)
            ref.within(Y.array.to_host(), want, ref.turn_slack(x, rot, factor, layout), (d, rot, heads, n, adjoint))
            Y.check((d, rot))
            assert bits_equal(gpu.rotary_(X.copy(), X, P, plan, adjoint=adjoint).to_host(), Y.array.to_host())
            inplace = X.copy()
            gpu.rotary_(inplace, inplace, P, plan, adjoint=adjoint)
            assert bits_equal(inplace.to_host(), Y.array.to_host())


def test_far_and_negative_positions(gpu):
    """The same accuracy at 2^31 as at 1; binary64 angles are themselves good to 2^-22 there, so the
    reference takes them in extended precision."""
    d = 64
    freq, _ = gpu.rotary.rotary_frequencies(d)
    plan = gpu.rotary_plan(d)
    pos = np.array([1, -1, 1 << 20, (1 << 31) - 1, 1 << 33, -(1 << 33), 5_000_000_019], dtype=np.int64)
    x = np.random.default_rng(0).standard_normal((d, 2, len(pos))).astype(np.float32)
    got = gpu.rotary_(gpu.ROCArray(np.float32, x.shape), gpu.ROCArray.from_host(x), gpu.ROCArray.from_host(pos), plan).to_host()
    # turns in exact integer arithmetic on the frequencies as binary64 has them
    from fractions import Fraction
    two_pi = Fraction(6283185307179586476925286766559005768394338798750211641949889, 10 ** 60)
    turns = np.array([[float((Fraction(f) * int(p) / two_pi) % 1) for p in pos] for f in freq])
    c, s = np.cos(2 * np.pi * turns)[:, None], np.sin(2 * np.pi * turns)[:, None]
    a, b = x[: d // 2].astype(np.float64), x[d // 2:].astype(np.float64)
    want = np.concatenate([a * c - b * s, b * c + a * s])
    # the table holds turns per position as binary64 rounds them: |pos| 2^-53 of the angle's turns
    table = 2 * np.pi * np.abs(pos).astype(np.float64)[None, None] * 2.0 ** -53 * 2
    ref.within(got, want, ref.turn_slack(x, d, 1.0, "half") + table * (np.abs(np.concatenate([a, a])) + np.abs(np.concatenate([b, b]))))


def test_views_of_a_projection(gpu):
    """Queries and keys as slices of one array, heads and tokens swapped, a batch, misaligned heads."""
    rng = np.random.default_rng(4)
    t = ref.BF16
    for d, rot in ((64, 64), (72, 24), (36, 18)):
        for layout in ("half", "interleaved"):
            freq, _ = gpu.rotary.rotary_frequencies(rot)
            plan = gpu.rotary_plan(rot, layout=layout)
            qkv = rng.standard_normal((d, 10, 21)).astype(t)
            pos = rng.integers(0, 4000, 21).astype(np.int32)
            A, P = gpu.ROCArray.from_host(qkv), gpu.ROCArray.from_host(pos)
            V = A.subview(slice(None), slice(6, 8), slice(None))
            got = gpu.rotary_(gpu.ROCArray(t, (d, 2, 21)), V, P, plan).to_host()
            x = qkv[:, 6:8]
            ref.within(got, ref.turn(x, pos, freq, 1.0, layout), ref.turn_slack(x, rot, 1.0, layout), (d, layout))
            gpu.rotary_(V, V, P, plan)                                                    # in place in the projection
            h = A.to_host()
            assert bits_equal(h[:, 6:8], got) and bits_equal(h[:, :6], qkv[:, :6]) and bits_equal(h[:, 8:], qkv[:, 8:])
            S = gpu.ROCArray.from_host(np.ascontiguousarray(qkv.transpose(0, 2, 1))).permuteddims((1, 3, 2))
            out = gpu.ROCArray(t, (d, 21, 10)).permuteddims((1, 3, 2))
            gpu.rotary_(out, S, P, plan)
            ref.within(out.to_host(), ref.turn(qkv, pos, freq, 1.0, layout), ref.turn_slack(qkv, rot, 1.0, layout), (d, layout, "swapped"))
            b = rng.standard_normal((d, 3, 5, 4)).astype(t)
            pb = rng.integers(0, 4000, (5, 4)).astype(np.int64)
            B = gpu.ROCArray.from_host(b)
            got = gpu.rotary_(B.similar(), B, gpu.ROCArray.from_host(pb), plan).to_host()
            ref.within(got, ref.turn(b, pb, freq, 1.0, layout), ref.turn_slack(b, rot, 1.0, layout), (d, layout, "batch"))
            got = gpu.rotary_(B.similar(), B, gpu.ROCArray.from_host(pb[:, 0].copy()), plan).to_host()      # one row of positions for all
            ref.within(got, ref.turn(b, np.repeat(pb[:, :1], 4, 1), freq, 1.0, layout), ref.turn_slack(b, rot, 1.0, layout), (d, layout, "shared"))
            off = gpu.ROCArray.from_host(rng.standard_normal(d * 8 + 1).astype(t))        # heads off 16 bytes
            O = off.view(1, d * 8 + 1).reshape(d, 2, 4)
            got = gpu.rotary_(gpu.ROCArray(t, (d, 2, 4)), O, gpu.ROCArray.from_host(pos[:4].copy()), plan).to_host()
            ref.within(got, ref.turn(O.to_host(), pos[:4], freq, 1.0, layout), ref.turn_slack(O.to_host(), rot, 1.0, layout), (d, "off"))
    e = gpu.ROCArray(np.float32, (8, 2, 0))
    assert gpu.rotary_(e.similar(), e, gpu.ROCArray(np.int32, 0), gpu.rotary_plan(8)).dims == (8, 2, 0)


def test_gradient_is_the_adjoint(gpu):
    """<turn(x), y> = <x, adjoint(y)>, and turning there and back scales by factor^2."""
    rng = np.random.default_rng(6)
    d, n = 32, 50
    plan = gpu.rotary_plan(d, scaling="yarn", stretch=16.0, original_length=1024, layout="interleaved")
    x, y = (rng.standard_normal((d, 3, n)).astype(np.float32) for _ in range(2))
    P = gpu.ROCArray.from_host(rng.integers(0, 1 << 20, n).astype(np.int64))
    X, Y = gpu.ROCArray.from_host(x), gpu.ROCArray.from_host(y)
    tx, ay = gpu.rotary_(X.similar(), X, P, plan), gpu.rotary_(Y.similar(), Y, P, plan, adjoint=True)
    left, right = (tx.to_host().astype(np.float64) * y).sum(), (x.astype(np.float64) * ay.to_host()).sum()
    assert abs(left - right) <= 16 * ref.U * plan.factor * (np.abs(x).sum() + np.abs(y).sum())
    back = gpu.rotary_(X.similar(), tx, P, plan, adjoint=True).to_host()
    pair = np.abs(x[0::2]) + np.abs(x[1::2])
    assert (np.abs(back - plan.factor ** 2 * x.astype(np.float64)) <= 40 * ref.U * plan.factor ** 2 * np.repeat(pair, 2, 0)).all()


def test_large_launches(gpu):
    """Many tokens of few heads, and few tokens of many heads."""
    rng = np.random.default_rng(8)
    for d, heads, n in ((64, 1, 70_000), (64, 3000, 2), (128, 5, 6001)):
        x = rng.standard_normal((d, heads, n)).astype(np.float32)
        pos = rng.integers(0, 1 << 17, n).astype(np.int32)
        freq, _ = gpu.rotary.rotary_frequencies(d)
        X = gpu.ROCArray.from_host(x)
        got = gpu.rotary_(X.similar(), X, gpu.ROCArray.from_host(pos), gpu.rotary_plan(d)).to_host()
        ref.within(got, ref.turn(x, pos, freq, 1.0, "half"), ref.turn_slack(x, d, 1.0, "half"), (d, heads, n))


def test_positions_of_any_size(gpu):
    """An angle is off by half of 2^-64 turns per position from the frequency as binary64 has it: as exact at
    2^40 as at 1."""
    from fractions import Fraction
    two_pi = Fraction(6283185307179586476925286766559005768394338798750211641949889, 10 ** 60)
    d = 128
    freq, _ = gpu.rotary.rotary_frequencies(d, base=500_000.0)
    plan = gpu.rotary_plan(d, base=500_000.0)
    pos = np.array([3, 1 << 31, -(1 << 31) - 5, (1 << 36) + 77, 1 << 40, -(1 << 40) - 1], dtype=np.int64)
    x = np.random.default_rng(1).standard_normal((d, 2, len(pos))).astype(np.float32)
    got = gpu.rotary_(gpu.ROCArray(np.float32, x.shape), gpu.ROCArray.from_host(x), gpu.ROCArray.from_host(pos), plan).to_host()
    turns = np.array([[float((Fraction(f) * int(p) / two_pi) % 1) for p in pos] for f in freq])
    c, s = np.cos(2 * np.pi * turns)[:, None], np.sin(2 * np.pi * turns)[:, None]
    a, b = x[: d // 2].astype(np.float64), x[d // 2:].astype(np.float64)
    pair = np.abs(np.concatenate([a, a])) + np.abs(np.concatenate([b, b]))
    angle = 2 * np.pi * np.abs(pos).astype(np.float64)[None, None] * 2.0 ** -65
    ref.within(got, np.concatenate([a * c - b * s, b * c + a * s]), ref.turn_slack(x, d, 1.0, "half") + angle * pair)
