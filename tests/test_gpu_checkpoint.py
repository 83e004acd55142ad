"""8-bit codes, and the activations that keep their inputs in them, against binary64.

Codes and scale bytes are exact by definition and compared bit for bit.  Activations: the
exponential, reciprocal and products of 16-bit results are off by at most 16 U of f's terms (the fast
exponential 2 + 1.17 |u| ulp, and f falls as exp(-|u|) where |u| is large), see ``act_slack``."""
import numpy as np
import pytest

import row_reference as ref
from helpers import Guarded, bits_equal

pytestmark = pytest.mark.gpu
U = ref.U
SHAPES = [(1, 1), (1, 9), (8, 3), (31, 4), (32, 7), (33, 5), (40, 1000), (64, 64), (96, 11), (100, 3), (256, 129), (1000, 7), (1024, 33),
          (4097, 2), (65_536, 1), (100_000, 1), (3, 20_000)]


def values(rng, d, n, dtype, wide):
    x = rng.standard_normal((d, n))
    if wide:                                       # every exponent of the type
        lo, hi = (-24, 15) if dtype == np.float16 else (-140, 126)
        x *= np.ldexp(1.0, rng.integers(lo, hi, (d, n)))
    with np.errstate(over="ignore"):
        x = x.astype(dtype)
    return np.where(np.isfinite(x.astype(np.float64)), x, np.zeros((), dtype)).astype(dtype)


@pytest.mark.parametrize("form", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", list(ref.TYPES))
@pytest.mark.parametrize("wide", [False, True])
def test_codes_and_back(gpu, dtype, form, wide):
    t = ref.TYPES[dtype]
    for d, n in SHAPES:
        x = values(np.random.default_rng(d + n), d, n, t, wide)
        X = gpu.ROCArray.from_host(x)
        codes, scales = Guarded(gpu, np.int8 if form == "int8" else np.uint8, (d, n)), Guarded(gpu, np.uint8, (-(-d // 32), n))
        q = gpu.Quantized8.wrap(codes.array, scales.array)
        gpu.quantize_(q, X)
        c, e = ref.quantize(x.astype(np.float64), form)
        assert np.array_equal(scales.array.to_host(), e), (d, n)
        got = codes.array.to_host()
        same = got == c if form == "int8" else (got == c) | ((got & 0x7F == 0) & (c & 0x7F == 0))     # zeros of either sign
        assert same.all(), (d, n)
        for back in ref.TYPES.values():
            y = Guarded(gpu, back, (d, n))
            gpu.dequantize_(y.array, q)
            ref.within(y.array.to_host(), ref.saturated(ref.restore(got, e), back), 0.0, (d, n, back))
            y.check((d, n))
        codes.check((d, n)); scales.check((d, n))
        again = gpu.quantize(gpu.dequantize(q, np.float32), form)                        # what codes stand for has those codes
        assert np.array_equal(ref.restore(again.codes.to_host(), again.scales.to_host()), ref.restore(got, e))


def test_extremes(gpu):
    """Blocks of zeros, the least and the largest values, ties, infinities and NaN."""
    for form in ("int8", "e4m3"):
        for name, t in ref.TYPES.items():
            info = np.finfo(np.float32) if name == "f32" else __import__("ml_dtypes").finfo(t)
            top, least = float(info.max), float(info.smallest_subnormal)
            x = np.zeros((32 * 8, 1))
            x[32:64] = np.array([top, -top] * 16)[:, None]
            x[64:96, 0] = least
            x[96:128, 0] = np.arange(32) + 0.5                                           # ties where the scale is one
            x[96, 0] = 127.0 if form == "int8" else 448.0
            x[128, 0] = np.nan
            x[160, 0], x[161, 0] = np.inf, 1.0
            x[192:224, 0] = -0.0
            x[224:256, 0] = np.linspace(-1, 1, 32)
            x = x.astype(t)
            q = gpu.quantize(gpu.ROCArray.from_host(x), form)
            c, e = ref.quantize(x.astype(np.float64), form)
            assert np.array_equal(q.scales.to_host(), e) and list(e[[4, 5], 0]) == [255, 255]
            assert np.array_equal(ref.restore(q.codes.to_host(), e), ref.restore(c, e), equal_nan=True)
            y = gpu.dequantize(q, t).to_host().astype(np.float64)
            assert np.isnan(y[128:192]).all() and np.isfinite(np.delete(y, np.s_[128:192])).all()
            assert (np.abs(y[32:64]) <= top).all()
            wide = gpu.quantize(gpu.ROCArray.from_host(np.array([[1e6], [-1e6]], np.float32)), form)
            assert np.array_equal(np.abs(gpu.dequantize(wide, np.float16).to_host()), np.full((2, 1), 65504, np.float16))


def act_slack(f, df, a, exact):
    """Errors of f(a) and f'(a).  Of gelu's argument u the cube's roundings, 5 U |2u|, count times the
    sigmoid's slope, and near a root of f' nothing may be taken relative to it."""
    u = np.abs(a) if f == "silu" else 2 * 0.7978845608 * np.abs(a + 0.044715 * a ** 3)
    with np.errstate(over="ignore", under="ignore"):
        s = np.exp(-np.minimum(u, 700.0)) / (1 + np.exp(-np.minimum(u, 700.0))) ** 2      # slope of the sigmoid
    q = np.where(a >= 0, 1.0, 0.0) + np.where(a >= 0, -1.0, 1.0) * np.exp(-np.minimum(u, 700.0)) / (1 + np.exp(-np.minimum(u, 700.0)))
    du = 1.0 if f == "silu" else 1.6 * (1 + 3 * 0.044715 * a * a)
    rel = (6 if exact else 10) * U + (0 if f == "silu" and exact else 2 * U * u) + (5 * U * u if f == "gelu" else 0)
    tiny = 2.0 ** -148 * (1 + np.abs(a) * du)                                               # exponentials below binary32's normal range
    return np.abs(a) * q * rel + tiny + 2 * U * np.abs(a) * q, (q + np.abs(a) * s * du) * (rel + 8 * U) + tiny


@pytest.mark.parametrize("f", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", list(ref.TYPES))
def test_activations(gpu, dtype, f):
    t = ref.TYPES[dtype]
    for d, n in SHAPES:
        rng = np.random.default_rng(d + n + 7)
        a, b, dy = ((s * rng.standard_normal((d, n))).astype(t) for s in (3.0, 1.0, 1.0))
        a.reshape(-1)[: 9] = np.array([0.0, -0.0, 1e-4, 20.0, -20.0, 90.0, -90.0, 300.0, -300.0])[: a.size].astype(t)
        A, B, DY = (gpu.ROCArray.from_host(v) for v in (a, b, dy))
        a64, b64, dy64 = (v.astype(np.float64) for v in (a, b, dy))
        fa, dfa = ref.act(f, a64)
        sf, sdf = act_slack(f, dfa, a64, t == np.float32)
        Y, DA, DB = (Guarded(gpu, t, (d, n)) for _ in range(3))
        gpu.activation_(f, Y.array, A)
        ref.within(Y.array.to_host(), fa, sf, (d, n, "f"))
        gpu.activation_(f, Y.array, A, B)
        ref.within(Y.array.to_host(), fa * b64, (sf + U * np.abs(fa)) * np.abs(b64), (d, n, "gated"))
        gpu.activation_backward_(f, DA.array, DY, A)
        ref.within(DA.array.to_host(), dy64 * dfa, np.abs(dy64) * (sdf + U * np.abs(dfa)), (d, n, "df"))
        gpu.activation_backward_(f, DA.array, DY, A, B, dgate=DB.array)
        ref.within(DA.array.to_host(), dy64 * b64 * dfa, np.abs(dy64 * b64) * (sdf + 2 * U * np.abs(dfa)), (d, n, "gated df"))
        ref.within(DB.array.to_host(), dy64 * fa, np.abs(dy64) * (sf + U * np.abs(fa)), (d, n, "dgate"))
        for form in ("int8", "e4m3"):
            qa, qb = gpu.Quantized8((d, n), form), gpu.Quantized8((d, n), form)
            gpu.activation_(f, Y.array, A, B, checkpoint=qa, gate_checkpoint=qb)
            ref.within(Y.array.to_host(), fa * b64, (sf + U * np.abs(fa)) * np.abs(b64), (d, n, form))
            kept = []
            for q, v in ((qa, a64), (qb, b64)):
                c, e = ref.quantize(v, form)
                assert np.array_equal(q.scales.to_host(), e) and np.array_equal(ref.restore(q.codes.to_host(), e), ref.restore(c, e)), (d, n, form)
                kept.append(ref.saturated(ref.restore(c, e), t))
            ka, kb = kept
            fk, dfk = ref.act(f, ka)
            sk, sdk = act_slack(f, dfk, ka, t == np.float32)
            gpu.activation_backward_(f, DA.array, DY, qa, qb, dgate=DB.array)
            ref.within(DA.array.to_host(), dy64 * kb * dfk, np.abs(dy64 * kb) * (sdk + 2 * U * np.abs(dfk)), (d, n, form, "gated df"))
            ref.within(DB.array.to_host(), dy64 * fk, np.abs(dy64) * (sk + U * np.abs(fk)), (d, n, form, "dgate"))
            gpu.activation_(f, Y.array, A, checkpoint=qa)
            gpu.activation_backward_(f, DA.array, DY, qa)
            ref.within(DA.array.to_host(), dy64 * dfk, np.abs(dy64) * (sdk + U * np.abs(dfk)), (d, n, form, "df"))
        for g in (Y, DA, DB):
            g.check((d, n))


def test_activation_limits(gpu):
    """silu and gelu run to 0 and a at the infinities, their derivatives to 0 and 1; NaN stays."""
    x = np.array([[np.inf], [-np.inf], [np.nan], [3e38], [-3e38]], np.float32)
    X, one = gpu.ROCArray.from_host(x), gpu.ones(np.float32, (5, 1))
    for f in ("silu", "gelu"):
        y = gpu.activation(f, X).to_host()[:, 0]
        assert y[0] == np.inf and y[1] == 0 and np.isnan(y[2]) and y[3] == np.float32(3e38) and y[4] == 0
        d = gpu.activation_backward_(f, X.similar(), one, X).to_host()[:, 0]
        assert d[0] == 1 and d[1] == 0 and np.isnan(d[2]) and d[3] == 1 and d[4] == 0


def test_layouts_and_aliases(gpu):
    rng = np.random.default_rng(11)
    t = ref.BF16
    for d in (64, 37):
        both = rng.standard_normal((2 * d, 30)).astype(t)                                # one projection, two halves
        P = gpu.ROCArray.from_host(both)
        A, B = P.subview(slice(0, d), slice(None)), P.subview(slice(d, 2 * d), slice(None))
        want = gpu.activation("silu", gpu.ROCArray.from_host(both[:d].copy()), gpu.ROCArray.from_host(both[d:].copy())).to_host()
        qa, qb = gpu.Quantized8((d, 30)), gpu.Quantized8((d, 30))
        y = gpu.activation_("silu", gpu.ROCArray(t, (d, 30)), A, B, checkpoint=qa, gate_checkpoint=qb).to_host()
        assert bits_equal(y, want)
        # both gradients into the halves of one array
        G = gpu.ROCArray(t, (2 * d, 30))
        DY = gpu.ROCArray.from_host(rng.standard_normal((d, 30)).astype(t))
        da, db = gpu.ROCArray(t, (d, 30)), gpu.ROCArray(t, (d, 30))
        gpu.activation_backward_("silu", da, DY, qa, qb, dgate=db)
        gpu.activation_backward_("silu", G.subview(slice(0, d), slice(None)), DY, qa, qb, dgate=G.subview(slice(d, 2 * d), slice(None)))
        assert bits_equal(G.to_host()[:d], da.to_host()) and bits_equal(G.to_host()[d:], db.to_host())
        gpu.activation_backward_("silu", DY, DY, qa, qb, dgate=db)
        assert bits_equal(DY.to_host(), da.to_host())
        # transposed operands go through dense copies
        T = gpu.ROCArray.from_host(np.ascontiguousarray(both[:d].T)).transpose()
        assert bits_equal(gpu.activation_("silu", gpu.ROCArray(t, (30, d)).transpose(), T).to_host(),
                          gpu.activation("silu", gpu.ROCArray.from_host(both[:d].copy())).to_host())
        q = gpu.quantize(T)
        assert bits_equal(q.codes.to_host(), gpu.quantize(gpu.ROCArray.from_host(both[:d].copy())).codes.to_host())
        assert bits_equal(gpu.dequantize_(gpu.ROCArray(t, (30, d)).transpose(), q).to_host(), gpu.dequantize(q, t).to_host())
        x = gpu.ROCArray.from_host(both)
        want = gpu.activation("gelu", x).to_host()
        assert bits_equal(gpu.activation_("gelu", x, x).to_host(), want)
    for dims in ((0,), (0, 4), (4, 0)):
        x = gpu.ROCArray(np.float32, dims)
        assert gpu.activation("silu", x).dims == dims and gpu.dequantize(gpu.quantize(x)).dims == dims
    x = gpu.ROCArray.from_host(rng.standard_normal((33, 4, 5)).astype(np.float32))
    assert gpu.dequantize(gpu.quantize(x, "e4m3")).dims == (33, 4, 5)


@pytest.mark.parametrize("d,n", [(33, 1000), (46, 333), (63, 700), (1023, 50), (40, 513), (2049, 9), (33, 8), (35, 117)])
def test_blocks_across_vectors(gpu, d, n):
    """Dense rows of odd widths: blocks begin and end inside vectors and across the tiles of a launch; codes,
    scale bytes and what comes back stay those of the rows, for every type, and so do both passes."""
    for name, t in ref.TYPES.items():
        rng = np.random.default_rng(d)
        x = values(rng, d, n, t, True)
        x[:, ::3] = values(rng, d, n, t, False)[:, ::3]
        if n > 5:
            x[d // 2, 5], x[d - 1, 3] = np.nan, np.inf
        X, G = gpu.ROCArray.from_host(x), gpu.ROCArray.from_host(np.roll(x, 1, axis=1))
        for form in ("int8", "e4m3"):
            codes, scales = Guarded(gpu, np.int8 if form == "int8" else np.uint8, (d, n)), Guarded(gpu, np.uint8, (-(-d // 32), n))
            q = gpu.Quantized8.wrap(codes.array, scales.array)
            gpu.quantize_(q, X)
            c, e = ref.quantize(x.astype(np.float64), form)
            assert np.array_equal(scales.array.to_host(), e), (name, form)
            assert np.array_equal(ref.restore(codes.array.to_host(), e), ref.restore(c, e), equal_nan=True), (name, form)
            y = Guarded(gpu, t, (d, n))
            gpu.dequantize_(y.array, q)
            ref.within(y.array.to_host(), ref.saturated(ref.restore(c, e), t), 0.0, (name, form))
            y.check(); codes.check(); scales.check()
            qa, qb = gpu.Quantized8((d, n), form), gpu.Quantized8((d, n), form)
            Y = Guarded(gpu, t, (d, n))
            gpu.activation_("silu", Y.array, X, G, checkpoint=qa, gate_checkpoint=qb)
            Y.check()
            assert bits_equal(qa.codes.to_host(), q.codes.to_host()) and bits_equal(qa.scales.to_host(), e)
            assert np.array_equal(qb.scales.to_host(), np.roll(e, 1, axis=1))
            # in place: the same results by the kernel that reads nothing of its neighbours
            Z, qz, qy = X.copy(), gpu.Quantized8((d, n), form), gpu.Quantized8((d, n), form)
            gpu.activation_("silu", Z, Z, G, checkpoint=qz, gate_checkpoint=qy)
            assert np.array_equal(Z.to_host(), Y.array.to_host(), equal_nan=True) and bits_equal(qz.codes.to_host(), qa.codes.to_host())
            assert bits_equal(qy.scales.to_host(), qb.scales.to_host())


@pytest.mark.parametrize("form", ["int8", "e4m3"])
def test_every_code_at_every_scale(gpu, form):
    """All 256 codes beside all 256 scale bytes, those that no call of this library writes among them (Int8
    -128, e4m3 NaN): values past a type's range become its largest, NaN stays NaN."""
    t8 = np.int8 if form == "int8" else np.uint8
    e = np.arange(256, dtype=np.uint8)
    for d in (256, 259):                           # rows of whole vectors, blocks that end inside vectors
        row = np.resize(np.arange(256, dtype=np.uint8), d).view(t8)
        codes, scales = np.repeat(row[:, None], 256, 1), np.repeat(e[None], -(-d // 32), 0)
        q = gpu.Quantized8.wrap(gpu.ROCArray.from_host(codes), gpu.ROCArray.from_host(scales))
        for t in ref.TYPES.values():
            want = ref.saturated(ref.restore(codes, scales), t)
            ref.within(gpu.dequantize(q, t).to_host(), want, 0.0, (d, t))
            off = gpu.ROCArray(t, d * 256 + 1).view(1, d * 256 + 1).reshape(d, 256)       # an element per lane
            ref.within(gpu.dequantize_(off, q).to_host(), want, 0.0, (d, t, "off"))
            side = gpu.Quantized8.wrap(q.codes.reshape(d, 1, 256, 1), q.scales.reshape(-(-d // 32), 1, 256, 1))
            out = [gpu.zeros(t, (d, 1, 256, 1)) for _ in range(2)]
            one = gpu.ROCArray.from_host(np.array([[1]], np.int32))
            gpu.cache_read_(*out, gpu.QuantizedCache(side, side), one, gpu.ROCArray.from_host(np.array([256], np.int32)))
            ref.within(out[0].to_host().reshape(d, 256), want, 0.0, (d, t, "cache"))
            # far out the derivatives are 0 and 1
            far = (np.abs(want) > 1000) | np.isnan(want)
            slope = np.where(np.isnan(want), np.nan, want > 0)
            for f in ("silu", "gelu"):
                got = gpu.activation_backward_(f, gpu.ROCArray(t, (d, 256)), gpu.ones(t, (d, 256)), q).to_host().astype(np.float64)
                assert np.array_equal(got[far], slope[far], equal_nan=True), (d, t, f)
