"""Row operators without a device: refusals of the C entry points (arguments are checked before the
stream is looked at), of the Python layer, and the host-side arithmetic of the rotary plans."""
import math

import numpy as np
import pytest


class _FakeBuffer:
    """Stands in for pool memory: descriptors are checked, nothing is read."""
    ptr, freed, stream, device = 1 << 20, False, None, 0


def fake(pkg, dtype, dims, offset=0, strides=None):
    return pkg.ROCArray(dtype, dims, _buf=_FakeBuffer(), _offset=offset, _strides=strides)


def status(pkg, name, *args):
    """Status and text of a C call without a stream: valid arguments get as far as the null handle."""
    L = pkg._lib
    refs = [a._ref() if isinstance(a, pkg.ROCArray) else a for a in args]
    code = getattr(L.lib, name)(None, *refs)
    return code, L.last_error()


def assert_valid(pkg, name, *args):
    code, text = status(pkg, name, *args)
    assert code == pkg._lib.INVALID_ARG and "null stream" in text, (code, text)


def assert_refused(pkg, code, part, name, *args):
    got, text = status(pkg, name, *args)
    assert got == code and part in text, (got, text)


def test_layernorm_arguments(pkg):
    L, f = pkg._lib, lambda *a, **k: fake(pkg, *a, **k)
    x, y = f(np.float32, (64, 5)), f(np.float32, (64, 5))
    g, m = f(np.float32, (64,)), f(np.float32, (5,))
    q, s = f(np.int8, (64, 5)), f(np.uint8, (2, 5))
    call = lambda Y, X, lead=1, gam=None, bet=None, eps=1e-5, mean=None, rstd=None, Q=None, S=None: (Y, X, lead, gam, bet, eps, mean, rstd, Q, S)
    assert_valid(pkg, "b200_layernorm", *call(y, x, 1, g, g, 0.0, m, m, q, s))
    assert_valid(pkg, "b200_layernorm", *call(x, x))
    no = lambda code, part, *a, **k: assert_refused(pkg, code, part, "b200_layernorm", *call(*a, **k))
    no(L.INVALID_ARG, "differ in shape", f(np.float32, (64, 6)), x)
    no(L.INVALID_ARG, "element type", f(np.float16, (64, 5)), x)
    no(L.UNSUPPORTED, "Float16, BFloat16 or Float32", f(np.float64, (64, 5)), f(np.float64, (64, 5)))
    no(L.INVALID_ARG, "at least 3 dimensions", y, x, 3)
    no(L.INVALID_ARG, "at least one dimension", y, x, 0)
    no(L.INVALID_ARG, "one value per element", y, x, 1, f(np.float32, (63,)))
    no(L.UNSUPPORTED, "Float32 or of the rows' type", y, x, 1, f(np.float16, (64,)))
    no(L.INVALID_ARG, "one element type", f(np.float16, (64, 5)), f(np.float16, (64, 5)), 1, g, f(np.float16, (64,)))
    no(L.INVALID_ARG, "eps", y, x, eps=-1.0)
    no(L.INVALID_ARG, "eps", y, x, eps=float("nan"))
    no(L.INVALID_ARG, "one value per row", y, x, mean=f(np.float32, (4,)))
    no(L.UNSUPPORTED, "must be Float32", y, x, rstd=f(np.float16, (5,)))
    no(L.INVALID_ARG, "belong together", y, x, Q=q)
    no(L.INVALID_ARG, "one byte per 32", y, x, Q=q, S=f(np.uint8, (3, 5)))
    no(L.UNSUPPORTED, "codes are Int8", y, x, Q=f(np.int16, (64, 5)), S=s)
    no(L.INVALID_ARG, "differs in shape", y, x, Q=f(np.int8, (64, 4)), S=f(np.uint8, (2, 4)))
    no(L.UNSUPPORTED, "along the first dimension", y, x, 2, Q=q, S=s)
    no(L.INVALID_ARG, "overlap", f(np.float32, (64, 5), strides=(1, 32)), x)
    no(L.UNSUPPORTED, "neighbours", y, f(np.float32, (64, 5), strides=(2, 128)))
    no(L.UNSUPPORTED, "collapse", f(np.float32, (8, 4, 5)), f(np.float32, (8, 4, 5), strides=(1, 8, 64)))
    no(L.INVALID_ARG, "null tensor", None, x)
    no(L.INVALID_ARG, "aligned", y, f(np.float32, (64, 5), offset=2))


def test_layernorm_backward_arguments(pkg):
    L, f = pkg._lib, lambda *a, **k: fake(pkg, *a, **k)
    x = f(np.float16, (96, 7))
    g, m = f(np.float32, (96,)), f(np.float32, (7,))
    q, s = f(np.uint8, (96, 7)), f(np.uint8, (3, 7))
    call = lambda dX=x, dg=None, db=None, dY=x, lead=1, X=x, Q=None, S=None, gam=g, mean=m, rstd=m: (dX, dg, db, dY, lead, X, Q, S, gam, mean, rstd)
    assert_valid(pkg, "b200_layernorm_backward", *call(dg=g, db=g))
    assert_valid(pkg, "b200_layernorm_backward", *call(X=None, Q=q, S=s, mean=None))
    no = lambda code, part, **k: assert_refused(pkg, code, part, "b200_layernorm_backward", *call(**k))
    no(L.INVALID_ARG, "no gradient", dX=None)
    no(L.INVALID_ARG, "one of the two", Q=q, S=s)
    no(L.INVALID_ARG, "one of the two", X=None)
    no(L.INVALID_ARG, "needs rstd", rstd=None)
    no(L.INVALID_ARG, "needs the mean", mean=None)
    no(L.INVALID_ARG, "one element type", dg=f(np.float16, (96,)))
    no(L.INVALID_ARG, "source and dY", X=f(np.float32, (96, 7)))
    no(L.INVALID_ARG, "dX and dY", dX=f(np.float16, (96, 8)))
    no(L.INVALID_ARG, "one value per element", db=f(np.float32, (95,)))


def test_checkpoint_arguments(pkg):
    L, f = pkg._lib, lambda *a, **k: fake(pkg, *a, **k)
    x, y = f(np.float32, (40, 3)), f(np.float32, (40, 3))
    q, s, q8, s8 = f(np.int8, (40, 3)), f(np.uint8, (2, 3)), f(np.uint8, (40, 3)), f(np.uint8, (2, 3))
    assert_valid(pkg, "b200_quantize", q, s, x)
    assert_valid(pkg, "b200_dequantize", x, q8, s8)
    assert_refused(pkg, L.INVALID_ARG, "differs in shape", "b200_quantize", f(np.int8, (40, 4)), f(np.uint8, (2, 4)), x)
    assert_refused(pkg, L.UNSUPPORTED, "must be dense", "b200_quantize", f(np.int8, (40, 3), strides=(1, 48)), s, x)
    assert_refused(pkg, L.UNSUPPORTED, "Float16, BFloat16 or Float32", "b200_quantize", q, s, f(np.float64, (40, 3)))
    assert_refused(pkg, L.UNSUPPORTED, "scales are UInt8", "b200_quantize", q, f(np.int8, (2, 3)), x)
    act = "b200_activation"
    assert_valid(pkg, act, 0, y, x, None, q, s, None, None)
    assert_valid(pkg, act, 1, y, x, x, q, s, q, s)
    assert_refused(pkg, L.UNSUPPORTED, "silu", act, 2, y, x, None, None, None, None, None)
    assert_refused(pkg, L.INVALID_ARG, "no gate", act, 0, y, x, None, None, None, q, s)
    assert_refused(pkg, L.INVALID_ARG, "belong together", act, 0, y, x, None, q, None, None, None)
    assert_refused(pkg, L.INVALID_ARG, "one format", act, 0, y, x, x, q, s, q8, s8)
    assert_refused(pkg, L.INVALID_ARG, "differ in element type", act, 0, f(np.float16, (40, 3)), x, None, None, None, None, None)
    back = "b200_activation_backward"
    assert_valid(pkg, back, 0, y, None, x, x, None, None, None, None, None)
    assert_valid(pkg, back, 0, y, y, x, None, None, q, s, q, s)
    assert_refused(pkg, L.INVALID_ARG, "one of the two", back, 0, y, None, x, x, None, q, s, None, None)
    assert_refused(pkg, L.INVALID_ARG, "one of the two", back, 0, y, None, x, None, None, None, None, None, None)
    assert_refused(pkg, L.INVALID_ARG, "needs dB", back, 0, y, y, x, x, None, None, None, q, s)
    assert_refused(pkg, L.INVALID_ARG, "needs dB", back, 0, y, None, x, None, None, q, s, q, s)
    with pytest.raises(ValueError):
        pkg.activation_("tanh", y, x)
    with pytest.raises(ValueError):
        pkg.activation_backward_("silu", y, x, x, gate=x)
    with pytest.raises(ValueError):
        pkg.Quantized8.wrap(q, f(np.uint8, (1, 3)))
    with pytest.raises(ValueError):
        pkg.Quantized8((4, 4), "fp4")


def test_rotary_arguments(pkg):
    L, f = pkg._lib, lambda *a, **k: fake(pkg, *a, **k)
    x, t, p = f(np.float16, (64, 4, 9)), f(np.uint64, (32,)), f(np.int32, (9,))
    call = lambda Y=x, X=x, pos=p, table=t, layout=0, factor=1.0, adjoint=0: (Y, X, pos, table, layout, factor, adjoint)
    assert_valid(pkg, "b200_rotary", *call())
    assert_valid(pkg, "b200_rotary", *call(Y=f(np.float16, (64, 4, 9, 2)), X=f(np.float16, (64, 4, 9, 2), strides=(1, 64, 512, 9000)), pos=f(np.int64, (9, 2))))
    no = lambda code, part, **k: assert_refused(pkg, code, part, "b200_rotary", *call(**k))
    no(L.INVALID_ARG, "head size, heads", X=f(np.float16, (64, 4)), Y=f(np.float16, (64, 4)))
    no(L.INVALID_ARG, "differ", Y=f(np.float32, (64, 4, 9)))
    no(L.INVALID_ARG, "more elements than a head", table=f(np.uint64, (33,)))
    no(L.INVALID_ARG, "one position per token", pos=f(np.int32, (8,)))
    no(L.UNSUPPORTED, "Int32 or Int64", pos=f(np.float32, (9,)))
    no(L.UNSUPPORTED, "UInt64", table=f(np.int64, (32,)))
    no(L.UNSUPPORTED, "layout", layout=2)
    no(L.UNSUPPORTED, "neighbours", X=f(np.float16, (64, 4, 9), strides=(4, 1, 256)))
    no(L.INVALID_ARG, "overlap", Y=f(np.float16, (64, 4, 9), strides=(1, 32, 256)))
    no(L.UNSUPPORTED, "Float16, BFloat16", X=f(np.float64, (64, 4, 9)), Y=f(np.float64, (64, 4, 9)))


def test_cache_arguments(pkg):
    L, f = pkg._lib, lambda *a, **k: fake(pkg, *a, **k)
    kq, ks = f(np.int8, (64, 2, 16, 5)), f(np.uint8, (2, 2, 16, 5))
    vq, vs = f(np.int8, (40, 2, 16, 5)), f(np.uint8, (2, 2, 16, 5))
    k, v, sl = f(np.float32, (64, 2, 7)), f(np.float32, (40, 2, 7)), f(np.int64, (7,))
    t = f(np.uint64, (32,))
    call = lambda KQ=kq, KS=ks, VQ=vq, VS=vs, K=k, V=v, slots=sl, pos=None, table=None, layout=0: (KQ, KS, VQ, VS, K, V, slots, pos, table, layout, 1.0)
    assert_valid(pkg, "b200_cache_write", *call())
    assert_valid(pkg, "b200_cache_write", *call(pos=sl, table=t))
    no = lambda code, part, **kw: assert_refused(pkg, code, part, "b200_cache_write", *call(**kw))
    no(L.INVALID_ARG, "head size or heads", K=f(np.float32, (64, 3, 7)))
    no(L.INVALID_ARG, "differ in tokens", V=f(np.float32, (40, 2, 8)))
    no(L.INVALID_ARG, "keys and values differ in element type", V=f(np.float16, (40, 2, 7)))
    no(L.INVALID_ARG, "needs 7 entries", slots=f(np.int64, (6,)))
    no(L.UNSUPPORTED, "Int32 or Int64", slots=f(np.float32, (7,)))
    no(L.INVALID_ARG, "belong together", pos=sl)
    no(L.INVALID_ARG, "more elements than a head", pos=sl, table=f(np.uint64, (33,)))
    no(L.UNSUPPORTED, "layout", pos=sl, table=t, layout=3)
    no(L.INVALID_ARG, "one byte per 32", KS=f(np.uint8, (1, 2, 16, 5)))
    no(L.INVALID_ARG, "differ in heads", VQ=f(np.int8, (40, 2, 8, 5)), VS=f(np.uint8, (2, 2, 8, 5)))
    no(L.INVALID_ARG, "format", VQ=f(np.uint8, (40, 2, 16, 5)))
    no(L.INVALID_ARG, "overlap", KQ=f(np.int8, (64, 2, 16, 5), strides=(1, 32, 128, 2048)))
    no(L.UNSUPPORTED, "neighbours", KQ=f(np.int8, (64, 2, 16, 5), strides=(2, 128, 256, 4096)))
    K, V = f(np.float16, (64, 2, 30, 3)), f(np.float16, (40, 2, 30, 3))
    pages, ln = f(np.int32, (2, 3)), f(np.int32, (3,))
    assert_valid(pkg, "b200_cache_read", K, V, kq, ks, vq, vs, pages, ln)
    assert_refused(pkg, L.INVALID_ARG, "page table", "b200_cache_read", K, V, kq, ks, vq, vs, f(np.int32, (2, 4)), ln)
    assert_refused(pkg, L.INVALID_ARG, "needs 3 entries", "b200_cache_read", K, V, kq, ks, vq, vs, pages, f(np.int32, (2,)))
    assert_refused(pkg, L.INVALID_ARG, "places or sequences", "b200_cache_read", K, f(np.float16, (40, 2, 31, 3)), kq, ks, vq, vs, pages, ln)
    with pytest.raises(ValueError):
        pkg.QuantizedCache(pkg.Quantized8.wrap(kq, ks), pkg.Quantized8.wrap(f(np.uint8, (40, 2, 16, 5)), vs))
    with pytest.raises(ValueError):
        pkg.cache_write_(pkg.QuantizedCache(pkg.Quantized8.wrap(kq, ks), pkg.Quantized8.wrap(vq, vs)), k, v, sl, positions=sl)


def test_cache_scales_that_overlap(pkg):
    """Scale bytes of two heads, places or pages in one place are refused like codes are."""
    f = lambda *a, **k: fake(pkg, *a, **k)
    k, sl = f(np.float32, (64, 2, 7)), f(np.int64, (7,))
    q, s = f(np.int8, (64, 2, 16, 5)), f(np.uint8, (2, 2, 16, 5))
    assert_valid(pkg, "b200_cache_write", q, s, q, s, k, k, sl, None, None, 0, 1.0)
    for strides in ((1, 0, 4, 64), (1, 1, 4, 64), (1, 2, 0, 64), (1, 2, 4, 1)):
        bad = f(np.uint8, (2, 2, 16, 5), strides=strides)
        assert_refused(pkg, pkg._lib.INVALID_ARG, "overlap", "b200_cache_write", q, bad, q, s, k, k, sl, None, None, 0, 1.0)
        assert_refused(pkg, pkg._lib.INVALID_ARG, "overlap", "b200_cache_write", q, s, q, bad, k, k, sl, None, None, 0, 1.0)


def test_python_checks(pkg):
    f = lambda *a, **k: fake(pkg, *a, **k)
    x = f(np.float32, (8, 3))
    for bad in (lambda: pkg.layernorm_(f(np.float32, (8, 4)), x),
                lambda: pkg.layernorm_(x, x, f(np.float32, (7,))),
                lambda: pkg.layernorm_(x, x, lead=3),
                lambda: pkg.layernorm_(x, x, f(np.float32, (8,)), lead=2),
                lambda: pkg.layernorm_backward_(x, x, x, rstd=x),
                lambda: pkg.layernorm_backward_(f(np.float16, (8, 3)), x, x, rstd=x, mean=x),
                lambda: pkg.rotary_(x, f(np.float32, (8, 4)), x, None),
                lambda: pkg.rotary_plan(7), lambda: pkg.rotary_plan(8, layout="third"),
                lambda: pkg.rotary_plan(8, scaling="square"), lambda: pkg.rotary_plan(8, scaling="yarn", stretch=2.0)):
        with pytest.raises(ValueError):
            bad()
    class Other:                                   # a stream of another device than the arrays'
        device, handle = 1, None
    with pytest.raises(ValueError, match="device"):
        pkg.layernorm_(x, x, stream=Other())


def test_row_views_that_need_no_copy(pkg):
    f = lambda dims, strides: fake(pkg, np.float32, dims, strides=strides)
    rows = pkg.quantization.is_rows
    assert rows(f((8, 3), (1, 8)), 1) and rows(f((8, 3), (1, 20)), 1) and rows(f((8, 3), (1, 0)), 1)
    assert rows(f((8, 3, 4), (1, 20, 60)), 1) and not rows(f((8, 3, 4), (1, 20, 80)), 1)
    assert rows(f((8, 3, 4), (1, 8, 30)), 2) and not rows(f((8, 3, 4), (1, 9, 30)), 2)
    assert not rows(f((8, 3), (3, 1)), 1) and rows(f((1, 3), (3, 1)), 1) and rows(f((8, 1, 4), (1, 77, 16)), 1)


def test_rotary_frequencies(pkg):
    freq = pkg.rotary.rotary_frequencies
    f, m = freq(8)
    assert m == 1.0 and np.allclose(f, [1.0, 0.1, 0.01, 0.001], rtol=1e-14)
    assert np.allclose(freq(8, scaling="linear", stretch=4.0)[0], np.array(f) / 4, rtol=1e-14)
    # "ntk" leaves the first pair and interpolates the last in full
    n = freq(8, scaling="ntk", stretch=4.0)[0]
    assert n[0] == 1.0 and math.isclose(n[-1], f[-1] / 4, rel_tol=1e-12)
    y, m = freq(64, scaling="yarn", stretch=8.0, original_length=4096)
    f = freq(64)[0]
    assert math.isclose(m, 0.1 * math.log(8.0) + 1.0)
    for a, b in zip(y, f):
        turns = 4096 * b / (2 * math.pi)
        if turns >= 32:
            assert a == b
        elif turns <= 1:
            assert math.isclose(a, b / 8, rel_tol=1e-12)
        else:
            assert b / 8 < a < b


class _OtherDevice:
    """A stream of another device than the arrays'."""
    device, handle = 1, None


def test_arrays_of_another_device(pkg):
    """Refused whatever stream used them last (a copy between devices leaves them with the destination's), and
    before a stand-in or a dense copy is made of arrays whose strides are not those of rows."""
    st = _OtherDevice()

    def lent(dtype, dims, strides=None):
        a = fake(pkg, dtype, dims, strides=strides)
        a.buf.stream = st                          # as after copyto_ on that stream
        return a
    f32 = np.float32
    for make in (lambda *a, **k: fake(pkg, *a, **k), lent):
        x, s = make(f32, (32, 6)), make(f32, (32, 6), strides=(6, 1))
        q = pkg.Quantized8.wrap(make(np.int8, (32, 6)), make(np.uint8, (1, 6)))
        m, i = make(f32, (6,)), make(np.int32, (3,))
        h, hs = make(f32, (32, 2, 3)), make(f32, (32, 2, 3), strides=(6, 3, 1))
        side = pkg.Quantized8.wrap(make(np.int8, (32, 2, 4, 5)), make(np.uint8, (1, 2, 4, 5)))
        cache = pkg.QuantizedCache(side, side)
        plan = object.__new__(pkg.RotaryPlan)
        plan.table, plan.layout, plan._layout, plan.factor = make(np.uint64, (16,)), "half", 0, 1.0
        for v in (x, s):
            for call in (lambda: pkg.layernorm_(v, x, stream=st), lambda: pkg.layernorm_(x, v, stream=st),
                         lambda: pkg.layernorm_backward_(x, v, x, rstd=m, mean=m, stream=st),
                         lambda: pkg.layernorm_backward_(v, x, q, rstd=m, stream=st),
                         lambda: pkg.activation_("silu", v, x, stream=st), lambda: pkg.activation_("silu", x, x, v, stream=st),
                         lambda: pkg.activation_backward_("gelu", v, x, q, stream=st),
                         lambda: pkg.activation_backward_("gelu", x, x, x, v, dgate=x, stream=st),
                         lambda: pkg.quantize_(q, v, stream=st), lambda: pkg.dequantize_(v, q, stream=st)):
                with pytest.raises(ValueError, match="device"):
                    call()
        for v in (h, hs):
            for call in (lambda: pkg.rotary_(h, v, i, plan, stream=st), lambda: pkg.cache_write_(cache, v, h, i, stream=st),
                         lambda: pkg.cache_write_(cache, h, v, i, stream=st)):
                with pytest.raises(ValueError, match="device"):
                    call()


def test_rotary_table_is_exact(pkg, monkeypatch):
    """Entries are the frequencies, as binary64 has them, in 2^-64 turns, rounded once: no error but that
    rounding is multiplied by a position."""
    from fractions import Fraction
    from decimal import Decimal, localcontext
    with localcontext() as ctx:                    # pi by Machin's formula, in decimals
        ctx.prec = 700

        def arctan(n):
            term, total, k = Decimal(1) / n, Decimal(0), 0
            while abs(term) > Decimal(10) ** -690:
                total += term / (2 * k + 1) * (-1) ** k
                term /= n * n
                k += 1
            return total
        two_pi = Fraction(8 * (4 * arctan(5) - arctan(239)))
    tables = []

    class Kept:
        @staticmethod
        def from_host(a, stream=None):
            tables.append(a)
    monkeypatch.setattr(pkg.rotary, "ROCArray", Kept)
    sets = [pkg.rotary.rotary_frequencies(128)[0], pkg.rotary.rotary_frequencies(64, base=1e6, scaling="yarn", stretch=8.0, original_length=4096)[0],
            [0.0, 1.0, -1.0, 2.0 * math.pi, 5e-324, 1e-30, -0.1, 1e22, 1.7976931348623157e308]]
    for f in sets:
        pkg.RotaryPlan(f)
        assert tables[-1].dtype == np.uint64
        for got, x in zip(tables[-1], f):
            turns = Fraction(x) / two_pi * (1 << 64)
            off = (int(got) - turns) % (1 << 64)
            assert min(off, (1 << 64) - off) <= Fraction(1, 2) + Fraction(1, 1 << 60), x


def test_rotary_frequencies_of_any_iterable(pkg, monkeypatch):
    """A generator is gone through once: its frequencies are looked at and kept."""
    tables = []

    class Kept:
        @staticmethod
        def from_host(a, stream=None):
            tables.append(a)
    monkeypatch.setattr(pkg.rotary, "ROCArray", Kept)
    f = pkg.rotary.rotary_frequencies(16)[0]
    for given in (f, tuple(f), np.array(f), (x for x in f)):
        pkg.RotaryPlan(given)
        assert np.array_equal(tables[-1], tables[0]) and len(tables[-1]) == 8
    with pytest.raises(ValueError, match="finite"):
        pkg.RotaryPlan(x for x in (1.0, math.inf))
