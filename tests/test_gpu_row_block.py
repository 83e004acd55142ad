"""The row operators together, as a transformer block calls them around its matrix products: norm with
a checkpoint, rotation of queries, keys into the cache and back, gated activation with checkpoints, and
the gradients on the way back; each stage against binary64 at what the stage before it gave, and the
formulas themselves against differences (on the CPU)."""
import numpy as np
import pytest

import row_reference as ref

U = ref.U


def test_formulas_against_differences():
    """d/dt of the forward formulas by central differences in binary64."""
    rng = np.random.default_rng(0)
    x, dy = rng.standard_normal((12, 5)), rng.standard_normal((12, 5))
    gamma, beta = rng.standard_normal(12), rng.standard_normal(12)
    _, mean, rstd, hat = ref.norm(x, gamma, beta, 1e-5)
    dx, dg, db = ref.norm_grad(dy, hat, rstd, gamma)
    h = 1e-6
    loss = lambda x, g, b: (ref.norm(x, g, b, 1e-5)[0] * dy).sum()
    for got, f, shape in ((dx, lambda v: loss(x + v, gamma, beta), x.shape), (dg, lambda v: loss(x, gamma + v, beta), (12,)),
                          (db, lambda v: loss(x, gamma, beta + v), (12,))):
        for i in np.ndindex(shape):
            v = np.zeros(shape)
            v[i] = h
            assert abs((f(v) - f(-v)) / (2 * h) - got[i]) <= 1e-7 * (1 + np.abs(got).max())
    a = np.linspace(-6, 6, 101)
    for f in ("silu", "gelu"):
        d = (ref.act(f, a + h)[0] - ref.act(f, a - h)[0]) / (2 * h)
        assert np.abs(d - ref.act(f, a)[1]).max() <= 1e-8
    x, y = rng.standard_normal((8, 2, 3)), rng.standard_normal((8, 2, 3))
    pos, freq = np.array([0, 7, 123]), [1.0, 0.1, 0.01]
    for layout in ("half", "interleaved"):
        left = (ref.turn(x, pos, freq, 1.3, layout) * y).sum()
        assert abs(left - (x * ref.turn(y, pos, freq, 1.3, layout, True)).sum()) <= 1e-12 * np.abs(x).sum() * 8


@pytest.mark.gpu
def test_gradients_against_differences(gpu):
    """The device's gradients in binary32 against central differences of the formulas in binary64."""
    rng = np.random.default_rng(1)
    d, n = 40, 3
    x, dy = rng.standard_normal((d, n)).astype(np.float32), rng.standard_normal((d, n)).astype(np.float32)
    gamma = rng.standard_normal(d).astype(np.float32)
    X, DY, G = (gpu.ROCArray.from_host(v) for v in (x, dy, gamma))
    M, R = gpu.ROCArray(np.float32, n), gpu.ROCArray(np.float32, n)
    gpu.layernorm_(X.similar(), X, G, mean=M, rstd=R)
    dx, dg, db = (v.to_host() for v in gpu.layernorm_backward(DY, X, G, mean=M, rstd=R))
    zero, h = np.zeros(d), 1e-6
    loss = lambda x, g: (ref.norm(x, g, zero, 1e-5)[0] * dy.astype(np.float64)).sum()
    x64, g64 = x.astype(np.float64), gamma.astype(np.float64)
    for i in np.ndindex(d, n):
        v = np.zeros((d, n))
        v[i] = h
        assert abs((loss(x64 + v, g64) - loss(x64 - v, g64)) / (2 * h) - dx[i]) <= 1e-5 * (1 + np.abs(dx).max())
    for i in range(d):
        v = np.zeros(d)
        v[i] = h
        assert abs((loss(x64, g64 + v) - loss(x64, g64 - v)) / (2 * h) - dg[i]) <= 1e-5 * (1 + np.abs(dg).max())
    assert np.abs(db - dy.astype(np.float64).sum(1)).max() <= 4 * U * np.abs(dy).sum(1).max()


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["int8", "e4m3"])
def test_block(gpu, form):
    rng = np.random.default_rng(7)
    t = ref.BF16
    d_head, heads, n, page = 64, 4, 37, 16
    d = d_head * heads
    x = (rng.standard_normal((d, n)) + 0.5).astype(t)
    gamma, beta = (1 + 0.1 * rng.standard_normal(d)).astype(t), (0.1 * rng.standard_normal(d)).astype(t)
    X, G, B = (gpu.ROCArray.from_host(v) for v in (x, gamma, beta))
    # norm
    kept, R, Y = gpu.Quantized8((d, n), form), gpu.ROCArray(np.float32, n), X.similar()
    gpu.layernorm_(Y, X, G, B, rstd=R, checkpoint=kept)
    y = Y.to_host()
    want, _, rstd, hat = ref.norm(x.astype(np.float64), gamma.astype(np.float64), beta.astype(np.float64), 1e-5)
    ref.within(y, want, 60 * U * (2 + np.abs(want)), "norm")
    # queries turned, keys (here: the same heads) turned into the cache and read back
    Q = Y.reshape(d_head, heads, n)
    plan = gpu.rotary_plan(d_head)
    freq, _ = gpu.rotary.rotary_frequencies(d_head)
    pos = np.arange(100, 100 + n)
    P = gpu.ROCArray.from_host(pos.astype(np.int32))
    Qt = gpu.rotary_(Q.similar(), Q, P, plan)
    q = y.reshape(d_head, heads, n, order="F")
    turned = ref.turn(q, pos, freq, 1.0, "half")
    ref.within(Qt.to_host(), turned, ref.turn_slack(q, d_head, 1.0, "half"), "rotary")
    cache = gpu.quantized_cache(d_head, heads, page, 4, form)
    table = np.array([[3], [1], [4]], np.int32)
    l = np.arange(n)
    slots = (table[l // page, 0] - 1) * page + l % page + 1
    gpu.cache_write_(cache, Q, Q, gpu.ROCArray.from_host(slots.astype(np.int32)), rotary=plan, positions=P)
    Kr, Vr = gpu.zeros(t, (d_head, heads, n, 1)), gpu.zeros(t, (d_head, heads, n, 1))
    gpu.cache_read_(Kr, Vr, cache, gpu.ROCArray.from_host(table), gpu.ROCArray.from_host(np.array([n], np.int32)))
    ref.within(Vr.to_host()[..., 0], ref.restore(*ref.quantize(q.astype(np.float64), form)), 0.0, "values")
    scale = np.repeat(np.ldexp(1.0, ref.exponents(turned, form).astype(int) - 127), 32, 0)
    off = ref.turn_slack(q, d_head, 1.0, "half")
    half = 0.5 * scale if form == "int8" else np.maximum(2.0 ** -4 * (np.abs(turned) + off), 2.0 ** -10 * scale)
    assert (np.abs(Kr.to_host()[..., 0].astype(np.float64) - turned) <= (half + off) * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(turned)).all()
    # gated activation of the read-back values and the turned queries, both kept
    A, Bg = Vr.reshape(d, n), Qt.reshape(d, n)
    ka, kb = gpu.Quantized8((d, n), form), gpu.Quantized8((d, n), form)
    Z = gpu.activation_("silu", X.similar(), A, Bg, checkpoint=ka, gate_checkpoint=kb)
    a, b = A.to_host().astype(np.float64), Bg.to_host().astype(np.float64)
    f, _ = ref.act("silu", a)
    ref.within(Z.to_host(), f * b, 40 * U * np.abs(a * b) + 1e-30, "gated")
    # back: through the activation, the rotation, the norm
    dz = rng.standard_normal((d, n)).astype(t)
    DA, DB = X.similar(), X.similar()
    gpu.activation_backward_("silu", DA, gpu.ROCArray.from_host(dz), ka, kb, dgate=DB)
    ra, rb = (ref.restore(*ref.quantize(v, form)) for v in (a, b))
    fk, dfk = ref.act("silu", ra)
    dz64 = dz.astype(np.float64)
    ref.within(DA.to_host(), dz64 * rb * dfk, 40 * U * np.abs(dz64 * rb) * (1 + np.abs(ra)), "dA")
    ref.within(DB.to_host(), dz64 * fk, 40 * U * np.abs(dz64 * ra) + 1e-30, "dgate")
    DQ = DB.reshape(d_head, heads, n)
    dq = DQ.to_host()
    DQt = gpu.rotary_(DQ.similar(), DQ, P, plan, adjoint=True)
    ref.within(DQt.to_host(), ref.turn(dq, pos, freq, 1.0, "half", True), ref.turn_slack(dq, d_head, 1.0, "half"), "adjoint")
    DY = DQt.reshape(d, n)
    DX, DG, DBt = gpu.layernorm_backward(DY, kept, G, rstd=R)
    dy = DY.to_host().astype(np.float64)
    h = ref.restore(kept.codes.to_host(), kept.scales.to_host())
    dx, dg, db = ref.norm_grad(dy, h, R.to_host().astype(np.float64), gamma.astype(np.float64))
    g = np.abs(dy * gamma.astype(np.float64)[:, None])
    ref.within(DX.to_host(), dx, 60 * U * rstd * (g + g.mean(0) + np.abs(h) * (g * np.abs(h)).mean(0)), "dx")
    ref.within(DG.to_host(), dg, (n + 16) * U * np.abs(dy * h).sum(1), "dgamma")
    ref.within(DBt.to_host(), db, (n + 16) * U * np.abs(dy).sum(1), "dbeta")
    gpu.synchronize()
