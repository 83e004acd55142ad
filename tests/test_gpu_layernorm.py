"""Layer norm, its gradient and its 8-bit checkpoint against binary64 (tests/row_reference.py).

Tolerances: half a step of the stored type, plus the roundings of the binary32 sums counted in
``norm_steps``: a sum of a row is off by at most n U sum|terms|, the root by half of what the
variance is off."""
import numpy as np
import pytest

import row_reference as ref
from helpers import Guarded, bits_equal

pytestmark = pytest.mark.gpu
U = ref.U
EPS = 1e-5


def rows(rng, d, n, dtype, offset=0.4, wide=True):
    x = rng.standard_normal((d, n)) * (0.5 + rng.random((1, n))) + offset
    if wide and d > 4:
        x[:: max(1, d // 5)] *= 6.0
    return x.astype(dtype)


def params(rng, d, dtype):
    return (1.0 + 0.3 * rng.standard_normal(d)).astype(dtype), (0.2 * rng.standard_normal(d)).astype(dtype)


def forward_slack(x, gamma, beta, mean, rstd, hat):
    n = ref.norm_steps(x.shape[0])
    h = n * U * np.abs(hat) + (n + 1) * U * np.abs(x).mean(0) * rstd
    return np.abs(gamma)[:, None] * h + 2 * U * (np.abs(gamma[:, None] * hat) + np.abs(beta)[:, None])


def check_forward(gpu, x, gamma, beta, Y, M, R, eps=EPS, what=""):
    x64 = x.astype(np.float64)
    g = np.ones(x.shape[0]) if gamma is None else gamma.astype(np.float64)
    b = np.zeros(x.shape[0]) if beta is None else beta.astype(np.float64)
    y, mean, rstd, hat = ref.norm(x64, g, b, eps)
    n = ref.norm_steps(x.shape[0])
    ref.within(Y, y, forward_slack(x64, g, b, mean, rstd, hat), (what, "y"))
    ref.within(M, mean, n * U * np.abs(x64).mean(0), (what, "mean"))
    # the variance is off by the squares' roundings and, to first order not at all, by the mean's
    ref.within(R, rstd, (n + 4) * U * rstd, (what, "rstd"))
    return mean, rstd, hat


def check_backward(x_hat, rstd, dy, gamma, dX, dG, dB, hat_slack, what=""):
    d, n = x_hat.shape
    g64 = np.ones(d) if gamma is None else gamma.astype(np.float64)
    dy64 = dy.astype(np.float64)
    dx, dg, db = ref.norm_grad(dy64, x_hat, rstd, g64)
    g = dy64 * g64[:, None]
    k = ref.norm_steps(d) + 4
    mg, mgh = np.abs(g).mean(0), np.abs(g * x_hat).mean(0)
    c2 = np.abs((g * x_hat).mean(0))
    slack = rstd * (k * U * (np.abs(g) + mg + np.abs(x_hat) * mgh) + hat_slack * c2 + np.abs(x_hat) * (np.abs(g) * hat_slack).mean(0))
    if dX is not None:
        ref.within(dX, dx, slack + 4 * U * np.abs(dx), (what, "dx"))
    # sums over the rows: no more roundings than rows, and the fold of the blocks' partials
    k = n + 16
    if dG is not None:
        ref.within(dG, dg, (k * U * np.abs(dy64 * x_hat) + np.abs(dy64) * hat_slack).sum(1), (what, "dgamma"))
    if dB is not None:
        ref.within(dB, db, (k * U * np.abs(dy64)).sum(1), (what, "dbeta"))


SHAPES = [(1, 1), (1, 40), (7, 3), (8, 5), (31, 9), (32, 1), (33, 100), (64, 300), (100, 17), (128, 1), (256, 33), (513, 12), (768, 70),
          (1000, 5), (1023, 21), (1024, 8), (2047, 6), (2048, 16), (4096, 5), (5000, 3), (5120, 4), (8192, 3), (8193, 2), (8200, 3),
          (10_000, 2), (16_384, 2), (16_385, 1), (40_000, 2)]


@pytest.mark.parametrize("dtype", list(ref.TYPES))
@pytest.mark.parametrize("pf32", [True, False])
def test_forward_and_gradient(gpu, dtype, pf32):
    t = ref.TYPES[dtype]
    p = np.dtype(np.float32) if pf32 else t
    for d, n in SHAPES:
        rng = np.random.default_rng(d * 1000 + n)
        x, dy = rows(rng, d, n, t), rng.standard_normal((d, n)).astype(t)
        gamma, beta = params(rng, d, p)
        X, G, B, DY = (gpu.ROCArray.from_host(a) for a in (x, gamma, beta, dy))
        Y, M, R = Guarded(gpu, t, (d, n)), Guarded(gpu, np.float32, n), Guarded(gpu, np.float32, n)
        gpu.layernorm_(Y.array, X, G, B, eps=EPS, mean=M.array, rstd=R.array)
        check_forward(gpu, x, gamma, beta, Y.array.to_host(), M.array.to_host(), R.array.to_host(), what=(d, n))
        # the gradient at the moments that the forward pass gave
        mean, rstd = M.array.to_host().astype(np.float64), R.array.to_host().astype(np.float64)
        hat = (x.astype(np.float64) - mean) * rstd
        DX, DG, DB = Guarded(gpu, t, (d, n)), Guarded(gpu, p, d), Guarded(gpu, p, d)
        gpu.layernorm_backward_(DX.array, DY, X, G, mean=M.array, rstd=R.array, dgamma=DG.array, dbeta=DB.array)
        check_backward(hat, rstd, dy, gamma, DX.array.to_host(), DG.array.to_host(), DB.array.to_host(),
                       2 * U * np.abs(hat), (d, n))
        for g in (Y, M, R, DX, DG, DB):
            g.check((d, n))
    gpu.synchronize()


@pytest.mark.parametrize("form", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", list(ref.TYPES))
def test_checkpoint(gpu, dtype, form):
    """The forward pass's codes stand for the normalised rows to half a code, and the gradient taken
    from them is the formula's at what they stand for."""
    t = ref.TYPES[dtype]
    for d, n in SHAPES:
        rng = np.random.default_rng(d * 1000 + n + 1)
        x, dy = rows(rng, d, n, t), rng.standard_normal((d, n)).astype(t)
        gamma, beta = params(rng, d, t)
        X, G, B, DY = (gpu.ROCArray.from_host(a) for a in (x, gamma, beta, dy))
        codes, scales = Guarded(gpu, np.int8 if form == "int8" else np.uint8, (d, n)), Guarded(gpu, np.uint8, (-(-d // 32), n))
        q = gpu.Quantized8.wrap(codes.array, scales.array)
        Y, M, R = gpu.ROCArray(t, (d, n)), gpu.ROCArray(np.float32, n), gpu.ROCArray(np.float32, n)
        gpu.layernorm_(Y, X, G, B, eps=EPS, mean=M, rstd=R, checkpoint=q)
        mean, rstd, hat = check_forward(gpu, x, gamma, beta, Y.to_host(), M.to_host(), R.to_host(), what=(d, n))
        codes.check((d, n)); scales.check((d, n))
        k = ref.norm_steps(d)
        off = k * U * np.abs(hat) + (k + 1) * U * np.abs(x.astype(np.float64)).mean(0) * rstd
        e = scales.array.to_host()
        big = np.abs(ref.blocks(hat)).max(1)
        slack = ref.blocks(off).max(1)
        lo, hi = ref.exponents(np.repeat(big - slack, 32, 0), form), ref.exponents(np.repeat(big + slack, 32, 0), form)
        assert ((e >= np.where(big > slack, lo, 0)) & (e <= hi)).all(), (d, n)
        kept = ref.restore(codes.array.to_host(), e)
        scale = np.repeat(np.ldexp(1.0, e.astype(int) - 127), 32, 0)[:d]
        step = 0.5 * scale if form == "int8" else np.maximum(2.0 ** -4 * (np.abs(hat) + off), 2.0 ** -10 * scale)
        assert (np.abs(kept - hat) <= step + off).all(), (d, n)
        DX, DG, DB = gpu.ROCArray(t, (d, n)), gpu.ROCArray(t, d), gpu.ROCArray(t, d)
        gpu.layernorm_backward_(DX, DY, q, G, rstd=R, dgamma=DG, dbeta=DB)
        check_backward(kept, R.to_host().astype(np.float64), dy, gamma, DX.to_host(), DG.to_host(), DB.to_host(), 0.0, (d, n))
    gpu.synchronize()


def test_many_rows(gpu):
    """More rows than blocks, both ways of dealing them out."""
    for d, n in ((64, 70_001), (520, 5003), (4096, 1100)):
        rng = np.random.default_rng(d)
        x, dy = rows(rng, d, n, np.float32), rng.standard_normal((d, n)).astype(np.float32)
        gamma, beta = params(rng, d, np.float32)
        X, G, B, DY = (gpu.ROCArray.from_host(a) for a in (x, gamma, beta, dy))
        Y, M, R = gpu.ROCArray(np.float32, (d, n)), gpu.ROCArray(np.float32, n), gpu.ROCArray(np.float32, n)
        gpu.layernorm_(Y, X, G, B, mean=M, rstd=R)
        check_forward(gpu, x, gamma, beta, Y.to_host(), M.to_host(), R.to_host(), what=(d, n))
        DX, DG, DB = gpu.ROCArray(np.float32, (d, n)), gpu.ROCArray(np.float32, d), gpu.ROCArray(np.float32, d)
        gpu.layernorm_backward_(DX, DY, X, G, mean=M, rstd=R, dgamma=DG, dbeta=DB)
        mean, rstd = M.to_host().astype(np.float64), R.to_host().astype(np.float64)
        hat = (x - mean) * rstd
        check_backward(hat, rstd, dy, gamma, DX.to_host(), DG.to_host(), DB.to_host(), 2 * U * np.abs(hat), (d, n))
        first = DG.to_host(), DB.to_host()
        gpu.layernorm_backward_(None, DY, X, G, mean=M, rstd=R, dgamma=DG, dbeta=DB)      # parameters alone, the same bits
        assert bits_equal(DG.to_host(), first[0]) and bits_equal(DB.to_host(), first[1])


def test_large_offset_keeps_the_variance(gpu):
    """Rows whose mean is a thousand times their spread: a sum of squares would lose the variance."""
    rng = np.random.default_rng(3)
    for d in (96, 1024, 3000, 9000):
        x = (1000.0 + rng.standard_normal((d, 4))).astype(np.float32)
        X = gpu.ROCArray.from_host(x)
        Y, M, R = X.similar(), gpu.ROCArray(np.float32, 4), gpu.ROCArray(np.float32, 4)
        gpu.layernorm_(Y, X, mean=M, rstd=R)
        check_forward(gpu, x, None, None, Y.to_host(), M.to_host(), R.to_host(), what=d)


def test_options_and_layouts(gpu):
    rng = np.random.default_rng(5)
    t = ref.BF16
    # no parameters; gamma alone; beta alone; eps 0
    x = rows(rng, 200, 6, t)
    g, b = params(rng, 200, t)
    X, G, B = (gpu.ROCArray.from_host(a) for a in (x, g, b))
    M, R = gpu.ROCArray(np.float32, 6), gpu.ROCArray(np.float32, 6)
    for gg, bb in ((None, None), (g, None), (None, b)):
        Y = gpu.layernorm_(X.similar(), X, None if gg is None else G, None if bb is None else B, eps=0.0, mean=M, rstd=R)
        check_forward(gpu, x, gg, bb, Y.to_host(), M.to_host(), R.to_host(), eps=0.0)
    # rows a distance apart, rows off 16 bytes, several row dimensions, a transposed source
    for d, n, pad, off in ((64, 9, 8, 0), (64, 9, 3, 0), (64, 9, 0, 1), (777, 4, 23, 5)):
        big = gpu.ROCArray.from_host(rng.standard_normal((d + pad) * n + off).astype(t))
        V = big.view(off, off + (d + pad) * n).reshape(d + pad, n).subview(slice(0, d), slice(None))
        out = gpu.ROCArray(t, ((d + pad) * n + off,)).fill_(7.0)
        W = out.view(off, off + (d + pad) * n).reshape(d + pad, n).subview(slice(0, d), slice(None))
        g, b = params(rng, d, t)
        M, R = gpu.ROCArray(np.float32, n), gpu.ROCArray(np.float32, n)
        gpu.layernorm_(W, V, gpu.ROCArray.from_host(g), gpu.ROCArray.from_host(b), mean=M, rstd=R)
        check_forward(gpu, V.to_host(), g, b, W.to_host(), M.to_host(), R.to_host(), what=(d, n, pad, off))
        h = out.to_host().astype(np.float32)[off:].reshape(d + pad, n, order="F")
        assert (h[d:] == 7.0).all()
    x = rows(rng, 6 * 5, 4 * 3, np.float32)
    g, b = params(rng, 30, np.float32)
    X = gpu.ROCArray.from_host(x.reshape(6, 5, 4, 3, order="F"))
    M, R = gpu.ROCArray(np.float32, (4, 3)), gpu.ROCArray(np.float32, (4, 3))
    Y = gpu.layernorm_(X.similar(), X, gpu.ROCArray.from_host(g.reshape(6, 5, order="F")), gpu.ROCArray.from_host(b.reshape(6, 5, order="F")), mean=M, rstd=R)
    check_forward(gpu, x, g, b, Y.to_host().reshape(30, 12, order="F"), M.to_host().reshape(-1, order="F"), R.to_host().reshape(-1, order="F"))
    xt = rows(rng, 40, 11, np.float32)
    T = gpu.ROCArray.from_host(np.ascontiguousarray(xt.T)).transpose()                   # (40, 11), element stride 11
    M, R = gpu.ROCArray(np.float32, 11), gpu.ROCArray(np.float32, 11)
    Y = gpu.layernorm_(gpu.ROCArray(np.float32, (11, 40)).transpose(), T, mean=M, rstd=R)
    check_forward(gpu, xt, None, None, Y.to_host(), M.to_host(), R.to_host())
    # in place, forward and gradient
    x = rows(rng, 96, 10, np.float32)
    X = gpu.ROCArray.from_host(x)
    M, R = gpu.ROCArray(np.float32, 10), gpu.ROCArray(np.float32, 10)
    want = gpu.layernorm_(X.similar(), X, mean=M, rstd=R).to_host()
    dy = rng.standard_normal((96, 10)).astype(np.float32)
    DY = gpu.ROCArray.from_host(dy)
    dx, dg, db = (a.to_host() for a in gpu.layernorm_backward(DY, X, mean=M, rstd=R))
    DG, DB = gpu.ROCArray(np.float32, 96), gpu.ROCArray(np.float32, 96)
    gpu.layernorm_backward_(DY, DY, X, mean=M, rstd=R, dgamma=DG, dbeta=DB)
    assert bits_equal(DY.to_host(), dx) and bits_equal(DG.to_host(), dg) and bits_equal(DB.to_host(), db)
    gpu.layernorm_(X, X)
    assert bits_equal(X.to_host(), want)
    # long rows: the gradient's destination over the source
    x = rows(rng, 9001, 3, np.float32)
    X, DY = gpu.ROCArray.from_host(x), gpu.ROCArray.from_host(rng.standard_normal((9001, 3)).astype(np.float32))
    M, R = gpu.ROCArray(np.float32, 3), gpu.ROCArray(np.float32, 3)
    gpu.layernorm_(X.similar(), X, mean=M, rstd=R)
    dx, dg, db = (a.to_host() for a in gpu.layernorm_backward(DY, X, mean=M, rstd=R))
    DG, DB = gpu.ROCArray(np.float32, 9001), gpu.ROCArray(np.float32, 9001)
    gpu.layernorm_backward_(X, DY, X, mean=M, rstd=R, dgamma=DG, dbeta=DB)
    assert bits_equal(X.to_host(), dx) and bits_equal(DG.to_host(), dg) and bits_equal(DB.to_host(), db)


def test_empty_and_special_rows(gpu):
    f32 = np.float32
    assert gpu.layernorm(gpu.ROCArray(f32, (8, 0))).dims == (8, 0)
    assert gpu.layernorm(gpu.ROCArray(f32, (0, 5))).dims == (0, 5)
    E = gpu.ROCArray(f32, (8, 0))
    DG, DB = gpu.ones(f32, 8), gpu.ones(f32, 8)
    gpu.layernorm_backward_(None, E, E, mean=gpu.ROCArray(f32, 0), rstd=gpu.ROCArray(f32, 0), dgamma=DG, dbeta=DB)
    assert not DG.to_host().any() and not DB.to_host().any()
    # rows of one value, and rows with an infinity or a NaN: their own outputs only
    for d in (1, 32, 100, 2048, 9000):
        x = np.random.default_rng(d).standard_normal((d, 5)).astype(f32)
        x[:, 1] = 3.25
        x[d // 2, 2] = np.nan
        x[0, 3] = np.inf
        X = gpu.ROCArray.from_host(x)
        R = gpu.ROCArray(f32, 5)
        q = gpu.Quantized8((d, 5))
        y = gpu.layernorm_(X.similar(), X, rstd=R, checkpoint=q).to_host()
        assert np.isfinite(y[:, [0, 1, 4]]).all() and (y[:, 1] == 0).all()
        assert np.isnan(y[:, [2, 3]]).all()
        assert abs(R.to_host()[1] - 1 / np.sqrt(EPS)) <= 1e-6 / np.sqrt(EPS)
        kept = gpu.dequantize(q).to_host()
        assert np.isnan(kept[:, [2, 3]]).all() and np.isfinite(kept[:, [0, 1, 4]]).all()


def test_streams_threads_and_graphs(gpu):
    """Gradients captured on one stream keep workspaces of their own: two graphs replayed side by side
    on two streams, with eager calls on the capturing stream in between."""
    rng = np.random.default_rng(9)
    d, n = 1024, 600
    sets = []
    for k in range(2):
        x, dy = rows(rng, d, n, ref.BF16), rng.standard_normal((d, n)).astype(ref.BF16)
        X, DY = gpu.ROCArray.from_host(x), gpu.ROCArray.from_host(dy)
        M, R = gpu.ROCArray(np.float32, n), gpu.ROCArray(np.float32, n)
        gpu.layernorm_(X.similar(), X, mean=M, rstd=R)
        want = [a.to_host() for a in gpu.layernorm_backward(DY, X, mean=M, rstd=R)]
        out = [X.similar(), gpu.ROCArray(np.float32, d), gpu.ROCArray(np.float32, d)]
        sets.append((X, DY, M, R, want, out))
    gpu.synchronize()
    st, other = gpu.Stream(), gpu.Stream()
    with gpu.using_stream(st):
        graphs = []
        for X, DY, M, R, want, out in sets:
            graphs.append(gpu.captured(lambda: gpu.layernorm_backward_(out[0], DY, X, mean=M, rstd=R, dgamma=out[1], dbeta=out[2])))
        st.synchronize()
        for _, _, _, _, _, out in sets:
            for a in out:
                a.fill_(0)
        st.synchronize()
        X, DY, M, R, want, _ = sets[0]
        eager = [X.similar(), gpu.ROCArray(np.float32, d), gpu.ROCArray(np.float32, d)]
        for _ in range(5):
            gpu.launch(graphs[0], st)
            gpu.launch(graphs[1], other)
            gpu.layernorm_backward_(eager[0], DY, X, mean=M, rstd=R, dgamma=eager[1], dbeta=eager[2])
        st.synchronize()
        other.synchronize()
        for _, _, _, _, want, out in sets:
            for a, w in zip(out, want):
                assert bits_equal(a.to_host(), w)
        for a, w in zip(eager, sets[0][4]):
            assert bits_equal(a.to_host(), w)
    st.synchronize()


def test_unaligned_parameters_and_broadcast_gradients(gpu):
    """Parameters off 16 bytes beside aligned rows, a gradient that is one row for all (row stride 0), and
    gradients asked for one by one."""
    rng = np.random.default_rng(21)
    for t in ref.TYPES.values():
        for p in (np.dtype(np.float32), t):
            for d, n in ((512, 7), (4096, 5), (1023, 6), (390, 9)):
                x = rows(rng, d, n, t)
                gamma, beta = params(rng, d, p)
                G = gpu.ROCArray.from_host(np.concatenate([gamma[:1], gamma])).view(1, d + 1)
                B = gpu.ROCArray.from_host(np.concatenate([beta[:1], beta])).view(1, d + 1)
                X = gpu.ROCArray.from_host(x)
                M, R = gpu.ROCArray(np.float32, n), gpu.ROCArray(np.float32, n)
                Y = gpu.layernorm_(X.similar(), X, G, B, eps=EPS, mean=M, rstd=R)
                check_forward(gpu, x, gamma, beta, Y.to_host(), M.to_host(), R.to_host(), what=(d, n))
                one = rng.standard_normal(d).astype(t)
                buf = gpu.ROCArray.from_host(one)
                DY = gpu.ROCArray(t, (d, n), _buf=buf.buf, _strides=(1, 0))
                dy = np.repeat(one[:, None], n, axis=1)
                mean, rstd = M.to_host().astype(np.float64), R.to_host().astype(np.float64)
                hat = (x.astype(np.float64) - mean) * rstd
                DX, DG, DB = gpu.ROCArray(t, (d, n)), gpu.ROCArray(p, d), gpu.ROCArray(p, d)
                gpu.layernorm_backward_(DX, DY, X, G, mean=M, rstd=R, dgamma=DG)
                gpu.layernorm_backward_(None, DY, X, G, mean=M, rstd=R, dbeta=DB)
                check_backward(hat, rstd, dy, gamma, DX.to_host(), DG.to_host(), DB.to_host(), 2 * U * np.abs(hat), (d, n))
    gpu.synchronize()


def test_rows_over_several_streams(gpu):
    """Operators on two streams by turns, on the same arrays: each waits for what the other wrote."""
    rng = np.random.default_rng(22)
    d, n = 2048, 3000
    x = rows(rng, d, n, ref.BF16)
    X = gpu.ROCArray.from_host(x)
    a, b = gpu.Stream(), gpu.Stream()
    want = gpu.layernorm(gpu.layernorm(gpu.layernorm(X))).to_host()
    Y, Z, W = (X.similar() for _ in range(3))
    for _ in range(3):
        gpu.layernorm_(Y, X, stream=a)
        gpu.layernorm_(Z, Y, stream=b)
        gpu.layernorm_(W, Z, stream=a)
        assert bits_equal(W.to_host(), want)


NARROW = [(34, 40), (66, 50), (70, 9), (101, 300), (127, 33), (129, 64), (130, 17), (201, 41), (202, 40), (255, 7), (257, 5), (258, 30),
          (390, 20), (511, 9), (514, 11), (1026, 9), (1536, 40), (2046, 5), (3000, 7), (4094, 4), (4095, 3), (6144, 9), (6145, 2), (8190, 2)]


def uneven_rows(rng, d, n, t):
    """Rows whose blocks of 32 differ in magnitude, so that no block's scale fits its neighbour."""
    x = rng.standard_normal((d, n)) * np.ldexp(1.0, (np.arange(d) // 32 * 5 % 9) - 4)[:, None] + 0.25
    return x.astype(t)


@pytest.mark.parametrize("dtype", list(ref.TYPES))
def test_rows_of_many_widths(gpu, dtype, monkeypatch):
    """Widths on either side of what a thread, a warp and a block of threads hold, at every alignment of 16-bit rows."""
    import sys
    here = sys.modules[__name__]
    monkeypatch.setattr(here, "SHAPES", NARROW)
    monkeypatch.setattr(here, "rows", uneven_rows)
    test_forward_and_gradient(gpu, dtype, True)
    for form in ("int8", "e4m3"):
        test_checkpoint(gpu, dtype, form)


def test_moments_of_rows_without_elements(gpu):
    """0/0, as a mean over nothing is everywhere: what stood in the arrays before does not stay."""
    for t in ref.TYPES.values():
        X = gpu.ROCArray(t, (0, 5))
        M, R = gpu.fill(np.float32(7), 5), gpu.fill(np.float32(7), 5)
        gpu.layernorm_(X, X, mean=M, rstd=R)
        assert np.isnan(M.to_host()).all() and np.isnan(R.to_host()).all()


@pytest.mark.parametrize("form", ["int8", "e4m3"])
def test_codes_of_any_alignment(gpu, form):
    """Checkpoints that are views off 16, 8, 4 and 2 bytes, scale bytes off theirs: the codes are those of an
    aligned checkpoint, and the gradient is the formula's."""
    rng = np.random.default_rng(31)
    for t in ref.TYPES.values():
        for d, n in ((64, 300), (101, 400), (1000, 30), (1024, 40), (4096, 9), (9002, 3)):
            x, dy = uneven_rows(rng, d, n, t), rng.standard_normal((d, n)).astype(t)
            gamma, _ = params(rng, d, t)
            X, DY, G = (gpu.ROCArray.from_host(a) for a in (x, dy, gamma))
            want, R = gpu.Quantized8((d, n), form), gpu.ROCArray(np.float32, n)
            gpu.layernorm_(X.similar(), X, rstd=R, checkpoint=want)
            # element by element codes may lie beside a rounding's border: sums in another order
            kept64 = ref.restore(want.codes.to_host(), want.scales.to_host())
            for off in (1, 2, 4, 8):
                codes, scales = (Guarded(gpu, a.dtype, a.dims, misalign=off) for a in (want.codes, want.scales))
                q = gpu.Quantized8.wrap(codes.array, scales.array)
                gpu.layernorm_(X.similar(), X, rstd=R, checkpoint=q)
                codes.check((d, n, off)); scales.check((d, n, off))
                kept = ref.restore(codes.array.to_host(), scales.array.to_host())
                scale = np.repeat(np.ldexp(1.0, np.maximum(scales.array.to_host(), want.scales.to_host()).astype(int) - 127), 32, 0)[:d]
                step = scale if form == "int8" else np.maximum(2.0 ** -3 * np.maximum(np.abs(kept), np.abs(kept64)), 2.0 ** -9 * scale)
                assert (np.abs(kept - kept64) <= step).all(), (d, n, off)
                DX, DG, DB = gpu.ROCArray(t, (d, n)), gpu.ROCArray(t, d), gpu.ROCArray(t, d)
                gpu.layernorm_backward_(DX, DY, q, G, rstd=R, dgamma=DG, dbeta=DB)
                check_backward(kept, R.to_host().astype(np.float64), dy, gamma, DX.to_host(), DG.to_host(), DB.to_host(), 0.0, (d, n, off))
