"""Threads that take several rows, heads or calls one after another: stages of the rings, buffers of
the sums, scale bytes and moments loaded ahead, and workspaces are used again and again.

Inputs are drawn from a small pool.  A call on the pool alone gives a group of threads one row (a
thread one head) at most, and is checked against binary64; with every row of the pool taken many times
in any order, each result has to have the pool's bits, since a row's arithmetic does not depend on where
it lies.  Sums over the rows are made of integers and halves whose partial sums binary32 holds exactly,
in whatever order they are added: they have to be equal, so that no row may be lost or taken twice."""
import threading

import ml_dtypes
import numpy as np
import pytest

import row_reference as ref
from helpers import bits_equal
from test_gpu_layernorm import EPS, check_backward, check_forward, params, rows

pytestmark = pytest.mark.gpu
POOL = 97

# Row length, rows: three to eleven rows for a group of threads on 148 SMs, in every kernel: aligned rows
# that fill the threads and that do not, rows of odd and of even width in 4, 8 and 16 columns a thread,
# and rows longer than either form holds.
MANY = [(64, 30_001), (101, 12_001), (202, 12_001), (1022, 5003), (1023, 5003), (1536, 4001), (2048, 4001), (2624, 2501), (4095, 1501),
        (4096, 2001), (5120, 1301), (8191, 701), (9001, 1301), (12_288, 701), (16_384, 701)]


def taken(pool, pick):
    """``pool[..., pick]`` in column-major order."""
    return np.ascontiguousarray(pool.T)[pick].T


def same_as_pool(got, pool, pick, what):
    assert bits_equal(got.T, taken(pool, pick).T), what


@pytest.mark.parametrize("dtype", list(ref.TYPES))
def test_forward_over_many_rows(gpu, dtype):
    t = ref.TYPES[dtype]
    for d, n in MANY:
        rng = np.random.default_rng(d)
        pool, pick = rows(rng, d, POOL, t), rng.integers(0, POOL, n)
        gamma, beta = params(rng, d, np.float32)
        G, B = gpu.ROCArray.from_host(gamma), gpu.ROCArray.from_host(beta)
        for form in (None, "int8", "e4m3"):
            results = []
            for x in (pool, taken(pool, pick)):
                X, m = gpu.ROCArray.from_host(x), x.shape[1]
                M, R = gpu.ROCArray(np.float32, m), gpu.ROCArray(np.float32, m)
                q = None if form is None else gpu.Quantized8((d, m), form)
                Y = gpu.layernorm_(X.similar(), X, G, B, eps=EPS, mean=M, rstd=R, checkpoint=q)
                results.append([a.to_host() for a in (Y, M, R) + (() if q is None else (q.codes, q.scales))])
            check_forward(gpu, pool, gamma, beta, *results[0][:3], what=(d, form))
            for name, small, large in zip(("y", "mean", "rstd", "codes", "scales"), *results):
                same_as_pool(large, small, pick, (d, form, name))


def whole_rows(rng, d, t):
    """Rows of integers, moments and codes for which the normalised rows are integers and halves."""
    x = rng.integers(-8, 9, (d, POOL)).astype(t)
    mean = rng.integers(-2, 3, POOL).astype(np.float32)
    rstd = np.ldexp(1.0, rng.integers(-1, 2, POOL)).astype(np.float32)
    codes = rng.integers(-8, 9, (d, POOL))
    scales = rng.integers(126, 129, (-(-d // 32), POOL)).astype(np.uint8)
    return x, mean, rstd, codes, scales


@pytest.mark.parametrize("dtype", list(ref.TYPES))
@pytest.mark.parametrize("form", ["rows", "int8", "e4m3"])
def test_gradients_over_many_rows(gpu, dtype, form):
    """Terms of dgamma are multiples of 1/2 up to 3 * 20 (8 bits: 3 * 16), those of dbeta up to 3: with
    30 001 rows the sums stay below 2^23 halves, exact in binary32."""
    t = ref.TYPES[dtype]
    for d, n in MANY:
        rng = np.random.default_rng(d + 1)
        x, mean, rstd, codes, scales = whole_rows(rng, d, t)
        dy = rng.integers(1, 4, (d, POOL)).astype(t)
        gamma, _ = params(rng, d, np.float32)
        pick = rng.integers(0, POOL, n)
        G = gpu.ROCArray.from_host(gamma)
        if form == "rows":
            hat = (x.astype(np.float64) - mean) * rstd
        else:
            codes = codes.astype(np.int8) if form == "int8" else codes.astype(np.float32).astype(ml_dtypes.float8_e4m3fn).view(np.uint8)
            hat = ref.restore(codes, scales)
        dxs, sums = [], []
        for p in (np.arange(POOL), pick):
            up = lambda a: gpu.ROCArray.from_host(taken(a, p))
            DY, R = up(dy), up(rstd)
            source = dict(X=up(x), mean=up(mean)) if form == "rows" else dict(X=gpu.Quantized8.wrap(up(codes), up(scales)))
            DX, DG, DB = gpu.ROCArray(t, (d, len(p))), gpu.ROCArray(np.float32, d), gpu.ROCArray(np.float32, d)
            gpu.layernorm_backward_(DX, DY, gamma=G, rstd=R, dgamma=DG, dbeta=DB, **source)
            dxs.append(DX.to_host())
            sums.append((DG.to_host(), DB.to_host()))
            if len(p) == n:                        # in place, and the parameters alone: the same bits
                gpu.layernorm_backward_(DY, DY, gamma=G, rstd=R, **source)
                assert bits_equal(DY.to_host(), dxs[1]), (d, "in place")
        check_backward(hat, rstd.astype(np.float64), dy, gamma, dxs[0], None, None, 0.0, (d, form))
        same_as_pool(dxs[1], dxs[0], pick, (d, form, "dx"))
        for (dg, db), p in zip(sums, (np.arange(POOL), pick)):
            count = np.bincount(p, minlength=POOL).astype(np.float64)
            assert np.array_equal(db.astype(np.float64), dy.astype(np.float64) @ count), (d, form, len(p), "dbeta")
            assert np.array_equal(dg.astype(np.float64), (dy.astype(np.float64) * hat) @ count), (d, form, len(p), "dgamma")


def test_parameters_of_the_rows_type(gpu):
    """Sums in 16 bits are the exact sums, rounded once."""
    for dtype in ("f16", "bf16"):
        t = ref.TYPES[dtype]
        for d, n in ((101, 12_001), (1024, 4001), (9001, 601)):
            rng = np.random.default_rng(d + 2)
            x, mean, rstd, _, _ = whole_rows(rng, d, t)
            dy = (rng.integers(1, 4, (d, POOL)) * 0.25).astype(t)          # below Float16's largest value
            pick = rng.integers(0, POOL, n)
            up = lambda a: gpu.ROCArray.from_host(taken(a, pick))
            gamma = gpu.ones(t, d)
            DX, DG, DB = gpu.layernorm_backward(up(dy), up(x), gamma, rstd=up(rstd), mean=up(mean))
            count = np.bincount(pick, minlength=POOL).astype(np.float64)
            hat = (x.astype(np.float64) - mean) * rstd
            ref.within(DB.to_host(), dy.astype(np.float64) @ count, 0.0, (dtype, d, "dbeta"))
            ref.within(DG.to_host(), (dy.astype(np.float64) * hat) @ count, 0.0, (dtype, d, "dgamma"))


@pytest.mark.parametrize("dtype", list(ref.TYPES))
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_over_many_heads(gpu, dtype, layout):
    """With 20 011 tokens a thread takes five or six heads: by vectors, by uneven vectors, element by
    element, and the elements that pass through; out of place, in place and backwards."""
    t = ref.TYPES[dtype]
    for d, rot, heads, off in ((64, 64, 5, 0), (64, 64, 12, 0), (96, 64, 12, 0), (80, 26, 5, 0), (80, 26, 12, 0), (36, 18, 5, 0), (64, 32, 5, 1)):
        rng = np.random.default_rng(d + rot + heads)
        n, few = 20_011, 48
        pool = rng.standard_normal((d, heads, few)).astype(t)
        pos = rng.integers(-1000, 100_000, few).astype(np.int32)
        pick = rng.integers(0, few, n)
        freq, factor = gpu.rotary.rotary_frequencies(rot, scaling="yarn", stretch=4.0, original_length=2048)
        plan = gpu.RotaryPlan(freq, layout, factor)

        def placed(x):                             # `off`: heads that start off 16 bytes
            A = gpu.ROCArray(t, x.size + off)
            V = A.view(off, off + x.size).reshape(x.shape)
            return V.copy_from_host(x)
        for adjoint in (False, True):
            small = gpu.rotary_(placed(pool), placed(pool), gpu.ROCArray.from_host(pos), plan, adjoint=adjoint).to_host()
            ref.within(small, ref.turn(pool, pos, freq, factor, layout, adjoint), ref.turn_slack(pool, rot, factor, layout), (d, rot, heads, adjoint))
            X, P = placed(taken(pool, pick)), gpu.ROCArray.from_host(pos[pick])
            Y = placed(np.zeros((d, heads, n), t))
            same_as_pool(gpu.rotary_(Y, X, P, plan, adjoint=adjoint).to_host(), small, pick, (d, rot, heads, adjoint))
            same_as_pool(gpu.rotary_(X, X, P, plan, adjoint=adjoint).to_host(), small, pick, (d, rot, heads, adjoint, "in place"))


@pytest.mark.parametrize("shared", [False, True])
def test_host_threads(gpu, shared):
    """Two host threads with operators that need workspaces (the sums of a gradient, the claims of many
    slots), on a stream each or both on one: each gets what it gets alone."""
    d, n, tokens = 1000, 900, 3000
    jobs = []
    for k in range(2):
        rng = np.random.default_rng(k)
        width = d + 24 * k                          # workspaces of different sizes
        x, dy = rows(rng, width, n, ref.BF16), rng.standard_normal((width, n)).astype(ref.BF16)
        kv = rng.standard_normal((32, 2, tokens)).astype(np.float32)
        slots = rng.integers(1, 500 * (k + 1), tokens).astype(np.int32)
        jobs.append((x, dy, kv, slots))
    streams = [gpu.Stream(), gpu.Stream()]
    if shared:
        streams[1] = streams[0]
    failures = []

    def work(k, results, turns):
        try:
            gpu.device_(0)
            st = streams[k]
            with gpu.using_stream(st):
                x, dy, kv, slots = jobs[k]
                X, DY, K, S = (gpu.ROCArray.from_host(a) for a in (x, dy, kv, slots))
                M, R = gpu.ROCArray(np.float32, n), gpu.ROCArray(np.float32, n)
                gpu.layernorm_(X.similar(), X, mean=M, rstd=R)
                for _ in range(turns):
                    cache = gpu.quantized_cache(32, 2, 50, 10 * (k + 1))
                    grads = gpu.layernorm_backward(DY, X, mean=M, rstd=R)
                    gpu.cache_write_(cache, K, K, S)
                    results.append([a.to_host() for a in grads + cache._arrays()])
        except Exception as e:                      # raised again by the test's own thread
            failures.append(e)

    alone = [[], []]
    for k in range(2):
        work(k, alone[k], 1)
    together = [[], []]
    threads = [threading.Thread(target=work, args=(k, together[k], 20)) for k in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    if failures:
        raise failures[0]
    for k in range(2):
        assert len(together[k]) == 20
        for got in together[k]:
            for a, w in zip(got, alone[k][0]):
                assert bits_equal(a, w)
