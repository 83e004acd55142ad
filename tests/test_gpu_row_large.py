"""Row operators on arrays of more than 2^31 elements: rows at the front, across element 2^31 and at the
end get the bits that a call on those rows alone gives (which the other tests check against binary64)."""
import numpy as np
import pytest

import row_reference as ref
from helpers import bits_equal
from test_gpu_layernorm import params, rows

pytestmark = pytest.mark.gpu
T = ref.BF16
FAR = 1 << 31
U = ref.U


class Windows:
    """Arrays of zeros (d, n) with the same few rows in three places."""

    def __init__(self, gpu, d, few):
        self.gpu, self.d, self.few = gpu, d, few
        self.n = FAR // d + 3001
        self.at = (0, FAR // d - few // 2, self.n - few)

    def place(self, small):
        A = self.gpu.zeros(small.dtype, small.dims[:-1] + (self.n,))
        per = small.size // self.few
        for lo in self.at:
            self.gpu.copyto_(A.view(lo * per, (lo + self.few) * per), small.reshape(small.size))
        return A

    def check(self, large, small, what):
        per = small.size // self.few
        want = small.to_host().reshape(-1, order="F")
        for lo in self.at:
            assert bits_equal(large.view(lo * per, (lo + self.few) * per).to_host(), want), (what, lo)


@pytest.mark.parametrize("d", [4096, 4101, 4102, 9001])
def test_layernorm(gpu, d):
    rng = np.random.default_rng(d)
    w = Windows(gpu, d, 64)
    x, dy = rows(rng, d, 64, T), rng.standard_normal((d, 64)).astype(T)
    gamma, beta = params(rng, d, np.float32)
    G, B = gpu.ROCArray.from_host(gamma), gpu.ROCArray.from_host(beta)
    results = []
    small = [gpu.ROCArray.from_host(a) for a in (x, dy)]
    for X, DY in (small, [w.place(a) for a in small]):
        n = X.dims[1]
        M, R, q = gpu.ROCArray(np.float32, n), gpu.ROCArray(np.float32, n), gpu.Quantized8((d, n))
        Y = gpu.layernorm_(X.similar(), X, G, B, mean=M, rstd=R, checkpoint=q)
        back = gpu.layernorm_backward(DY, X, G, mean=M, rstd=R)
        kept = gpu.layernorm_backward(DY, q, G, rstd=R)
        results.append((Y, M, R, q.codes, q.scales, back[0], kept[0]))
        sums = [a.to_host().astype(np.float64) for a in back[1:] + kept[1:]]
        if n == 64:
            ones = sums
    for k, (a, b) in enumerate(zip(*results)):
        w.check(b, a, (d, k))
    # every other row adds nothing; rows of a group, groups of a block, the fold: below 1000 additions
    hat = np.abs((x.astype(np.float64) - results[0][1].to_host()) * results[0][2].to_host()) + 0.5
    dy64 = np.abs(dy.astype(np.float64))
    for got, one, terms in zip(sums, ones, (dy64 * hat, dy64) * 2):
        assert (np.abs(got - 3 * one) <= 4 * 1000 * U * terms.sum(1)).all(), d


@pytest.mark.parametrize("d", [20, 4096, 4101])
def test_codes_and_activations(gpu, d):
    rng = np.random.default_rng(d)
    few = 64 if d > 32 else 640
    w = Windows(gpu, d, few)
    small = [gpu.ROCArray.from_host(rng.standard_normal((d, few)).astype(T)) for _ in range(3)]
    results = []
    for A, B, DY in (small, [w.place(a) for a in small]):
        dims = A.dims
        q = gpu.quantize(A, "e4m3")
        back = gpu.dequantize(q, T)
        qa, qb = gpu.Quantized8(dims), gpu.Quantized8(dims)
        Y = gpu.activation_("silu", gpu.ROCArray(T, dims), A, B, checkpoint=qa, gate_checkpoint=qb)
        DA, DB, DC = (gpu.ROCArray(T, dims) for _ in range(3))
        gpu.activation_backward_("silu", DA, DY, qa, qb, dgate=DB)
        gpu.activation_backward_("gelu", DC, DY, A)
        results.append((q.codes, q.scales, back, qa.codes, qa.scales, qb.codes, Y, DA, DB, DC))
    for k, (a, b) in enumerate(zip(*results)):
        w.check(b, a, (d, k))


@pytest.mark.parametrize("d,rot,heads", [(128, 128, 8), (80, 26, 5), (36, 18, 1)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary(gpu, d, rot, heads, layout):
    rng = np.random.default_rng(d)
    w = Windows(gpu, d * heads, 40)
    plan = gpu.rotary_plan(rot, layout=layout)
    X = gpu.ROCArray.from_host(rng.standard_normal((d, heads, 40)).astype(T))
    P = gpu.ROCArray.from_host(rng.integers(0, 1 << 20, 40).astype(np.int32))
    small = gpu.rotary_(X.similar(), X, P, plan)
    L, LP = w.place(X), w.place(P)
    w.check(gpu.rotary_(L.similar(), L, LP, plan), small, "apart")
    w.check(gpu.rotary_(L, L, LP, plan), small, "in place")


def test_cache(gpu):
    d, heads, page, few = 128, 8, 64, 48
    w = Windows(gpu, d * heads, few)
    rng = np.random.default_rng(5)
    K, V = (gpu.ROCArray.from_host(rng.standard_normal((k, heads, few)).astype(T)) for k in (d, 32))
    plan = gpu.rotary_plan(d)
    # the first and the last window's tokens go to slots that the middle one's, behind it, do not take
    slots = rng.permutation(40 * page)[: 3 * few].astype(np.int32) + 1
    pos = rng.integers(0, 1 << 20, few).astype(np.int32)
    one = gpu.quantized_cache(d, heads, page, 40, value_dim=32)
    for k in range(3):
        gpu.cache_write_(one, K, V, gpu.ROCArray.from_host(slots[k * few:(k + 1) * few].copy()), rotary=plan, positions=gpu.ROCArray.from_host(pos))
    many = gpu.quantized_cache(d, heads, page, 40, value_dim=32)
    S = gpu.zeros(np.int32, w.n)                   # slot 0: left out
    for k, lo in enumerate(w.at):
        gpu.copyto_(S.view(lo, lo + few), gpu.ROCArray.from_host(slots[k * few:(k + 1) * few].copy()))
    gpu.cache_write_(many, w.place(K), w.place(V), S, rotary=plan, positions=w.place(gpu.ROCArray.from_host(pos)))
    gpu.synchronize()
    for a, b in zip(one._arrays(), many._arrays()):
        assert bits_equal(a.to_host(), b.to_host())
    # reading back: places past 2^31 elements
    places = w.n // page * page
    table = rng.integers(1, 41, places // page).astype(np.int32)
    out = [gpu.zeros(T, (k, heads, places, 1)) for k in (d, 32)]
    gpu.cache_read_(*out, one, gpu.ROCArray.from_host(table[:, None].copy()), gpu.ROCArray.from_host(np.array([places - 3], np.int32)))
    gpu.synchronize()
    for o, q in zip(out, (one.keys, one.values)):
        per = o.size // places
        v = ref.rounded(ref.restore(q.codes.to_host(), q.scales.to_host()), T)
        for lo in (0, FAR // (d * heads) - 100, places - 200):
            l = np.arange(lo, lo + 200)
            want = v[:, :, l % page, table[l // page] - 1]
            want[:, :, l >= places - 3] = 0
            got = o.view(lo * per, (lo + 200) * per).to_host().reshape(want.shape, order="F")
            assert np.array_equal(got.astype(np.float64), want), lo
