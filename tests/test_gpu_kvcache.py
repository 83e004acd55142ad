"""The quantised cache: tokens written to slots, contexts read back through page tables."""
import numpy as np
import pytest

import row_reference as ref
from helpers import Guarded, bits_equal

pytestmark = pytest.mark.gpu


def dequantized(cache):
    """(d, heads, slots) of keys and values as the codes stand, from the host."""
    out = []
    for q in (cache.keys, cache.values):
        v = ref.restore(q.codes.to_host(), q.scales.to_host())
        out.append(v.reshape(v.shape[:2] + (-1,), order="F"))
    return out


def kept(x, form):
    """What (d, ...) rows stand for in 8 bits."""
    return ref.restore(*ref.quantize(x, form))


# head size of keys and values, heads, page size, pages
CACHES = [(32, 32, 1, 1, 3), (64, 64, 4, 16, 9), (128, 128, 8, 64, 5), (72, 40, 3, 5, 11), (7, 33, 2, 3, 8), (256, 128, 1, 32, 4), (96, 96, 12, 2, 30)]


@pytest.mark.parametrize("form", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", list(ref.TYPES))
def test_write_and_read(gpu, dtype, form):
    t = ref.TYPES[dtype]
    for k, (dk, dv, heads, page, npages) in enumerate(CACHES):
        rng = np.random.default_rng(k)
        cache = gpu.quantized_cache(dk, heads, page, npages, form, value_dim=dv)
        n = min(cache.slots, 20)
        K, V = rng.standard_normal((dk, heads, n)).astype(t), rng.standard_normal((dv, heads, n)).astype(t)
        slots = (rng.permutation(cache.slots)[:n] + 1).astype(np.int32 if k % 2 else np.int64)
        slots[n // 2] = 0                                            # a padded token
        Kd, Vd, S = (gpu.ROCArray.from_host(a) for a in (K, V, slots))
        gpu.cache_write_(cache, Kd, Vd, S)
        want = [np.zeros((d, heads, cache.slots)) for d in (dk, dv)]
        for w, x in zip(want, (K, V)):
            live = slots > 0
            w[:, :, slots[live] - 1] = kept(x.astype(np.float64)[:, :, live], form)
        for got, w in zip(dequantized(cache), want):
            assert np.array_equal(got, w), (k, "codes")
        # sequences of many lengths over shuffled pages, one empty, one full
        seqs = 4
        most = max(1, npages - 1)
        pages = np.stack([rng.permutation(npages)[:most] + 1 for _ in range(seqs)], 1).astype(np.int32)
        lengths = np.array([0, 1, most * page, rng.integers(0, most * page + 1)], np.int64 if k % 2 else np.int32)
        places = most * page + 2
        pages[-(-int(lengths[3]) // page):, 3] = 0                   # entries behind the last page are not looked at
        outs = [Guarded(gpu, t, (d, heads, places, seqs)) for d in (dk, dv)]
        for o in outs:
            o.array.fill_(9.0)
        gpu.cache_read_(outs[0].array, outs[1].array, cache, gpu.ROCArray.from_host(pages), gpu.ROCArray.from_host(lengths))
        gpu.synchronize()
        for o, w in zip(outs, want):
            o.check(k)
            got = o.array.to_host()
            for b in range(seqs):
                m = int(lengths[b])
                l = np.arange(m)
                row = (pages[l // page, b].astype(np.int64) - 1) * page + l % page
                ref.within(got[:, :, :m, b], w[:, :, row], 0.0, (k, b))
                assert (got[:, :, m:, b].astype(np.float32) == 9.0).all(), (k, b)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_keys_turned_on_the_way(gpu, layout):
    """The keys in the cache are the turned keys to half a code (their codes may differ by one where
    the turned value, good to a few U, lies at a rounding's border); values are not turned."""
    for dtype in ref.TYPES.values():
        for form in ("int8", "e4m3"):
            for d, rot, heads, n in ((64, 64, 4, 9), (80, 26, 2, 40), (128, 64, 8, 3), (12, 6, 3, 5), (256, 256, 1, 2)):
                rng = np.random.default_rng(d + rot)
                kw = dict(scaling="yarn", stretch=4.0, original_length=1024)
                freq, factor = gpu.rotary.rotary_frequencies(rot, **kw)
                plan = gpu.rotary_plan(rot, layout=layout, **kw)
                cache = gpu.quantized_cache(d, heads, 8, 6, form)
                K, V = rng.standard_normal((d, heads, n)).astype(dtype), rng.standard_normal((d, heads, n)).astype(dtype)
                pos = rng.integers(0, 1 << 20, n)
                slots = rng.permutation(48)[:n] + 1
                gpu.cache_write_(cache, *(gpu.ROCArray.from_host(a) for a in (K, V, slots.astype(np.int64))), rotary=plan,
                                 positions=gpu.ROCArray.from_host(pos.astype(np.int32)))
                k_got, v_got = dequantized(cache)
                assert np.array_equal(v_got[:, :, slots - 1], kept(V.astype(np.float64), form))
                want = ref.turn(K, pos, freq, factor, layout)
                off = ref.turn_slack(K, rot, factor, layout)
                big, slack = np.abs(ref.blocks(want)).max(1), ref.blocks(off).max(1)
                scale = np.repeat(np.ldexp(1.0, ref.exponents(np.repeat(big + slack, 32, 0), form).astype(int) - 127), 32, 0)[:d]
                half = 0.5 * scale if form == "int8" else np.maximum(2.0 ** -4 * (np.abs(want) + off), 2.0 ** -10 * scale)
                assert (np.abs(k_got[:, :, slots - 1] - want) <= half + off).all(), (d, rot, form)


@pytest.mark.parametrize("n", [2, 300, 2048, 2049, 5000])
def test_the_last_of_equal_slots_is_kept(gpu, n):
    """As if the tokens were written in turn; with few tokens (a look through the later slots) and with
    many (a table of claims).  Twice, with other values, so that nothing is left from the first time."""
    rng = np.random.default_rng(n)
    cache = gpu.quantized_cache(32, 2, 16, 20)
    for _ in range(2):
        slots = rng.integers(0, 2 if n == 2 else 200, n)
        if n == 2:
            slots[:] = 7
        K, V = rng.standard_normal((32, 2, n)).astype(np.float32), rng.standard_normal((32, 2, n)).astype(np.float32)
        before = dequantized(cache)
        gpu.cache_write_(cache, *(gpu.ROCArray.from_host(a) for a in (K, V, slots.astype(np.int32))))
        for got, w, x in zip(dequantized(cache), before, (K, V)):
            for j in range(n):
                if slots[j]:
                    w[:, :, slots[j] - 1] = 0
            last = {int(s): j for j, s in enumerate(slots) if s}
            for s, j in last.items():
                w[:, :, s - 1] = kept(x[:, :, j].astype(np.float64), "int8")
            assert np.array_equal(got, w)
    gpu.synchronize()


def test_bad_slots_pages_and_lengths(gpu):
    """Nothing outside the cache or the destination is touched; the next synchronisation reports it."""
    rng = np.random.default_rng(2)
    raw = [Guarded(gpu, np.int8, (64, 2, 4, 3)), Guarded(gpu, np.uint8, (2, 2, 4, 3)), Guarded(gpu, np.int8, (64, 2, 4, 3)), Guarded(gpu, np.uint8, (2, 2, 4, 3))]
    for g in raw:
        g.array.fill_(0)
    cache = gpu.QuantizedCache(gpu.Quantized8.wrap(raw[0].array, raw[1].array), gpu.Quantized8.wrap(raw[2].array, raw[3].array))
    K = rng.standard_normal((64, 2, 5)).astype(np.float32)
    Kd = gpu.ROCArray.from_host(K)
    for n in (5, 3000):                                             # both ways of settling slots
        X = Kd if n == 5 else gpu.ROCArray.from_host(np.repeat(K, 600, 2))
        for bad in (13, -1, 1 << 40, -(1 << 62)):
            slots = np.zeros(n, np.int64)
            slots[:2] = [bad, 12]
            gpu.cache_write_(cache, X, X, gpu.ROCArray.from_host(slots))
            with pytest.raises(gpu.B200Error) as err:
                gpu.synchronize()
            assert err.value.code == gpu._lib.INVALID_ARG
            gpu.synchronize()                                       # reported once
            for g in raw:
                g.check((n, bad))
    k, v = dequantized(cache)
    assert np.abs(k[:, :, 11]).max() > 0 and not k[:, :, :11].any()
    outs = [Guarded(gpu, np.float32, (64, 2, 8, 2)) for _ in range(2)]

    def read(pages, lengths):
        for o in outs:
            o.array.fill_(5.0)
        gpu.cache_read_(outs[0].array, outs[1].array, cache, gpu.ROCArray.from_host(np.array(pages, np.int32)), gpu.ROCArray.from_host(np.array(lengths, np.int32)))
        for o in outs:
            try:
                gpu.synchronize()
                bad = False
            except gpu.B200Error as e:
                assert e.code == gpu._lib.INVALID_ARG
                bad = True
            break
        for o in outs:
            o.check((pages, lengths))
        return bad, outs[0].array.to_host()

    bad, h = read([[3, 1], [1, 2]], [8, 3])
    assert not bad and np.array_equal(h[:, :, 3, 0], k[:, :, 11].astype(np.float32)) and (h[:, :, 3:, 1] == 5).all()
    for page in (0, 4, -7, 2_000_000_000):
        bad, h = read([[3, 1], [page, 2]], [8, 3])                  # a page outside the cache: its places are left alone
        assert bad and (h[:, :, 4:, 0] == 5).all() and (h[:, :, :3, 1] == 0).all()
        bad, h = read([[3, 1], [page, page]], [4, 3])               # not looked at
        assert not bad
    bad, h = read([[3, 1], [1, 2]], [-1, 3])
    assert bad and (h[:, :, :, 0] == 5).all() and (h[:, :, :3, 1] == 0).all()
    bad, h = read([[3, 1], [1, 2]], [9, 3])                         # past the places
    assert bad and np.array_equal(h[:, :, 3, 0], k[:, :, 11].astype(np.float32))
    bad, h = read([[3, 1]], [5, 3])                                 # past the page table
    assert bad and (h[:, :, 4:, 0] == 5).all()


def test_layouts_of_the_cache(gpu):
    """Pages with heads outside places, keys and values interleaved in one buffer, tokens as slices of
    a projection, a destination with places outside heads."""
    rng = np.random.default_rng(12)
    t = ref.BF16
    d, heads, page, npages, n = 64, 3, 8, 5, 17
    plain = gpu.quantized_cache(d, heads, page, npages)
    qkv = rng.standard_normal((d, 4 * heads, n)).astype(t)
    P = gpu.ROCArray.from_host(qkv)
    K, V = P.subview(slice(None), slice(2 * heads, 3 * heads), slice(None)), P.subview(slice(None), slice(3 * heads, 4 * heads), slice(None))
    slots = gpu.ROCArray.from_host((rng.permutation(page * npages)[:n] + 1).astype(np.int32))
    gpu.cache_write_(plain, K, V, slots)
    codes = gpu.ROCArray(np.int8, (d, page, heads, 2, npages)).fill_(0)
    scales = gpu.ROCArray(np.uint8, (2, page, heads, 2, npages)).fill_(0)
    sides = [gpu.Quantized8.wrap(codes.subview(*(slice(None),) * 3, s, slice(None)).permuteddims((1, 3, 2, 4)),
                                 scales.subview(*(slice(None),) * 3, s, slice(None)).permuteddims((1, 3, 2, 4))) for s in (0, 1)]
    other = gpu.QuantizedCache(*sides)
    gpu.cache_write_(other, gpu.ROCArray.from_host(qkv[:, 2 * heads:3 * heads].copy()), gpu.ROCArray.from_host(qkv[:, 3 * heads:].copy()), slots)
    for a, b in zip(dequantized(plain), dequantized(other)):
        assert np.array_equal(a, b) and a.any()
    pages = gpu.ROCArray.from_host(np.array([[2, 5], [4, 1], [1, 3]], np.int64))
    lengths = gpu.ROCArray.from_host(np.array([19, 24], np.int32))
    a = [gpu.zeros(np.float32, (d, heads, 24, 2)) for _ in range(2)]
    b = [gpu.zeros(np.float32, (d, 24, heads, 2)).permuteddims((1, 3, 2, 4)) for _ in range(2)]
    gpu.cache_read_(*a, plain, pages, lengths)
    gpu.cache_read_(*b, other, pages, lengths)
    for x, y in zip(a, b):
        assert bits_equal(x.to_host(), y.to_host())
    # nothing to do
    gpu.cache_write_(plain, gpu.ROCArray(t, (d, heads, 0)), gpu.ROCArray(t, (d, heads, 0)), gpu.ROCArray(np.int32, 0))
    gpu.cache_read_(gpu.ROCArray(t, (d, heads, 0, 2)), gpu.ROCArray(t, (d, heads, 0, 2)), plain, pages, gpu.ROCArray.from_host(np.zeros(2, np.int32)))
    gpu.cache_read_(gpu.ROCArray(t, (d, heads, 4, 0)), gpu.ROCArray(t, (d, heads, 4, 0)), plain, gpu.ROCArray(np.int32, (3, 0)), gpu.ROCArray(np.int32, 0))
    gpu.synchronize()


def test_specials_in_a_token(gpu):
    """A NaN or an infinity costs its own block of 32 and no other."""
    cache = gpu.quantized_cache(64, 2, 4, 2)
    K = np.ones((64, 2, 2), np.float32)
    K[40, 1, 0] = np.nan
    K[3, 0, 1] = -np.inf
    gpu.cache_write_(cache, gpu.ROCArray.from_host(K), gpu.ROCArray.from_host(K), gpu.ROCArray.from_host(np.array([1, 2], np.int32)))
    out = [gpu.zeros(np.float32, (64, 2, 2, 1)) for _ in range(2)]
    gpu.cache_read_(*out, cache, gpu.ROCArray.from_host(np.array([[1]], np.int32)), gpu.ROCArray.from_host(np.array([2], np.int32)))
    for o in out:
        h = o.to_host()[..., 0]
        nan = np.zeros(h.shape, bool)
        nan[32:, 1, 0] = nan[:32, 0, 1] = True
        assert np.array_equal(np.isnan(h), nan) and (h[~nan] == 1).all()


def test_offsets_past_32_bits(gpu):
    """The last page of a cache of more than 2^32 codes."""
    d, heads, page, npages = 128, 8, 64, 66_000
    codes = gpu.ROCArray(np.int8, (d, heads, page, npages))
    scales = gpu.ROCArray(np.uint8, (4, heads, page, npages))
    assert codes.size > 1 << 32
    side = gpu.Quantized8.wrap(codes, scales)
    cache = gpu.QuantizedCache(side, gpu.Quantized8.wrap(gpu.zeros(np.int8, codes.dims), gpu.zeros(np.uint8, scales.dims)))
    x = np.random.default_rng(1).standard_normal((d, heads, 3)).astype(ref.BF16)
    X = gpu.ROCArray.from_host(x)
    slots = np.array([cache.slots, cache.slots - 1, 1], np.int64)
    gpu.cache_write_(cache, X, X, gpu.ROCArray.from_host(slots))
    out = [gpu.zeros(ref.BF16, (d, heads, page, 2)) for _ in range(2)]
    gpu.cache_read_(*out, cache, gpu.ROCArray.from_host(np.array([[npages, 1]], np.int32)), gpu.ROCArray.from_host(np.array([page, 1], np.int32)))
    gpu.synchronize()
    for o in out:
        h = o.to_host().astype(np.float64)
        want = kept(x.astype(np.float64), "int8")
        assert np.array_equal(h[:, :, page - 1, 0], want[:, :, 0]) and np.array_equal(h[:, :, page - 2, 0], want[:, :, 1])
        assert np.array_equal(h[:, :, 0, 1], want[:, :, 2])


def test_graph_replay(gpu):
    """A write (large: with the table of claims) and a read replayed with other tokens in place; two
    graphs of one stream side by side on two."""
    rng = np.random.default_rng(3)
    n, d, heads = 2500, 32, 2
    st, other = gpu.Stream(), gpu.Stream()
    with gpu.using_stream(st):
        sets = []
        for _ in range(2):
            cache = gpu.quantized_cache(d, heads, 16, 200)
            K = gpu.ROCArray.from_host(rng.standard_normal((d, heads, n)).astype(np.float32))
            slots = gpu.ROCArray.from_host((rng.permutation(3200)[:n] + 1).astype(np.int32))
            pages = gpu.ROCArray.from_host(np.arange(1, 201, dtype=np.int32).reshape(200, 1))
            lengths = gpu.ROCArray.from_host(np.array([3200], np.int32))
            out = [gpu.zeros(np.float32, (d, heads, 3200, 1)) for _ in range(2)]

            def step(cache=cache, K=K, slots=slots, pages=pages, lengths=lengths, out=out):
                gpu.cache_write_(cache, K, K, slots)
                gpu.cache_read_(*out, cache, pages, lengths)
            sets.append((cache, K, slots, out, gpu.captured(step)))
        st.synchronize()
        for round_ in range(3):
            new = []
            for cache, K, slots, out, graph in sets:
                x = rng.standard_normal((d, heads, n)).astype(np.float32)
                K.copy_from_host(x)
                new.append((x, slots.to_host()))
            st.synchronize()
            gpu.launch(sets[0][4], st)
            gpu.launch(sets[1][4], other)
            st.synchronize()
            other.synchronize()
            for (x, s), (_, _, _, out, _) in zip(new, sets):
                for o in out:
                    assert np.array_equal(o.to_host()[:, :, s - 1, 0].astype(np.float64), kept(x.astype(np.float64), "int8"))


def test_strided_indices_and_value_heads(gpu):
    """Slots, positions, pages and lengths as strided views; values of another head size; many heads, whose
    vectors of one token are more than a block's threads."""
    rng = np.random.default_rng(17)
    for dk, dv, heads in ((64, 32, 2), (128, 128, 40), (256, 64, 33)):
        cache = gpu.quantized_cache(dk, heads, 8, 6, value_dim=dv)
        n = 11
        K, V = rng.standard_normal((dk, heads, n)).astype(np.float32), rng.standard_normal((dv, heads, n)).astype(np.float32)
        slots = rng.permutation(48)[:n] + 1
        wide = np.zeros((3, n), np.int64)
        wide[1] = slots
        S = gpu.ROCArray.from_host(wide).subview(1, slice(None))
        gpu.cache_write_(cache, gpu.ROCArray.from_host(K), gpu.ROCArray.from_host(V), S)
        pages = np.zeros((2, 5, 3), np.int32)
        pages[1, :3, 1:] = np.array([[1, 6], [2, 5], [4, 3]])
        lengths = np.zeros((4, 2), np.int32)
        lengths[2] = [20, 24]
        out = [gpu.zeros(np.float32, (d, heads, 24, 2)) for d in (dk, dv)]
        gpu.cache_read_(*out, cache, gpu.ROCArray.from_host(pages).subview(1, slice(0, 3), slice(1, 3)), gpu.ROCArray.from_host(lengths).subview(2, slice(None)))
        gpu.synchronize()
        for o, x in zip(out, (K, V)):
            full = np.zeros((x.shape[0], heads, 48))
            full[:, :, slots - 1] = kept(x.astype(np.float64), "int8")
            h = o.to_host()
            for b, (table, m) in enumerate((([1, 2, 4], 20), ([6, 5, 3], 24))):
                l = np.arange(m)
                row = (np.array(table)[l // 8] - 1) * 8 + l % 8
                assert np.array_equal(h[:, :, :m, b], full[:, :, row]) and not h[:, :, m:, b].any()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_many_tokens_of_many_shapes(gpu, layout):
    """More tokens than are looked through one by one, with heads that take part of a warp, a warp, and several:
    the slots get what a call with few tokens writes there."""
    rng = np.random.default_rng(23)
    half, single = np.dtype(np.float16), np.dtype(np.float32)
    for d, dv, heads, t in ((32, 32, 1, ref.BF16), (72, 72, 3, half), (128, 64, 8, ref.BF16), (256, 256, 9, ref.BF16), (64, 64, 2, single),
                            (33, 40, 2, half), (1984, 32, 1, ref.BF16), (8192, 16, 1, half)):
        n, pages = (2500, 40) if d < 1000 else (2050, 33)
        K, V = (rng.standard_normal((k, heads, n)).astype(t) for k in (d, dv))
        slots = rng.permutation(64 * pages)[:n] + 1
        slots[rng.integers(0, n, 50)] = slots[rng.integers(0, n, 50)]
        slots[rng.integers(0, n, 20)] = 0
        positions = rng.integers(-10, 1 << 20, n)
        plan = gpu.rotary_plan(2 * (d // 3), layout=layout)
        one, many = (gpu.quantized_cache(d, heads, 64, pages, "e4m3", value_dim=dv) for _ in range(2))
        up = gpu.ROCArray.from_host
        gpu.cache_write_(many, up(K), up(V), up(slots), rotary=plan, positions=up(positions))
        for i in range(0, n, 1000):
            p = slice(i, i + 1000)
            gpu.cache_write_(one, up(np.asfortranarray(K[:, :, p])), up(np.asfortranarray(V[:, :, p])), up(slots[p]), rotary=plan, positions=up(positions[p]))
        gpu.synchronize()
        for a, b in zip(one._arrays(), many._arrays()):
            assert np.array_equal(a.to_host(), b.to_host()), (d, heads)
