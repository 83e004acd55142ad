// Activations kept in 8 bits between the forward and the backward pass: rows to codes and back, and
// the activations silu and gelu, plain or gated, that keep their inputs in 8 bits on the way forward
// and take their gradient from them.  Beside the element-wise expressions of src/broadcast.jl:3-30.
//
//   silu(a) = a s(a), s(u) = 1/(1+exp(-u));  gelu(a) = a s(2u), u = sqrt(2/pi) (a + 0.044715 a^3)
//   y = f(a) or f(a) b;  da = dy f'(a) or dy b f'(a), db = dy f(a), with a and b out of 8 bits
#include "rowops.cuh"

namespace b200 {

enum { kSilu = 0, kGelu = 1 };
enum { kNoCodes = 0 };

// f(a) and f'(a) for binary32 results.  With e = exp(-|u|) and r = 1/(1+e) the sigmoid is r or e r and its
// derivative e r^2: no cancellation, and nothing overflows.  Beyond 128 the sigmoid is 0 or 1 in binary32
// and its derivative 0: the clamps give the limits at the infinities, and let a NaN through.
template <int ACT>
__device__ __forceinline__ void activate(float a, float& f, float& df) {
    const float low = jl_max(a, -128.f), ac = jl_min(low, 128.f), a2 = ac * ac;
    const float c = 1.5957691216057308f;                         // 2 sqrt(2/pi)
    const float u = ACT == kSilu ? ac : c * ac * fmaf(0.044715f, a2, 1.f);
    const float e = expf(-fabsf(u)), r = 1.f / (1.f + e);
    const float q = u >= 0.f ? r : e * r, dq = e * r * r;
    const float du = ACT == kSilu ? 1.f : c * fmaf(3.f * 0.044715f, a2, 1.f);
    f = low * q;
    df = fmaf(ac * dq, du, q);
}
// The same for 16-bit results, two at a time, with the fast base-2 exponential and reciprocal (both good
// to a few ulp of binary32; the exponent's product adds half an ulp per unit of |u|).  q: sigmoid(u),
// rest: 1 - q, for x = -u log2(e) / 2: the square of exp(-|u|/2) reaches down to the subnormals, which a
// BFloat16 product shows, while the exponential itself stays where its fast form works.
__device__ __forceinline__ void fast_sigmoid(float x, float& q, float& rest) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-fabsf(x)));
    e *= e;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    const float er = e * r;
    q = x <= 0.f ? r : er;
    rest = x <= 0.f ? er : r;
}
// FINITE: there are no infinities among the inputs (they come out of 8 bits).
template <int ACT, bool DERIV, bool FINITE>
__device__ __forceinline__ void activate2(F2 a, F2& f, F2& df) {
    const float half_log2e = 0.7213475204444817f, c = 1.5957691216057308f;
    F2 low = a, ac = a, minus, du = f2(1.f);
    if constexpr (!FINITE) {
        const float2 v = f2_parts(a);
        ac = low = f2(jl_max(v.x, -128.f), jl_max(v.y, -128.f));
    }
    if constexpr (ACT == kGelu || (DERIV && !FINITE)) {          // a^2 must not overflow, nor infinity meet zero
        const float2 l = f2_parts(low);
        ac = FINITE ? f2(jl_min(jl_max(l.x, -128.f), 128.f), jl_min(jl_max(l.y, -128.f), 128.f)) : f2(jl_min(l.x, 128.f), jl_min(l.y, 128.f));
    }
    if constexpr (ACT == kSilu) {
        minus = f2_mul(ac, f2(-half_log2e));
    } else {
        const F2 a2 = f2_mul(ac, ac);
        minus = f2_mul(ac, f2_fma(a2, f2(-half_log2e * c * 0.044715f), f2(-half_log2e * c)));
        if constexpr (DERIV) du = f2_fma(a2, f2(c * 3.f * 0.044715f), f2(c));
    }
    const float2 m = f2_parts(minus);
    float qx, qy, rx, ry;
    fast_sigmoid(m.x, qx, rx);
    fast_sigmoid(m.y, qy, ry);
    const F2 q = f2(qx, qy);
    f = f2_mul(low, q);
    if constexpr (DERIV) {
        const F2 rest = f2(rx, ry);
        const F2 slope = ACT == kSilu ? f2_mul(ac, rest) : f2_mul(f2_mul(ac, du), rest);
        df = f2_fma(q, slope, q);
    }
}

// ---- rows of any alignment --------------------------------------------------------------------------
// Rows are dealt out as vectors of V elements, each row filled up to whole blocks so that the 32/V lanes of
// a block are neighbours in one warp.  `flat`: the rows have no gaps and d is a multiple of 32, so they are
// one long row and no index is divided.
struct RowsArgs {
    const void *a, *b, *dy;
    void *y, *da, *db;
    uint8_t *qa, *sa, *qb, *sb;
    int64_t lda, ldb, lddy, ldy, ldda, lddb, rows, d, blocks, slots, total;   // slots: rows * vectors per filled row
    FastDiv per_row;                                                   // vectors per filled row (dense rows of any width: d)
    int32_t e4m3, act, flat, small, wide;                              // wide: 32-byte accesses are aligned
};

struct Slot { int64_t row; int64_t i; bool in; };
template <int V>
__device__ __forceinline__ Slot slot_of(const RowsArgs& a, int64_t n) {
    Slot s;
    if (a.flat) { s.row = 0; s.i = n * V; }
    else if (a.small) { s.row = a.per_row.div((uint32_t)n); s.i = (int64_t)((uint32_t)n - (uint32_t)s.row * a.per_row.d) * V; }
    else { s.row = n / a.per_row.d; s.i = (n - s.row * a.per_row.d) * V; }
    s.in = n < a.slots && s.i < a.d;
    return s;
}

// One element per lane and block of 32, kAny blocks per warp whose loads are on their way together.  Bound by
// instruction issue (quantising 32764 rows of 4101 BFloat16, 2 apart: issue slots 81 % taken, 86 instructions a
// lane and element, HBM at 12 %); for rows that lie apart off 16 bytes, rows shorter than a block, and in place.
constexpr int kAny = 8;

__device__ __forceinline__ void any_slots(const RowsArgs& a, Slot s[kAny]) {
    const int64_t first = ((int64_t)blockIdx.x * 8 + threadIdx.x / 32) * kAny;      // the warp's first block
#pragma unroll
    for (int k = 0; k < kAny; ++k) s[k] = slot_of<1>(a, (first + k) * kBlock + threadIdx.x % 32);
}
template <typename T>
__device__ __forceinline__ void any_load(const void* p, int64_t ld, const Slot s[kAny], float* v) {
    T r[kAny];
#pragma unroll
    for (int k = 0; k < kAny; ++k) {
        r[k] = Elem<T>::put(0.f);
        if (s[k].in) r[k] = reinterpret_cast<const T*>(p)[s[k].row * ld + s[k].i];
    }
#pragma unroll
    for (int k = 0; k < kAny; ++k) v[k] = Elem<T>::get(r[k]);
}
template <typename T>
__device__ __forceinline__ void any_store(void* p, int64_t ld, const Slot s[kAny], const float* v) {
#pragma unroll
    for (int k = 0; k < kAny; ++k) if (s[k].in) reinterpret_cast<T*>(p)[s[k].row * ld + s[k].i] = Elem<T>::put(v[k]);
}
// Magnitudes compare like their bits, NaN above all.
__device__ __forceinline__ void any_keep(const RowsArgs& a, const Slot s[kAny], const float* v, uint8_t* q, uint8_t* sc) {
#pragma unroll
    for (int k = 0; k < kAny; ++k) {
        const uint32_t m = __reduce_max_sync(0xffffffffu, s[k].in ? __float_as_uint(v[k]) & 0x7fffffffu : 0u);
        const uint32_t e = scale_byte(__uint_as_float(m), a.e4m3);
        if (!s[k].in) continue;
        q[s[k].row * a.d + s[k].i] = encode<1>(v + k, e, a.e4m3);
        if (threadIdx.x % 32 == 0) sc[s[k].row * a.blocks + s[k].i / kBlock] = (uint8_t)e;
    }
}
template <typename T>
__device__ __forceinline__ void any_restore(const RowsArgs& a, const Slot s[kAny], const uint8_t* q, const uint8_t* sc, float* v) {
    uint8_t c[kAny];
    uint32_t e[kAny];
#pragma unroll
    for (int k = 0; k < kAny; ++k) {
        c[k] = 0;
        e[k] = 0;
        if (!s[k].in) continue;
        c[k] = q[s[k].row * a.d + s[k].i];
        e[k] = sc[s[k].row * a.blocks + s[k].i / kBlock];
    }
#pragma unroll
    for (int k = 0; k < kAny; ++k) decode_as<T, 1>(c[k], e[k], a.e4m3, v + k);
}
// f and f' of kAny values.
template <typename T, bool DERIV, bool FINITE>
__device__ __forceinline__ void any_activate(int act, const float* v, float* f, float* df) {
#pragma unroll
    for (int k = 0; k < kAny; k += 2) {
        if constexpr (sizeof(T) == 2) {
            F2 x, y = 0;
            if (act == kSilu) activate2<kSilu, DERIV, FINITE>(f2(v[k], v[k + 1]), x, y);
            else activate2<kGelu, DERIV, FINITE>(f2(v[k], v[k + 1]), x, y);
            const float2 fx = f2_parts(x), dx = f2_parts(y);
            f[k] = fx.x; f[k + 1] = fx.y;
            df[k] = dx.x; df[k + 1] = dx.y;
        } else {
#pragma unroll
            for (int j = k; j < k + 2; ++j) {
                if (act == kSilu) activate<kSilu>(v[j], f[j], df[j]);
                else activate<kGelu>(v[j], f[j], df[j]);
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256)
quantize_any_kernel(RowsArgs a) {
    grid_dependency_wait();
    Slot s[kAny];
    any_slots(a, s);
    float v[kAny];
    any_load<T>(a.a, a.lda, s, v);
    any_keep(a, s, v, a.qa, a.sa);
}

template <typename T>
__global__ void __launch_bounds__(256)
dequantize_any_kernel(RowsArgs a) {
    grid_dependency_wait();
    Slot s[kAny];
    any_slots(a, s);
    float v[kAny];
    any_restore<T>(a, s, a.qa, a.sa, v);
    any_store<T>(a.y, a.ldy, s, v);
}

template <typename T, bool GATED>
__global__ void __launch_bounds__(256)
activation_any_kernel(RowsArgs a) {
    grid_dependency_wait();
    Slot s[kAny];
    any_slots(a, s);
    float v[kAny], g[kAny], o[kAny], df[kAny];
    any_load<T>(a.a, a.lda, s, v);
    if constexpr (GATED) any_load<T>(a.b, a.ldb, s, g);
    any_activate<T, false, false>(a.act, v, o, df);
    if constexpr (GATED) {
#pragma unroll
        for (int k = 0; k < kAny; ++k) o[k] *= g[k];
    }
    any_store<T>(a.y, a.ldy, s, o);
    if (a.qa) any_keep(a, s, v, a.qa, a.sa);
    if constexpr (GATED) { if (a.qb) any_keep(a, s, g, a.qb, a.sb); }
}

template <typename T, bool GATED, bool KEPT>
__global__ void __launch_bounds__(256)
activation_backward_any_kernel(RowsArgs a) {
    grid_dependency_wait();
    Slot s[kAny];
    any_slots(a, s);
    float dy[kAny], v[kAny], g[kAny], f[kAny], df[kAny];
    any_load<T>(a.dy, a.lddy, s, dy);
    if constexpr (KEPT) {
        any_restore<T>(a, s, a.qa, a.sa, v);
        if constexpr (GATED) any_restore<T>(a, s, a.qb, a.sb, g);
    } else {
        any_load<T>(a.a, a.lda, s, v);
        if constexpr (GATED) any_load<T>(a.b, a.ldb, s, g);
    }
    any_activate<T, true, KEPT>(a.act, v, f, df);
#pragma unroll
    for (int k = 0; k < kAny; ++k) {
        v[k] = dy[k] * df[k];
        if constexpr (GATED) { v[k] *= g[k]; g[k] = dy[k] * f[k]; }
    }
    any_store<T>(a.da, a.ldda, s, v);
    if constexpr (GATED) any_store<T>(a.db, a.lddb, s, g);
}

// ---- vectors ------------------------------------------------------------------------------------------
// The kernels above with V elements per thread, 32 bytes of rows and 16 (8) of codes: two (four) threads
// share a block of 32, so its scale is worked out twice instead of 32 times, and with the loads in order the
// arithmetic around the codes is what bounds these kernels.  A slot per thread and 256 per block, so that
// blocks that start as others end mix reads and writes.  Activation, format and gate are fixed at compile
// time.  One B200, 8192 x 8192 BFloat16, both operands of a gated silu in Int8: forward 84 us (6.4 TB/s),
// gradient 93 us (5.8 TB/s); with 16-byte accesses, a runtime format and the exponential's full range 121 and
// 136 us.
template <int V, int F>
__device__ __forceinline__ void keep2(const RowsArgs& a, const Slot& s, const F2* v, uint8_t* q, uint8_t* sc) {
    const uint32_t e = scale_byte(block_amax2<V>(v, s.in), F == kE4M3);
    if (!s.in) return;
    st_raw<uint8_t, V>(q + s.row * a.d + s.i, encode2<V>(v, e, F == kE4M3));
    if (s.i % kBlock == 0) sc[s.row * a.blocks + s.i / kBlock] = (uint8_t)e;
}
template <typename T, int V>
__device__ __forceinline__ RawVec<T, V> fetch(const void* p, int64_t ld, const Slot& s, bool wide) {
    RawVec<T, V> r{};
    if (s.in) r = ld_raw32(reinterpret_cast<const T*>(p) + s.row * ld + s.i, wide);
    return r;
}
template <typename T, int V>
__device__ __forceinline__ void store(void* p, int64_t ld, const Slot& s, const F2* v, bool wide) {
    if (s.in) st_raw32(reinterpret_cast<T*>(p) + s.row * ld + s.i, pack2<T, V>(v), wide);
}
template <int V>
__device__ __forceinline__ Slot my_slot(const RowsArgs& a) { return slot_of<V>(a, (int64_t)blockIdx.x * 256 + threadIdx.x); }

template <typename T, int V, int F>
__global__ void __launch_bounds__(256)
quantize_vec_kernel(RowsArgs a) {
    grid_dependency_wait();
    const Slot s = my_slot<V>(a);
    F2 v[V / 2];
    unpack2<T, V>(fetch<T, V>(a.a, a.lda, s, a.wide), v);
    keep2<V, F>(a, s, v, a.qa, a.sa);
}

template <int V>
__device__ __forceinline__ RawVec<uint8_t, V> fetch_codes(const RowsArgs& a, const uint8_t* q, const uint8_t* sc, const Slot& s, uint32_t& e) {
    RawVec<uint8_t, V> r{};
    e = 0;
    if (s.in) {
        // volatile, like the 32-byte loads: all of a thread's loads leave before the first is used
        const uint8_t *p = q + s.row * a.d + s.i, *pe = sc + s.row * a.blocks + s.i / kBlock;
        asm volatile("ld.global.u8 %0, [%1];" : "=r"(e) : "l"(pe));
        if constexpr (V == 16) asm volatile("ld.global.cs.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
        else asm volatile("ld.global.cs.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
    }
    return r;
}
// Four codes.  PLAIN: the block's scale is far from overflowing anything; else values past the type's range
// saturate, and NaN comes out.
template <typename T, int F, bool PLAIN>
__device__ __forceinline__ void decode_quad(uint32_t w, uint32_t e, F2* v) {
    if constexpr (PLAIN) {
        decode2<4>(w, e, F == kE4M3, v);
    } else {
        float x[4];
        decode_as<T, 4>(w, e, F == kE4M3, x);
        v[0] = f2(x[0], x[1]);
        v[1] = f2(x[2], x[3]);
    }
}

template <typename T, int V, int F>
__global__ void __launch_bounds__(256)
dequantize_vec_kernel(RowsArgs a) {
    grid_dependency_wait();
    const Slot s = my_slot<V>(a);
    uint32_t e;
    const RawVec<uint8_t, V> r = fetch_codes<V>(a, a.qa, a.sa, s, e);
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
    F2 v[V / 2];
    if (plain_scale<T>(e)) {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) decode_quad<T, F, true>(w[i], e, v + 2 * i);
    } else {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) decode_quad<T, F, false>(w[i], e, v + 2 * i);
    }
    store<T, V>(a.y, a.ldy, s, v, a.wide);
}

template <int ACT, bool FAST, bool DERIV, bool FINITE>
__device__ __forceinline__ void activate_pair(F2 a, F2& f, F2& df) {
    if constexpr (FAST) {
        activate2<ACT, DERIV, FINITE>(a, f, df);
    } else {
        const float2 v = f2_parts(a);
        float fx, fy, dx, dy;
        activate<ACT>(v.x, fx, dx);
        activate<ACT>(v.y, fy, dy);
        f = f2(fx, fy);
        df = f2(dx, dy);
    }
}

template <typename T, int V, int ACT, bool GATED, int F>
__global__ void __launch_bounds__(256)
activation_vec_kernel(RowsArgs a) {
    grid_dependency_wait();
    const Slot s = my_slot<V>(a);
    const RawVec<T, V> ra = fetch<T, V>(a.a, a.lda, s, a.wide);
    RawVec<T, V> rb{};
    if constexpr (GATED) rb = fetch<T, V>(a.b, a.ldb, s, a.wide);
    F2 v[V / 2], g[V / 2], o[V / 2];
    unpack2<T, V>(ra, v);
    if constexpr (GATED) unpack2<T, V>(rb, g);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        F2 df;
        activate_pair<ACT, sizeof(T) == 2, false, false>(v[i], o[i], df);
        if constexpr (GATED) o[i] = f2_mul(o[i], g[i]);
    }
    store<T, V>(a.y, a.ldy, s, o, a.wide);
    if constexpr (F != kNoCodes) {
        if (a.qa) keep2<V, F>(a, s, v, a.qa, a.sa);
        if constexpr (GATED) { if (a.qb) keep2<V, F>(a, s, g, a.qb, a.sb); }
    }
}

// Four elements of the gradient at a time, so that few values live at once.
template <typename T, int V, int ACT, bool GATED, int F>
__global__ void __launch_bounds__(256)
activation_backward_vec_kernel(RowsArgs a) {
    grid_dependency_wait();
    const Slot s = my_slot<V>(a);
    const RawVec<T, V> rd = fetch<T, V>(a.dy, a.lddy, s, a.wide);
    RawVec<T, V> ra{}, rb{};
    RawVec<uint8_t, V> ca{}, cb{};
    uint32_t ea = 0, eb = 0;
    if constexpr (F != kNoCodes) {
        ca = fetch_codes<V>(a, a.qa, a.sa, s, ea);
        if constexpr (GATED) cb = fetch_codes<V>(a, a.qb, a.sb, s, eb);
    } else {
        ra = fetch<T, V>(a.a, a.lda, s, a.wide);
        if constexpr (GATED) rb = fetch<T, V>(a.b, a.ldb, s, a.wide);
    }
    RawVec<T, V> oa, ob;
    auto quads = [&](auto plain) {
        constexpr int W = (int)sizeof(T);                // words of four elements
        [[maybe_unused]] const uint32_t *wd = reinterpret_cast<const uint32_t*>(&rd), *wa = reinterpret_cast<const uint32_t*>(&ra), *wb = reinterpret_cast<const uint32_t*>(&rb);
        [[maybe_unused]] const uint32_t *qa = reinterpret_cast<const uint32_t*>(&ca), *qb = reinterpret_cast<const uint32_t*>(&cb);
        [[maybe_unused]] uint32_t *pa = reinterpret_cast<uint32_t*>(&oa), *pb = reinterpret_cast<uint32_t*>(&ob);
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            [[maybe_unused]] F2 dy[2], v[2], g[2];
            unpack2<T, 4>(*reinterpret_cast<const RawVec<T, 4>*>(wd + W * i), dy);
            if constexpr (F != kNoCodes) {
                decode_quad<T, F, decltype(plain)::value>(qa[i], ea, v);
                if constexpr (GATED) decode_quad<T, F, decltype(plain)::value>(qb[i], eb, g);
            } else {
                unpack2<T, 4>(*reinterpret_cast<const RawVec<T, 4>*>(wa + W * i), v);
                if constexpr (GATED) unpack2<T, 4>(*reinterpret_cast<const RawVec<T, 4>*>(wb + W * i), g);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                F2 f, df;
                activate_pair<ACT, sizeof(T) == 2, true, F != kNoCodes>(v[j], f, df);
                v[j] = f2_mul(dy[j], df);
                if constexpr (GATED) { v[j] = f2_mul(v[j], g[j]); g[j] = f2_mul(dy[j], f); }
            }
            *reinterpret_cast<RawVec<T, 4>*>(pa + W * i) = pack2<T, 4>(v);
            if constexpr (GATED) *reinterpret_cast<RawVec<T, 4>*>(pb + W * i) = pack2<T, 4>(g);
        }
    };
    if (F == kNoCodes || (plain_scale<T>(ea) && plain_scale<T>(eb))) quads(std::true_type{});
    else quads(std::false_type{});
    if (!s.in) return;
    st_raw32(reinterpret_cast<T*>(a.da) + s.row * a.ldda + s.i, oa, a.wide);
    if constexpr (GATED) st_raw32(reinterpret_cast<T*>(a.db) + s.row * a.lddb + s.i, ob, a.wide);
}

// ---- dense rows of any width --------------------------------------------------------------------------
// Rows without gaps are one long row for the loads and stores, so its vectors are aligned whatever d is; but
// the blocks of 32 start anew with every row and begin and end inside vectors.  A vector of V <= 16 elements
// meets three blocks at most (d >= 32: only a row's last block is shorter than 32), whose scale bytes are
// neighbours.  A block's largest magnitude is collected in shared memory over the tile's threads; of the
// blocks that reach over the tile's ends the missing elements are read as well (31 at most either side).
// Where codes are involved instructions and the two barriers around the maxima hold it up (quantising: issue
// slots 64 % taken, 24 instructions a thread and element, HBM at 33 %).  One B200, 8191 x 4101 BFloat16, Int8: quantised in
// 34 us and restored in 19 us, gated silu with both operands kept 93 us, its gradient 70 us (an element per
// lane: 96, 78, 224 and 188 us; with a third block thought of in every vector 39, 22, 105 and 73 us); without
// codes 29 and 51 us.
struct Cuts {
    int64_t f, scale;          // first element, its block
    int b1, b2, n;             // elements of the first block, of the first two; elements in the array
    bool opens;                // the first block starts here
};
template <int V>
__device__ __forceinline__ Cuts cuts_of(const RowsArgs& a, int64_t f) {
    Cuts c;
    c.f = f;
    const int64_t left = a.total - f, d = a.per_row.d;
    c.n = left <= 0 ? 0 : left < V ? (int)left : V;
    const int64_t row = a.small ? (int64_t)a.per_row.div((uint32_t)f) : f / d;
    int64_t i = f - row * d;
    c.scale = row * a.blocks + i / kBlock;
    c.opens = i % kBlock == 0;
    c.b1 = (int)min((int64_t)kBlock - i % kBlock, d - i);
    i += c.b1;
    if (i == d) i = 0;
    c.b2 = c.b1 + (int)min((int64_t)kBlock, d - i);
    return c;
}
template <typename T, int V>
__device__ __forceinline__ RawVec<T, V> cut_load(const void* p, const Cuts& c, bool wide) {
    const T* at = reinterpret_cast<const T*>(p) + c.f;
    if (c.n == V) return ld_raw32(at, wide);
    RawVec<T, V> r{};
#pragma unroll
    for (int j = 0; j < V; ++j) if (j < c.n) reinterpret_cast<T*>(&r)[j] = at[j];
    return r;
}
template <typename T, int V>
__device__ __forceinline__ void cut_store(void* p, const Cuts& c, const RawVec<T, V>& r, bool wide) {
    T* at = reinterpret_cast<T*>(p) + c.f;
    if (c.n == V) { st_raw32(at, r, wide); return; }
#pragma unroll
    for (int j = 0; j < V; ++j) if (j < c.n) at[j] = reinterpret_cast<const T*>(&r)[j];
}
// TWO: no vector of the warp meets a third block (a row ends in few of them); f(constant) for the warp's case.
__device__ __forceinline__ bool cut_two(const Cuts& c) { return __all_sync(0xffffffffu, c.b2 >= c.n); }     // by whole warps
template <bool TWO, typename X>
__device__ __forceinline__ X cut_pick(const Cuts& c, int j, X x0, X x1, X x2) { return j < c.b1 ? x0 : TWO || j < c.b2 ? x1 : x2; }
template <typename F>
__device__ __forceinline__ void cut_cases(bool two, F f) {
    if (two) f(std::true_type{});
    else f(std::false_type{});
}

// Codes and scale bytes of the tile's rows; `most`: room for the magnitudes of the tile's blocks.
constexpr int kCutBlocks = 288;          // of 256 vectors of 16 elements: 2 blocks per 33 elements, and the ends
template <typename T, int V, int F>
__device__ __forceinline__ void cut_keep(const RowsArgs& a, const Cuts& c, const RawVec<T, V>& r, const T* p, uint8_t* q, uint8_t* sc, uint32_t* most) {
    const int64_t f0 = (int64_t)blockIdx.x * 256 * V;
    const Cuts lo = cuts_of<V>(a, f0);
    for (int i = threadIdx.x; i < kCutBlocks; i += 256) most[i] = 0;
    __syncthreads();
    F2 v[V / 2];
    unpack2<T, V>(r, v);
    const bool two = cut_two(c);
    uint32_t m[3] = {0, 0, 0};
    cut_cases(two, [&](auto t) {
#pragma unroll
        for (int j = 0; j < V; ++j) {                         // elements past the array are zeros
            const float2 x = f2_parts(v[j / 2]);
            const uint32_t bits = __float_as_uint(j & 1 ? x.y : x.x) & 0x7fffffffu;
            if (j < c.b1) m[0] = max(m[0], bits);
            else if (decltype(t)::value || j < c.b2) m[1] = max(m[1], bits);
            else m[2] = max(m[2], bits);
        }
    });
    const int at = (int)(c.scale - lo.scale);
    if (c.n > 0) {
        atomicMax(most + at, m[0]);
        if (c.b1 < c.n) atomicMax(most + at + 1, m[1]);
        if (c.b2 < c.n) atomicMax(most + at + 2, m[2]);
    }
    if (threadIdx.x < 32) {                                   // before the tile
        const int64_t row = lo.scale / a.blocks;
        const int64_t start = row * (int64_t)a.per_row.d + (lo.scale - row * a.blocks) * kBlock;
        if (start + threadIdx.x < f0) atomicMax(most, __float_as_uint(Elem<T>::get(p[start + threadIdx.x])) & 0x7fffffffu);
    } else if (threadIdx.x < 64) {                            // behind it
        const int64_t end = f0 + 256 * V;
        if (end < a.total) {
            const Cuts hi = cuts_of<V>(a, end);
            const int lane = threadIdx.x - 32;
            if (!hi.opens && lane < hi.b1 && end + lane < a.total)
                atomicMax(most + (hi.scale - lo.scale), __float_as_uint(Elem<T>::get(p[end + lane])) & 0x7fffffffu);
        }
    }
    __syncthreads();
    if (c.n == 0) return;
    uint32_t e[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        e[k] = scale_byte(__uint_as_float(most[at + k]), F == kE4M3);
        const int first = k == 0 ? 0 : k == 1 ? c.b1 : c.b2;
        if (first < c.n && (k > 0 || c.opens)) sc[c.scale + k] = (uint8_t)e[k];
    }
    RawVec<uint8_t, V> codes{};
    if (max(e[0], max(e[1], e[2])) < 255u) {
        const float i0 = inverse_scale(e[0]), i1 = inverse_scale(e[1]), i2 = inverse_scale(e[2]);
        uint32_t* w = reinterpret_cast<uint32_t*>(&codes);
        cut_cases(two, [&](auto t) {
            constexpr bool TWO = decltype(t)::value;
#pragma unroll
            for (int j = 0; j < V; j += 4) {
                const F2 p0 = f2(cut_pick<TWO>(c, j, i0, i1, i2), cut_pick<TWO>(c, j + 1, i0, i1, i2)), p1 = f2(cut_pick<TWO>(c, j + 2, i0, i1, i2), cut_pick<TWO>(c, j + 3, i0, i1, i2));
                if constexpr (F == kE4M3) {
                    const float2 x = f2_parts(f2_mul(v[j / 2], p0)), y = f2_parts(f2_mul(v[j / 2 + 1], p1));
                    w[j / 4] = e4m3_pair(x.x, x.y) | e4m3_pair(y.x, y.y) << 16;
                } else {
                    const F2 magic = f2(12582912.f);
                    const float2 x = f2_parts(f2_fma(v[j / 2], p0, magic)), y = f2_parts(f2_fma(v[j / 2 + 1], p1, magic));
                    w[j / 4] = __byte_perm(__byte_perm(__float_as_uint(x.x), __float_as_uint(x.y), 0x0040), __byte_perm(__float_as_uint(y.x), __float_as_uint(y.y), 0x0040), 0x5410);
                }
            }
        });
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float2 x = f2_parts(v[j / 2]);
            const float one = j & 1 ? x.y : x.x;
            reinterpret_cast<uint8_t*>(&codes)[j] = encode<1>(&one, cut_pick<false>(c, j, e[0], e[1], e[2]), F == kE4M3);
        }
    }
    uint8_t* to = q + c.f;
    if (c.n == V) {
        st_raw<uint8_t, V>(to, codes);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) if (j < c.n) to[j] = reinterpret_cast<const uint8_t*>(&codes)[j];
    }
}
template <typename T, int V, int F>
__device__ __forceinline__ void cut_restore(const Cuts& c, bool two, const uint8_t* q, const uint8_t* sc, F2* v) {
    RawVec<uint8_t, V> r{};
    const uint8_t* at = q + c.f;
    if (c.n == V) {
        r = ld_raw<uint8_t, V>(at);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) if (j < c.n) reinterpret_cast<uint8_t*>(&r)[j] = at[j];
    }
    const uint32_t e0 = sc[c.scale], e1 = c.b1 < c.n ? sc[c.scale + 1] : e0, e2 = c.b2 < c.n ? sc[c.scale + 2] : e0;
    if (plain_scale<T>(max(e0, max(e1, e2)))) {
        const float s0 = scale_value(e0), s1 = scale_value(e1), s2 = scale_value(e2);
        decode2<V>(r, 127u, F == kE4M3, v);                   // at scale one
        cut_cases(two, [&](auto t) {
            constexpr bool TWO = decltype(t)::value;
#pragma unroll
            for (int j = 0; j < V; j += 2) v[j / 2] = f2_mul(v[j / 2], f2(cut_pick<TWO>(c, j, s0, s1, s2), cut_pick<TWO>(c, j + 1, s0, s1, s2)));
        });
    } else {
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            float x[2];
            decode_as<T, 1>(reinterpret_cast<const uint8_t*>(&r)[j], cut_pick<false>(c, j, e0, e1, e2), F == kE4M3, x);
            decode_as<T, 1>(reinterpret_cast<const uint8_t*>(&r)[j + 1], cut_pick<false>(c, j + 1, e0, e1, e2), F == kE4M3, x + 1);
            v[j / 2] = f2(x[0], x[1]);
        }
    }
}

template <typename T, int V, int F>
__global__ void __launch_bounds__(256)
quantize_cut_kernel(RowsArgs a) {
    __shared__ uint32_t most[kCutBlocks];
    grid_dependency_wait();
    const Cuts c = cuts_of<V>(a, ((int64_t)blockIdx.x * 256 + threadIdx.x) * V);
    cut_keep<T, V, F>(a, c, cut_load<T, V>(a.a, c, a.wide), reinterpret_cast<const T*>(a.a), a.qa, a.sa, most);
}
template <typename T, int V, int F>
__global__ void __launch_bounds__(256)
dequantize_cut_kernel(RowsArgs a) {
    grid_dependency_wait();
    const Cuts c = cuts_of<V>(a, ((int64_t)blockIdx.x * 256 + threadIdx.x) * V);
    const bool two = cut_two(c);
    if (c.n == 0) return;
    F2 v[V / 2];
    cut_restore<T, V, F>(c, two, a.qa, a.sa, v);
    cut_store<T, V>(a.y, c, pack2<T, V>(v), a.wide);
}
template <typename T, int V, int ACT, bool GATED, int F>
__global__ void __launch_bounds__(256)
activation_cut_kernel(RowsArgs a) {
    __shared__ uint32_t most[GATED ? 2 : 1][F == kNoCodes ? 1 : kCutBlocks];
    grid_dependency_wait();
    const Cuts c = cuts_of<V>(a, ((int64_t)blockIdx.x * 256 + threadIdx.x) * V);
    const RawVec<T, V> ra = cut_load<T, V>(a.a, c, a.wide);
    RawVec<T, V> rb{};
    if constexpr (GATED) rb = cut_load<T, V>(a.b, c, a.wide);
    F2 v[V / 2], g[V / 2];
    unpack2<T, V>(ra, v);
    if constexpr (GATED) unpack2<T, V>(rb, g);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        F2 f, df;
        activate_pair<ACT, sizeof(T) == 2, false, false>(v[i], f, df);
        v[i] = GATED ? f2_mul(f, g[i]) : f;
    }
    cut_store<T, V>(a.y, c, pack2<T, V>(v), a.wide);
    if constexpr (F != kNoCodes) {
        if (a.qa) cut_keep<T, V, F>(a, c, ra, reinterpret_cast<const T*>(a.a), a.qa, a.sa, most[0]);
        if constexpr (GATED) { if (a.qb) cut_keep<T, V, F>(a, c, rb, reinterpret_cast<const T*>(a.b), a.qb, a.sb, most[1]); }
    }
}
template <typename T, int V, int ACT, bool GATED, int F>
__global__ void __launch_bounds__(256)
activation_backward_cut_kernel(RowsArgs a) {
    grid_dependency_wait();
    const Cuts c = cuts_of<V>(a, ((int64_t)blockIdx.x * 256 + threadIdx.x) * V);
    [[maybe_unused]] const bool two = F == kNoCodes || cut_two(c);
    if (c.n == 0) return;
    const RawVec<T, V> rd = cut_load<T, V>(a.dy, c, a.wide);
    F2 dy[V / 2], v[V / 2], g[V / 2];
    if constexpr (F != kNoCodes) {
        cut_restore<T, V, F>(c, two, a.qa, a.sa, v);
        if constexpr (GATED) cut_restore<T, V, F>(c, two, a.qb, a.sb, g);
    } else {
        unpack2<T, V>(cut_load<T, V>(a.a, c, a.wide), v);
        if constexpr (GATED) unpack2<T, V>(cut_load<T, V>(a.b, c, a.wide), g);
    }
    unpack2<T, V>(rd, dy);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        F2 f, df;
        activate_pair<ACT, sizeof(T) == 2, true, F != kNoCodes>(v[i], f, df);
        v[i] = f2_mul(dy[i], df);
        if constexpr (GATED) { v[i] = f2_mul(v[i], g[i]); g[i] = f2_mul(dy[i], f); }
    }
    cut_store<T, V>(a.da, c, pack2<T, V>(v), a.wide);
    if constexpr (GATED) cut_store<T, V>(a.db, c, pack2<T, V>(g), a.wide);
}

// ---- host ---------------------------------------------------------------------------------------
enum { kCut = -1 };

struct RowsCall {
    RowsArgs a{};
    bool dense = true, aligned = true, aligned32 = true;       // of every row; below: of the arrays' beginnings
    bool base = true, base32 = true, apart = true;             // apart: nothing is written over what a neighbour reads
    int32_t dtype = -1;

    int32_t in(const b200_tensor* t, const b200_tensor* like, const char* name, const void** p, int64_t* ld) {
        RowView v;
        B200_TRY(row_view(t, 1, name, &v));
        return add(t, like, name, v, const_cast<void**>(p), ld);
    }
    int32_t out(const b200_tensor* t, const b200_tensor* like, const char* name, void** p, int64_t* ld) {
        RowView v;
        B200_TRY(row_view_out(t, 1, name, &v));
        return add(t, like, name, v, p, ld);
    }
    int32_t add(const b200_tensor* t, const b200_tensor* like, const char* name, const RowView& v, void** p, int64_t* ld) {
        if (!is_row_type(v.dtype)) return fail(B200_UNSUPPORTED, "%s: Float16, BFloat16 or Float32 rows", name);
        if (dtype >= 0 && v.dtype != dtype) return fail(B200_INVALID_ARG, "%s: the operands differ in element type", name);
        if (like && !same_shape(t, like)) return fail(B200_INVALID_ARG, "%s: the operands differ in shape", name);
        dtype = v.dtype;
        a.rows = v.rows;
        a.d = v.d;
        dense = dense && (v.rows <= 1 || v.ld == v.d);
        aligned = aligned && rows_aligned(v, 16);
        aligned32 = aligned32 && rows_aligned(v, 32);
        base = base && reinterpret_cast<uintptr_t>(v.p) % 16 == 0;
        base32 = base32 && reinterpret_cast<uintptr_t>(v.p) % 32 == 0;
        *p = v.p;
        *ld = v.ld;
        return B200_OK;
    }
    int32_t codes(const b200_tensor* Q, const b200_tensor* S, const b200_tensor* like, const char* name, uint8_t** q, uint8_t** s, bool first) {
        B200_TRY(check_codes(Q, S, name));
        if (like && !same_shape(Q, like)) return fail(B200_INVALID_ARG, "%s: differs in shape from the rows", name);
        if (!tensor_is_contiguous(Q) || !tensor_is_contiguous(S)) return fail(B200_UNSUPPORTED, "%s: must be dense", name);
        const int32_t e4m3 = Q->dtype == B200_U8;
        if (!first && e4m3 != a.e4m3) return fail(B200_INVALID_ARG, "%s: one call keeps both operands in one format", name);
        a.e4m3 = e4m3;
        base = base && reinterpret_cast<uintptr_t>(Q->ptr) % 16 == 0;
        aligned = aligned && base;
        *q = (uint8_t*)Q->ptr;
        *s = (uint8_t*)S->ptr;
        return B200_OK;
    }
    int format() const { return !(a.qa || a.qb) ? (int)kNoCodes : a.e4m3 ? (int)kE4M3 : (int)kInt8; }
    // Vector width, and the slots for it (kCut: dense rows of any width); 0: nothing to do.
    int plan() {
        if (a.rows == 0 || a.d == 0) return 0;
        const int full = dtype == B200_F32 ? 8 : 16;
        const int v = aligned && a.d % full == 0 ? full : 1;
        a.wide = aligned32;
        a.total = a.rows * a.d;
        if (v == 1 && dense && base && apart && a.d >= kBlock && a.d <= 0x7fffffff) {
            a.wide = base32;
            a.blocks = row_blocks(a.d);
            a.slots = (a.total + full - 1) / full;
            a.small = a.total < (int64_t)0x7fff0000;
            a.per_row = FastDiv((uint32_t)a.d);
            return kCut;
        }
        a.blocks = row_blocks(a.d);
        a.flat = dense && a.d % kBlock == 0;
        if (a.flat) { a.d *= a.rows; a.blocks *= a.rows; a.rows = 1; }
        const int64_t per = a.blocks * (kBlock / v);
        a.slots = per * a.rows;
        // slots past the end are looked up too, up to one grid's worth of threads
        a.small = !a.flat && a.slots < (int64_t)1 << 30;
        a.per_row = FastDiv((uint32_t)(per < (int64_t)1 << 31 ? per : 1));
        return v;
    }
};

template <typename K>
static cudaError_t launch_any(b200_stream_t st, K kernel, const RowsArgs& a) {
    return launch_overlapped(kernel, (unsigned)((a.slots + 256 * kAny - 1) / (256 * kAny)), 256u, 0, st->s, a);
}
template <typename K>
static cudaError_t launch_tiles(b200_stream_t st, K kernel, const RowsArgs& a) {
    return launch_overlapped(kernel, (unsigned)((a.slots + 255) / 256), 256u, 0, st->s, a);
}
// f(element type, vector width) for the element type of the call
template <typename F>
static cudaError_t by_type(int32_t dtype, F f) {
    switch (dtype) {
        case B200_F16: return f(__half{}, std::integral_constant<int, 16>{});
        case B200_BF16: return f(__nv_bfloat16{}, std::integral_constant<int, 16>{});
        default: return f(float{}, std::integral_constant<int, 8>{});
    }
}
// f(constant) for one of the formats, activations, ...
template <int... Values, typename F>
static cudaError_t by_value(int value, F f) {
    cudaError_t e = cudaErrorInvalidValue;
    (void)((value == Values && ((e = f(std::integral_constant<int, Values>{})), true)) || ...);
    return e;
}

}  // namespace b200

using namespace b200;

static int32_t row_limit(const RowsCall& c) {
    // a row that is not part of one long dense row is counted in 32 bits
    return !c.a.flat && c.a.blocks > (int64_t)0x3ffffff ? fail(B200_TOO_LARGE, "rows of at most 2^31-1 elements") : B200_OK;
}

extern "C" int32_t b200_quantize(b200_stream_t st, const b200_tensor* Q, const b200_tensor* S, const b200_tensor* X) {
    RowsCall c;
    B200_TRY(c.in(X, nullptr, "quantize source", &c.a.a, &c.a.lda));
    B200_TRY(c.codes(Q, S, X, "quantize destination", &c.a.qa, &c.a.sa, true));
    const int v = c.plan();
    if (v) B200_TRY(row_limit(c));
    B200_TRY(enter(st));
    StreamGuard guard(st);
    if (!v) return B200_OK;
    B200_CUDA(by_type(c.dtype, [&](auto t, auto w) {
        using T = decltype(t);
        if (v == 1) return launch_any(st, quantize_any_kernel<T>, c.a);
        return by_value<kInt8, kE4M3>(c.format(), [&](auto f) {
            constexpr int V = decltype(w)::value, F = decltype(f)::value;
            return v == kCut ? launch_tiles(st, quantize_cut_kernel<T, V, F>, c.a) : launch_tiles(st, quantize_vec_kernel<T, V, F>, c.a);
        });
    }));
    return finish(st, "b200_quantize");
}

extern "C" int32_t b200_dequantize(b200_stream_t st, const b200_tensor* X, const b200_tensor* Q, const b200_tensor* S) {
    RowsCall c;
    B200_TRY(c.out(X, nullptr, "dequantize destination", &c.a.y, &c.a.ldy));
    B200_TRY(c.codes(Q, S, X, "dequantize source", &c.a.qa, &c.a.sa, true));
    const int v = c.plan();
    if (v) B200_TRY(row_limit(c));
    B200_TRY(enter(st));
    StreamGuard guard(st);
    if (!v) return B200_OK;
    B200_CUDA(by_type(c.dtype, [&](auto t, auto w) {
        using T = decltype(t);
        if (v == 1) return launch_any(st, dequantize_any_kernel<T>, c.a);
        return by_value<kInt8, kE4M3>(c.format(), [&](auto f) {
            constexpr int V = decltype(w)::value, F = decltype(f)::value;
            return v == kCut ? launch_tiles(st, dequantize_cut_kernel<T, V, F>, c.a) : launch_tiles(st, dequantize_vec_kernel<T, V, F>, c.a);
        });
    }));
    return finish(st, "b200_dequantize");
}

extern "C" int32_t b200_activation(b200_stream_t st, int32_t act, const b200_tensor* Y, const b200_tensor* A, const b200_tensor* B,
                                   const b200_tensor* QA, const b200_tensor* SA, const b200_tensor* QB, const b200_tensor* SB) {
    if (act != kSilu && act != kGelu) return fail(B200_UNSUPPORTED, "activation: silu (0) or gelu (1)");
    if ((QA != nullptr) != (SA != nullptr) || (QB != nullptr) != (SB != nullptr))
        return fail(B200_INVALID_ARG, "activation: codes and scales belong together");
    if (QB && !B) return fail(B200_INVALID_ARG, "activation: codes of a gate, but no gate");
    RowsCall c;
    c.a.act = act;
    B200_TRY(c.in(A, nullptr, "activation source", &c.a.a, &c.a.lda));
    if (B) B200_TRY(c.in(B, A, "activation gate", &c.a.b, &c.a.ldb));
    B200_TRY(c.out(Y, A, "activation destination", &c.a.y, &c.a.ldy));
    if (QA) B200_TRY(c.codes(QA, SA, A, "activation checkpoint", &c.a.qa, &c.a.sa, true));
    if (QB) B200_TRY(c.codes(QB, SB, A, "gate checkpoint", &c.a.qb, &c.a.sb, !QA));
    c.apart = !(QA || QB) || (c.a.y != c.a.a && c.a.y != c.a.b);
    const int v = c.plan();
    if (v) B200_TRY(row_limit(c));
    B200_TRY(enter(st));
    StreamGuard guard(st);
    if (!v) return B200_OK;
    B200_CUDA(by_type(c.dtype, [&](auto t, auto w) {
        using T = decltype(t);
        constexpr int V = decltype(w)::value;
        if (v == 1) return B ? launch_any(st, activation_any_kernel<T, true>, c.a) : launch_any(st, activation_any_kernel<T, false>, c.a);
        return by_value<kSilu, kGelu>(act, [&](auto f) {
            constexpr int ACT = decltype(f)::value;
            return by_value<kNoCodes, kInt8, kE4M3>(c.format(), [&](auto k) {
                constexpr int F = decltype(k)::value;
                if (v == kCut) return B ? launch_tiles(st, activation_cut_kernel<T, V, ACT, true, F>, c.a) : launch_tiles(st, activation_cut_kernel<T, V, ACT, false, F>, c.a);
                return B ? launch_tiles(st, activation_vec_kernel<T, V, ACT, true, F>, c.a) : launch_tiles(st, activation_vec_kernel<T, V, ACT, false, F>, c.a);
            });
        });
    }));
    return finish(st, "b200_activation");
}

extern "C" int32_t b200_activation_backward(b200_stream_t st, int32_t act, const b200_tensor* dA, const b200_tensor* dB, const b200_tensor* dY,
                                            const b200_tensor* A, const b200_tensor* B, const b200_tensor* QA, const b200_tensor* SA,
                                            const b200_tensor* QB, const b200_tensor* SB) {
    if (act != kSilu && act != kGelu) return fail(B200_UNSUPPORTED, "activation gradient: silu (0) or gelu (1)");
    if ((QA != nullptr) != (SA != nullptr) || (QB != nullptr) != (SB != nullptr))
        return fail(B200_INVALID_ARG, "activation gradient: codes and scales belong together");
    if ((A != nullptr) == (QA != nullptr)) return fail(B200_INVALID_ARG, "activation gradient: needs the input or its codes, one of the two");
    const bool gated = dB != nullptr;
    if (gated ? (A ? !B || QB : !QB || B) : (B || QB))
        return fail(B200_INVALID_ARG, "activation gradient: a gate needs dB, and comes in the form of the input (array or codes)");
    RowsCall c;
    c.a.act = act;
    B200_TRY(c.in(dY, nullptr, "activation gradient", &c.a.dy, &c.a.lddy));
    B200_TRY(c.out(dA, dY, "activation gradient destination", &c.a.da, &c.a.ldda));
    if (gated) B200_TRY(c.out(dB, dY, "gate gradient destination", &c.a.db, &c.a.lddb));
    if (A) {
        B200_TRY(c.in(A, dY, "activation source", &c.a.a, &c.a.lda));
        if (gated) B200_TRY(c.in(B, dY, "activation gate", &c.a.b, &c.a.ldb));
    } else {
        B200_TRY(c.codes(QA, SA, dY, "activation checkpoint", &c.a.qa, &c.a.sa, true));
        if (gated) B200_TRY(c.codes(QB, SB, dY, "gate checkpoint", &c.a.qb, &c.a.sb, false));
    }
    const int v = c.plan();
    if (v) B200_TRY(row_limit(c));
    B200_TRY(enter(st));
    StreamGuard guard(st);
    if (!v) return B200_OK;
    B200_CUDA(by_type(c.dtype, [&](auto t, auto w) {
        using T = decltype(t);
        constexpr int V = decltype(w)::value;
        if (v == 1) {
            if (gated) return A ? launch_any(st, activation_backward_any_kernel<T, true, false>, c.a) : launch_any(st, activation_backward_any_kernel<T, true, true>, c.a);
            return A ? launch_any(st, activation_backward_any_kernel<T, false, false>, c.a) : launch_any(st, activation_backward_any_kernel<T, false, true>, c.a);
        }
        return by_value<kSilu, kGelu>(act, [&](auto f) {
            constexpr int ACT = decltype(f)::value;
            return by_value<kNoCodes, kInt8, kE4M3>(c.format(), [&](auto k) {
                constexpr int F = decltype(k)::value;
                if (v == kCut)
                    return gated ? launch_tiles(st, activation_backward_cut_kernel<T, V, ACT, true, F>, c.a)
                                 : launch_tiles(st, activation_backward_cut_kernel<T, V, ACT, false, F>, c.a);
                return gated ? launch_tiles(st, activation_backward_vec_kernel<T, V, ACT, true, F>, c.a)
                             : launch_tiles(st, activation_backward_vec_kernel<T, V, ACT, false, F>, c.a);
            });
        });
    }));
    return finish(st, "b200_activation_backward");
}
