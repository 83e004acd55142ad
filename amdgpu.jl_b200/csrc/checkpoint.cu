// Activations kept in 8 bits between the forward and the backward pass: rows to codes and back, and
// the activations silu and gelu, plain or gated, that keep their inputs in 8 bits on the way forward
// and take their gradient from them.  Beside the element-wise expressions of src/broadcast.jl:3-30.
//
//   silu(a) = a s(a), s(u) = 1/(1+exp(-u));  gelu(a) = a s(2u), u = sqrt(2/pi) (a + 0.044715 a^3)
//   y = f(a) or f(a) b;  da = dy f'(a) or dy b f'(a), db = dy f(a), with a and b out of 8 bits
#include "rowops.cuh"

namespace b200 {

enum { kSilu = 0, kGelu = 1 };

// f(a) and f'(a).  With e = exp(-|u|) and r = 1/(1+e) the sigmoid is r or e r and its derivative
// e r^2: no cancellation, and nothing overflows.  16-bit results take the fast exponential and
// reciprocal (a few ulp of binary32), binary32 results the full ones.
template <bool FAST>
__device__ __forceinline__ void sigmoid_parts(float u, float& q, float& dq) {
    const float e = FAST ? __expf(-fabsf(u)) : expf(-fabsf(u));
    const float r = FAST ? __fdividef(1.f, 1.f + e) : 1.f / (1.f + e);
    q = u >= 0.f ? r : e * r;
    if (u != u) q = u;
    dq = e * r * r;
}
template <bool FAST, bool DERIV>
__device__ __forceinline__ void activate(int act, float a, float& f, float& df) {
    // beyond 128 the sigmoid is 0 or 1 in binary32 and its derivative 0
    const float ac = fminf(fmaxf(a, -128.f), 128.f);
    float q, dq;
    if (act == kSilu) {
        sigmoid_parts<FAST>(a, q, dq);
        if constexpr (DERIV) df = fmaf(ac, dq, q);
    } else {
        const float c = 1.5957691216057308f;                     // 2 sqrt(2/pi)
        const float a2 = ac * ac;
        const float u = a == a ? c * ac * fmaf(0.044715f, a2, 1.f) : a;
        sigmoid_parts<FAST>(u, q, dq);
        if constexpr (DERIV) df = fmaf(ac * dq, c * fmaf(3.f * 0.044715f, a2, 1.f), q);
    }
    f = fmaxf(a, -128.f) * q;                                    // -128 times 0: the limit at -infinity
    if (a != a) f = a;
}

// ---- rows of whole 8-bit blocks ------------------------------------------------------------------
// Rows dealt out as vectors of V elements, each row filled up to whole blocks so that the 32/V lanes
// of a block are neighbours in one warp.  `flat`: the rows have no gaps and d is a multiple of 32, so
// they are one long row and no index is divided.
struct RowsArgs {
    const void *a, *b, *dy;
    void *y, *da, *db;
    uint8_t *qa, *sa, *qb, *sb;
    int64_t lda, ldb, lddy, ldy, ldda, lddb, rows, d, blocks, slots;   // slots: rows * vectors per filled row
    FastDiv per_row;                                                   // vectors per filled row
    int32_t e4m3, act, flat, small;
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

template <int V>
__device__ __forceinline__ void keep(const RowsArgs& a, const Slot& s, const float* v, uint8_t* q, uint8_t* sc) {
    const uint32_t e = scale_byte(block_amax<V>(v), a.e4m3);
    if (!s.in) return;
    st_raw<uint8_t, V>(q + s.row * a.d + s.i, encode<V>(v, e, a.e4m3));
    if (s.i % kBlock == 0) sc[s.row * a.blocks + s.i / kBlock] = (uint8_t)e;
}

template <typename T, int V>
__global__ void __launch_bounds__(256)
quantize_kernel(RowsArgs a) {
    grid_dependency_wait();
    const int64_t step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t n0 = (int64_t)blockIdx.x * blockDim.x; n0 < a.slots; n0 += step) {
        const Slot s = slot_of<V>(a, n0 + threadIdx.x);
        RawVec<T, V> r{};
        if (s.in) r = ld_raw<T, V>(reinterpret_cast<const T*>(a.a) + s.row * a.lda + s.i);
        float v[V];
        unpack<T, V>(r, v);
        keep<V>(a, s, v, a.qa, a.sa);
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(256)
dequantize_kernel(RowsArgs a) {
    grid_dependency_wait();
    const int64_t step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t n = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; n < a.slots; n += step) {
        const Slot s = slot_of<V>(a, n);
        if (!s.in) continue;
        float v[V];
        decode_as<T, V>(ld_raw<uint8_t, V>(a.qa + s.row * a.d + s.i), a.sa[s.row * a.blocks + s.i / kBlock], a.e4m3, v);
        st_raw<T, V>(reinterpret_cast<T*>(a.y) + s.row * a.ldy + s.i, pack<T, V>(v));
    }
}

template <typename T, int V, bool GATED>
__global__ void __launch_bounds__(256)
activation_kernel(RowsArgs a) {
    grid_dependency_wait();
    const int64_t step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t n0 = (int64_t)blockIdx.x * blockDim.x; n0 < a.slots; n0 += step) {
        const Slot s = slot_of<V>(a, n0 + threadIdx.x);
        RawVec<T, V> ra{}, rb{};
        if (s.in) {
            ra = ld_raw<T, V>(reinterpret_cast<const T*>(a.a) + s.row * a.lda + s.i);
            if constexpr (GATED) rb = ld_raw<T, V>(reinterpret_cast<const T*>(a.b) + s.row * a.ldb + s.i);
        }
        float v[V], g[V], o[V];
        unpack<T, V>(ra, v);
        if constexpr (GATED) unpack<T, V>(rb, g);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float df;
            activate<sizeof(T) == 2, false>(a.act, v[i], o[i], df);
            if constexpr (GATED) o[i] *= g[i];
        }
        if (s.in) st_raw<T, V>(reinterpret_cast<T*>(a.y) + s.row * a.ldy + s.i, pack<T, V>(o));
        if (a.qa) keep<V>(a, s, v, a.qa, a.sa);
        if constexpr (GATED) { if (a.qb) keep<V>(a, s, g, a.qb, a.sb); }
    }
}

template <typename T, int V, bool GATED, bool KEPT>
__global__ void __launch_bounds__(256)
activation_backward_kernel(RowsArgs a) {
    grid_dependency_wait();
    const int64_t step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t n = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; n < a.slots; n += step) {
        const Slot s = slot_of<V>(a, n);
        if (!s.in) continue;
        float v[V], g[V], dy[V], o[V];
        unpack<T, V>(ld_raw<T, V>(reinterpret_cast<const T*>(a.dy) + s.row * a.lddy + s.i), dy);
        if constexpr (KEPT) {
            const int64_t c = s.row * a.d + s.i, b = s.row * a.blocks + s.i / kBlock;
            decode_as<T, V>(ld_raw<uint8_t, V>(a.qa + c), a.sa[b], a.e4m3, v);
            if constexpr (GATED) decode_as<T, V>(ld_raw<uint8_t, V>(a.qb + c), a.sb[b], a.e4m3, g);
        } else {
            unpack<T, V>(ld_raw<T, V>(reinterpret_cast<const T*>(a.a) + s.row * a.lda + s.i), v);
            if constexpr (GATED) unpack<T, V>(ld_raw<T, V>(reinterpret_cast<const T*>(a.b) + s.row * a.ldb + s.i), g);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float f, df;
            activate<sizeof(T) == 2, true>(a.act, v[i], f, df);
            o[i] = dy[i] * df;
            if constexpr (GATED) { o[i] *= g[i]; g[i] = dy[i] * f; }
        }
        st_raw<T, V>(reinterpret_cast<T*>(a.da) + s.row * a.ldda + s.i, pack<T, V>(o));
        if constexpr (GATED) st_raw<T, V>(reinterpret_cast<T*>(a.db) + s.row * a.lddb + s.i, pack<T, V>(g));
    }
}

// ---- host ---------------------------------------------------------------------------------------
struct RowsCall {
    RowsArgs a{};
    bool dense = true, aligned = true;
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
        aligned = aligned && reinterpret_cast<uintptr_t>(Q->ptr) % 8 == 0;
        *q = (uint8_t*)Q->ptr;
        *s = (uint8_t*)S->ptr;
        return B200_OK;
    }
    // Vector width, and the slots for it; 0: nothing to do.
    int plan() {
        if (a.rows == 0 || a.d == 0) return 0;
        const int full = dtype == B200_F32 ? 4 : 8;
        const int v = aligned && a.d % full == 0 ? full : 1;
        a.blocks = row_blocks(a.d);
        a.flat = dense && a.d % kBlock == 0;
        if (a.flat) { a.d *= a.rows; a.blocks *= a.rows; a.rows = 1; }
        const int64_t per = a.blocks * (kBlock / v);
        a.slots = per * a.rows;
        // slots past the end are looked up too, up to one grid's worth of threads
        a.small = !a.flat && a.slots < (int64_t)1 << 30 && per < (int64_t)1 << 30;
        a.per_row = FastDiv((uint32_t)(per < (int64_t)1 << 31 ? per : 1));
        return v;
    }
};

template <typename K>
static cudaError_t launch_rows(b200_stream_t st, K kernel, const RowsArgs& a) {
    return launch_overlapped(kernel, balanced_grid((a.slots + 255) / 256, resident_blocks(kernel, 256, 0, st->dev)), 256u, 0, st->s, a);
}
// f(element type, vector width) for the type and width of the call
template <typename F>
static cudaError_t by_type(int32_t dtype, int v, F f) {
    switch (dtype) {
        case B200_F16: return v == 1 ? f(__half{}, std::integral_constant<int, 1>{}) : f(__half{}, std::integral_constant<int, 8>{});
        case B200_BF16: return v == 1 ? f(__nv_bfloat16{}, std::integral_constant<int, 1>{}) : f(__nv_bfloat16{}, std::integral_constant<int, 8>{});
        default: return v == 1 ? f(float{}, std::integral_constant<int, 1>{}) : f(float{}, std::integral_constant<int, 4>{});
    }
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
    B200_CUDA(by_type(c.dtype, v, [&](auto t, auto w) { return launch_rows(st, quantize_kernel<decltype(t), decltype(w)::value>, c.a); }));
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
    B200_CUDA(by_type(c.dtype, v, [&](auto t, auto w) { return launch_rows(st, dequantize_kernel<decltype(t), decltype(w)::value>, c.a); }));
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
    const int v = c.plan();
    if (v) B200_TRY(row_limit(c));
    B200_TRY(enter(st));
    StreamGuard guard(st);
    if (!v) return B200_OK;
    B200_CUDA(by_type(c.dtype, v, [&](auto t, auto w) {
        using T = decltype(t);
        constexpr int V = decltype(w)::value;
        return B ? launch_rows(st, activation_kernel<T, V, true>, c.a) : launch_rows(st, activation_kernel<T, V, false>, c.a);
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
    B200_CUDA(by_type(c.dtype, v, [&](auto t, auto w) {
        using T = decltype(t);
        constexpr int V = decltype(w)::value;
        if (gated) return A ? launch_rows(st, activation_backward_kernel<T, V, true, false>, c.a) : launch_rows(st, activation_backward_kernel<T, V, true, true>, c.a);
        return A ? launch_rows(st, activation_backward_kernel<T, V, false, false>, c.a) : launch_rows(st, activation_backward_kernel<T, V, false, true>, c.a);
    }));
    return finish(st, "b200_activation_backward");
}
