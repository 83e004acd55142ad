// Rotary positions: the first `rot` elements of every head are turned in pairs by angles that grow
// with the token's position; pairs are (i, i + rot/2) or (2i, 2i+1).  The gradient is the same turn
// backwards (the adjoint of a rotation times a factor).  Element-wise over views, beside
// src/broadcast.jl:3-30 of the reference.
//
//   y_a = x_a cos - x_b sin,  y_b = x_b cos + x_a sin,  angle = position * frequency[pair]
//
// Angles are formed in the kernel from a table of frequencies in 2^-64 turns per position (rowops.cuh):
// no table of cosines is read, and far positions lose nothing.
#include "rowops.cuh"

namespace b200 {

struct RotaryArgs {
    const void* x;
    void* y;
    const void* pos;
    const uint64_t* table;
    int64_t xh, x1, x2, yh, y1, y2, p1, p2;     // element strides: head, token dimensions
    int64_t tokens, units;                      // units: threads per token
    int32_t d, rot, heads, chunk, turn_units, wide, adjoint, small;
    int64_t t1;
    FastDiv per_token, first;
    float factor;
};

// A thread owns one unit of every head of its share of a token: V pairs (half layout; V = 1 also
// interleaved) or V/2 pairs (interleaved) or V elements that pass through.  Its angles are computed
// once and used for `chunk` heads.
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(256)
rotary_kernel(RotaryArgs a) {
    grid_dependency_wait();
    constexpr bool PAIRED = HALF || V == 1;       // two separate vectors per unit
    constexpr int P = PAIRED ? V : V / 2;
    const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (n >= a.tokens * a.units) return;
    int64_t token;
    int unit;
    if (a.small) {
        token = a.per_token.div((uint32_t)n);
        unit = (int)((uint32_t)n - (uint32_t)token * a.per_token.d);
    } else {
        token = n / a.units;
        unit = (int)(n - token * a.units);
    }
    const int64_t t2 = a.small ? (int64_t)a.first.div((uint32_t)token) : token / a.t1;
    const int64_t t1 = token - t2 * a.t1;
    const T* x = reinterpret_cast<const T*>(a.x) + t1 * a.x1 + t2 * a.x2;
    T* y = reinterpret_cast<T*>(a.y) + t1 * a.y1 + t2 * a.y2;
    const int h0 = blockIdx.y * a.chunk, h1 = min(a.heads, h0 + a.chunk);
    if (unit >= a.turn_units) {
        const int i = a.rot + (unit - a.turn_units) * V;
        for (int h = h0; h < h1; ++h) st_raw<T, V>(y + h * a.yh + i, ld_raw<T, V>(x + h * a.xh + i));
        return;
    }
    const uint64_t pos = (uint64_t)load_int(a.pos, a.wide, t1 * a.p1 + t2 * a.p2);
    float sn[P], cs[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        phase_sincos(pos * a.table[unit * P + i], a.factor, sn[i], cs[i]);
        if (a.adjoint) sn[i] = -sn[i];
    }
    // places of the two members of a pair
    const int i0 = HALF ? unit * V : V == 1 ? 2 * unit : unit * V;
    const int i1 = HALF ? i0 + a.rot / 2 : i0 + 1;
    for (int h = h0; h < h1; ++h) {
        const T* xs = x + h * a.xh;
        T* ys = y + h * a.yh;
        if constexpr (PAIRED) {
            const RawVec<T, V> r0 = ld_raw<T, V>(xs + i0), r1 = ld_raw<T, V>(xs + i1);
            float u[V], v[V], o[V], w[V];
            unpack<T, V>(r0, u);
            unpack<T, V>(r1, v);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                o[i] = fmaf(u[i], cs[i], -(v[i] * sn[i]));
                w[i] = fmaf(v[i], cs[i], u[i] * sn[i]);
            }
            st_raw<T, V>(ys + i0, pack<T, V>(o));
            st_raw<T, V>(ys + i1, pack<T, V>(w));
        } else {
            float u[V], o[V];
            unpack<T, V>(ld_raw<T, V>(xs + i0), u);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                o[2 * i] = fmaf(u[2 * i], cs[i], -(u[2 * i + 1] * sn[i]));
                o[2 * i + 1] = fmaf(u[2 * i + 1], cs[i], u[2 * i] * sn[i]);
            }
            st_raw<T, V>(ys + i0, pack<T, V>(o));
        }
    }
}

template <typename T>
static cudaError_t run_rotary(b200_stream_t st, RotaryArgs a, bool half, bool vec, bool in_place) {
    constexpr int FV = 16 / (int)sizeof(T);
    const int v = vec ? FV : 1;
    a.turn_units = half || v == 1 ? a.rot / 2 / v : a.rot / v;
    a.units = a.turn_units + (in_place ? 0 : (a.d - a.rot) / v);
    const int64_t n = a.tokens * a.units;
    a.small = n < (int64_t)1 << 30;
    a.per_token = FastDiv((uint32_t)a.units);
    a.first = FastDiv((uint32_t)(a.t1 < (int64_t)1 << 30 ? a.t1 : 1));
    // heads per thread: as many as leave the device four waves of threads
    a.chunk = a.heads;
    while (a.chunk > 1 && n * ((a.heads + a.chunk - 1) / a.chunk) < (int64_t)sm_count(st->dev) * 2048 * 4) a.chunk = (a.chunk + 1) / 2;
    while ((a.heads + a.chunk - 1) / a.chunk > 65535) ++a.chunk;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((n + 255) / 256), (unsigned)((a.heads + a.chunk - 1) / a.chunk));
    cfg.blockDim = dim3(256);
    cfg.stream = st->s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = overlap_launches_enabled() ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (half) return v == 1 ? cudaLaunchKernelEx(&cfg, rotary_kernel<T, 1, true>, a) : cudaLaunchKernelEx(&cfg, rotary_kernel<T, FV, true>, a);
    return v == 1 ? cudaLaunchKernelEx(&cfg, rotary_kernel<T, 1, false>, a) : cudaLaunchKernelEx(&cfg, rotary_kernel<T, FV, false>, a);
}

}  // namespace b200

using namespace b200;

extern "C" int32_t b200_rotary(b200_stream_t st, const b200_tensor* Y, const b200_tensor* X, const b200_tensor* positions,
                               const b200_tensor* table, int32_t layout, double factor, int32_t adjoint) {
    B200_TRY(check_tensor(Y, "rotary destination"));
    B200_TRY(check_tensor(X, "rotary source"));
    B200_TRY(check_tensor(positions, "rotary positions"));
    B200_TRY(check_tensor(table, "rotary table"));
    if (X->ndim < 3 || X->ndim > 4) return fail(B200_INVALID_ARG, "rotary: needs (head size, heads, tokens) or (head size, heads, tokens, batch)");
    if (!same_shape(X, Y) || X->dtype != Y->dtype) return fail(B200_INVALID_ARG, "rotary: source and destination differ");
    if (!is_row_type(X->dtype)) return fail(B200_UNSUPPORTED, "rotary: Float16, BFloat16 or Float32");
    if (layout != kRotaryHalf && layout != kRotaryInterleaved) return fail(B200_UNSUPPORTED, "rotary: layout half (0) or interleaved (1)");
    if (!is_index_type(positions->dtype)) return fail(B200_UNSUPPORTED, "rotary: positions must be Int32 or Int64");
    if (table->dtype != B200_U64 || !tensor_is_contiguous(table)) return fail(B200_UNSUPPORTED, "rotary: the table must be dense UInt64");
    const int64_t d = X->shape[0], rot = 2 * tensor_numel(table), b = X->ndim == 4 ? X->shape[3] : 1;
    if (rot > d) return fail(B200_INVALID_ARG, "rotary: the table turns more elements than a head has");
    if (positions->ndim < 1 || positions->ndim > X->ndim - 2 || positions->shape[0] != X->shape[2] ||
        (positions->ndim == 2 && positions->shape[1] != b))
        return fail(B200_INVALID_ARG, "rotary: needs one position per token (or per token of one batch entry)");
    if (d > 65536 || X->shape[1] > (int64_t)1 << 24) return fail(B200_TOO_LARGE, "rotary: heads of at most 65536 elements, at most 2^24 heads");
    if ((d > 1 && X->stride[0] != 1) || (d > 1 && Y->stride[0] != 1)) return fail(B200_UNSUPPORTED, "rotary: the elements of a head must be neighbours");
    RotaryArgs a{};
    a.x = X->ptr; a.y = Y->ptr; a.pos = positions->ptr; a.table = reinterpret_cast<const uint64_t*>(table->ptr);
    a.xh = X->stride[1]; a.x1 = X->stride[2]; a.x2 = X->ndim == 4 ? X->stride[3] : 0;
    a.yh = Y->stride[1]; a.y1 = Y->stride[2]; a.y2 = Y->ndim == 4 ? Y->stride[3] : 0;
    a.p1 = positions->stride[0]; a.p2 = positions->ndim == 2 ? positions->stride[1] : 0;
    a.t1 = X->shape[2]; a.tokens = X->shape[2] * b;
    a.d = (int32_t)d; a.rot = (int32_t)rot; a.heads = (int32_t)X->shape[1];
    a.wide = positions->dtype == B200_I64; a.adjoint = adjoint != 0; a.factor = (float)factor;
    for (int k = 1; k < Y->ndim; ++k)
        if (tensor_numel(Y) > 0 && Y->shape[k] > 1 && (Y->stride[k] < d && Y->stride[k] > -d)) return fail(B200_INVALID_ARG, "rotary: heads of the destination overlap");
    B200_TRY(enter(st));
    StreamGuard guard(st);
    if (d == 0 || X->shape[1] == 0 || X->shape[2] == 0 || b == 0) return B200_OK;
    // 16-byte accesses: every head, and in half layout every half, starts on one
    const int64_t fv = X->dtype == B200_F32 ? 4 : 8;
    auto strides_ok = [&](const b200_tensor* t) {
        for (int k = 1; k < t->ndim; ++k) if (t->shape[k] > 1 && t->stride[k] % fv) return false;
        return reinterpret_cast<uintptr_t>(t->ptr) % 16 == 0;
    };
    const bool half = layout == kRotaryHalf;
    const bool vec = strides_ok(X) && strides_ok(Y) && d % fv == 0 && (half ? rot / 2 : rot) % fv == 0;
    bool in_place = X->ptr == Y->ptr;
    for (int k = 1; k < X->ndim; ++k) in_place = in_place && (X->shape[k] == 1 || X->stride[k] == Y->stride[k]);
    if (in_place && rot == 0) return B200_OK;
    if (a.tokens * (d / (vec ? fv : 1)) / 256 > 0x7ffffff0) return fail(B200_TOO_LARGE, "rotary: too many tokens for one call");
    switch (X->dtype) {
        case B200_F16: B200_CUDA(run_rotary<__half>(st, a, half, vec, in_place)); break;
        case B200_BF16: B200_CUDA(run_rotary<__nv_bfloat16>(st, a, half, vec, in_place)); break;
        default: B200_CUDA(run_rotary<float>(st, a, half, vec, in_place)); break;
    }
    return finish(st, "b200_rotary");
}
