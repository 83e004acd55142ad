// Rotary positions: the first `rot` elements of every head are turned in pairs by angles that grow
// with the token's position; pairs are (i, i + rot/2) or (2i, 2i+1).  The gradient is the same turn
// backwards (the adjoint of a rotation times a factor).  Element-wise over views, beside
// src/broadcast.jl:3-30 of the reference.
//
//   y_a = x_a cos - x_b sin,  y_b = x_b cos + x_a sin,  angle = position * frequency[pair]
//
// Angles are formed in the kernel from a table of frequencies in 2^-64 turns per position (rowops.cuh):
// no table of cosines is read, and a far position loses no more than its multiple of an entry's rounding.
#include "rowops.cuh"

namespace b200 {

struct RotaryArgs {
    const void* x;
    void* y;
    const void* pos;
    const uint64_t* table;
    int64_t xh, x1, x2, yh, y1, y2, p1, p2;     // element strides: head, token dimensions
    int64_t tokens, t1;
    uint32_t turn_blocks;
    int32_t d, rot, heads, chunk, turn_units, pass_units, wide, adjoint, small;     // units: threads per token
    FastDiv per_token, per_pass, first;
    float factor;
};

// A thread owns one unit of `chunk` heads of a token: V pairs (half layout; V = 1 also interleaved) or V/2
// pairs (interleaved) or V elements that pass through.  Its angles are worked out once (about 25
// instructions a pair, as much as turning three heads), and the loads of kHeads heads are on their way
// together.  Bound by HBM: 16384 tokens of 32 heads of 128 BFloat16 46 us (5.8 TB/s).
constexpr int kHeads = 4;

template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(256)
rotary_kernel(RotaryArgs a) {
    grid_dependency_wait();
    constexpr bool PAIRED = HALF || V == 1;       // two separate vectors per unit
    constexpr int P = PAIRED ? V : V / 2;
    // what turns and what passes through in blocks of their own: side by side in a warp one would wait for
    // the other
    const bool turns = blockIdx.x < a.turn_blocks;
    const int64_t n = (int64_t)(blockIdx.x - (turns ? 0 : a.turn_blocks)) * 256 + threadIdx.x;
    const int units = turns ? a.turn_units : a.pass_units;
    if (n >= a.tokens * units) return;
    const FastDiv& per_token = turns ? a.per_token : a.per_pass;
    const int64_t token = a.small ? (int64_t)per_token.div((uint32_t)n) : n / units;
    const int unit = (int)(n - token * units);
    const int64_t t2 = a.small ? (int64_t)a.first.div((uint32_t)token) : token / a.t1;
    const int64_t t1 = token - t2 * a.t1;
    const T* x = reinterpret_cast<const T*>(a.x) + t1 * a.x1 + t2 * a.x2;
    T* y = reinterpret_cast<T*>(a.y) + t1 * a.y1 + t2 * a.y2;
    const int h0 = blockIdx.y * a.chunk, h1 = min(a.heads, h0 + a.chunk);
    if (!turns) {
        const int i = a.rot + unit * V;
        for (int h = h0; h < h1; h += kHeads) {
            RawVec<T, V> r[kHeads];
#pragma unroll
            for (int k = 0; k < kHeads; ++k) if (h + k < h1) r[k] = ld_raw<T, V>(x + (h + k) * a.xh + i);
#pragma unroll
            for (int k = 0; k < kHeads; ++k) if (h + k < h1) st_raw<T, V>(y + (h + k) * a.yh + i, r[k]);
        }
        return;
    }
    // places of the two members of a pair
    const int i0 = HALF ? unit * V : V == 1 ? 2 * unit : unit * V;
    const int i1 = HALF ? i0 + a.rot / 2 : i0 + 1;
    x += i0;
    y += i0;
    RawVec<T, V> r0[kHeads], r1[kHeads];
    auto load = [&](int h) {
#pragma unroll
        for (int k = 0; k < kHeads; ++k) {
            if (h + k < h1) {
                const T* at = x + (h + k) * a.xh;
                r0[k] = ld_raw<T, V>(at);
                if constexpr (PAIRED) r1[k] = ld_raw<T, V>(at + (i1 - i0));
            }
        }
    };
    load(h0);
    const uint64_t pos = (uint64_t)load_int(a.pos, a.wide, t1 * a.p1 + t2 * a.p2);
    float sn[P], cs[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        phase_sincos(pos * a.table[unit * P + i], a.factor, sn[i], cs[i]);
        if (a.adjoint) sn[i] = -sn[i];
    }
    for (int h = h0; h < h1; h += kHeads) {
        if (h > h0) load(h);
#pragma unroll
        for (int k = 0; k < kHeads; ++k) {
            if (h + k >= h1) break;
            T* ys = y + (h + k) * a.yh;
            if constexpr (V == 1) {
                float u, v;
                unpack<T, 1>(r0[k], &u);
                unpack<T, 1>(r1[k], &v);
                const float o = fmaf(u, cs[0], -(v * sn[0])), w = fmaf(v, cs[0], u * sn[0]);
                st_raw<T, 1>(ys, pack<T, 1>(&o));
                st_raw<T, 1>(ys + (i1 - i0), pack<T, 1>(&w));
            } else if constexpr (HALF) {
                F2 u[V / 2], v[V / 2];
                unpack2<T, V>(r0[k], u);
                unpack2<T, V>(r1[k], v);
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    const F2 c = f2(cs[2 * i], cs[2 * i + 1]), s = f2(sn[2 * i], sn[2 * i + 1]), minus = f2(-sn[2 * i], -sn[2 * i + 1]);
                    const F2 o = f2_fma(u[i], c, f2_mul(v[i], minus));
                    v[i] = f2_fma(v[i], c, f2_mul(u[i], s));
                    u[i] = o;
                }
                st_raw<T, V>(ys, pack2<T, V>(u));
                st_raw<T, V>(ys + (i1 - i0), pack2<T, V>(v));
            } else {
                F2 u[V / 2];
                unpack2<T, V>(r0[k], u);
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const float2 z = f2_parts(u[i]);
                    u[i] = f2_fma(u[i], f2(cs[i]), f2_mul(f2(z.y, z.x), f2(-sn[i], sn[i])));
                }
                st_raw<T, V>(ys, pack2<T, V>(u));
            }
        }
    }
}

// Vectors of a head whose pairs do not lie vector to vector: rot/2 is no multiple of V (half layout), or
// the head turns in part (interleaved).  A thread reads its vector at once and, in half
// layout, the partners one by one; destination and source must be apart, since a vector's partners are
// other threads' vectors.  In half layout both members of a pair work out its angle, and the wait for the
// partners is what shows among the stalls: 8192 tokens of 64 heads, 26 of 80 turned, BFloat16 65 us (floor 26;
// interleaved 33), Float32 70 us (51).
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(256)
rotary_uneven_kernel(RotaryArgs a) {
    grid_dependency_wait();
    const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (n >= a.tokens * a.turn_units) return;
    const int64_t token = a.small ? (int64_t)a.per_token.div((uint32_t)n) : n / a.turn_units;
    const int i0 = (int)(n - token * a.turn_units) * V;
    const int64_t t2 = a.small ? (int64_t)a.first.div((uint32_t)token) : token / a.t1;
    const int64_t t1 = token - t2 * a.t1;
    const T* x = reinterpret_cast<const T*>(a.x) + t1 * a.x1 + t2 * a.x2;
    T* y = reinterpret_cast<T*>(a.y) + t1 * a.y1 + t2 * a.y2;
    const int h0 = blockIdx.y * a.chunk, h1 = min(a.heads, h0 + a.chunk), half = a.rot / 2;
    float sn[V], cs[V];
    if (i0 < a.rot) {
        const uint64_t pos = (uint64_t)load_int(a.pos, a.wide, t1 * a.p1 + t2 * a.p2);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int i = i0 + j;
            sn[j] = cs[j] = 0.f;
            if (i >= a.rot || (!HALF && (j & 1))) continue;
            phase_sincos(pos * a.table[HALF ? (i < half ? i : i - half) : i / 2], a.factor, sn[j], cs[j]);
            if (a.adjoint) sn[j] = -sn[j];
            if (HALF && i < half) sn[j] = -sn[j];
        }
    }
    for (int h = h0; h < h1; h += 2) {
        RawVec<T, V> r[2];
        float p[2][V];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (h + k >= h1) continue;
            const T* at = x + (h + k) * a.xh;
            r[k] = ld_raw_cached<T, V>(at + i0);
            if constexpr (HALF) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int i = i0 + j;
                    p[k][j] = i < a.rot ? Elem<T>::get(at[i < half ? i + half : i - half]) : 0.f;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (h + k >= h1) continue;
            float u[V];
            unpack<T, V>(r[k], u);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if constexpr (HALF) {
                    if (i0 + j < a.rot) u[j] = fmaf(u[j], cs[j], p[k][j] * sn[j]);
                } else if (!(j & 1) && i0 + j < a.rot) {
                    const float v = u[j + 1];
                    u[j + 1] = fmaf(v, cs[j], u[j] * sn[j]);
                    u[j] = fmaf(u[j], cs[j], -(v * sn[j]));
                }
            }
            st_raw<T, V>(y + (h + k) * a.yh + i0, pack<T, V>(u));
        }
    }
}

enum { kByElement = 0, kVectors = 1, kUneven = 2 };

template <typename T>
static cudaError_t run_rotary(b200_stream_t st, RotaryArgs a, bool half, int how, bool in_place) {
    constexpr int FV = 16 / (int)sizeof(T);
    const int v = how == kByElement ? 1 : FV;
    a.turn_units = how == kUneven ? a.d / v : half || v == 1 ? a.rot / 2 / v : a.rot / v;
    a.pass_units = how == kUneven || in_place ? 0 : (a.d - a.rot) / v;
    const int64_t n = a.tokens * (a.turn_units + a.pass_units);
    a.small = n < (int64_t)1 << 30;
    a.per_token = FastDiv((uint32_t)a.turn_units);
    a.per_pass = FastDiv((uint32_t)a.pass_units);
    a.first = FastDiv((uint32_t)(a.t1 < (int64_t)1 << 30 ? a.t1 : 1));
    // Heads per thread: up to two rounds of kHeads, then a block ends early enough for the last ones to even
    // out (16384 tokens of 32 heads of 128, half layout: all heads 52 us, 16 heads 47, 8 heads 46; of 8 heads of
    // 256: 8 heads 20 us, 4 heads 20, 2 heads 25 for the angles), fewer where that leaves SMs without work.
    const int rounds = (a.heads + 2 * kHeads - 1) / (2 * kHeads);
    a.chunk = (a.heads + rounds - 1) / rounds;
    while (a.chunk > 1 && n * ((a.heads + a.chunk - 1) / a.chunk) < (int64_t)sm_count(st->dev) * 512) a.chunk = (a.chunk + 1) / 2;
    while ((a.heads + a.chunk - 1) / a.chunk > 65535) ++a.chunk;
    cudaLaunchConfig_t cfg{};
    a.turn_blocks = (uint32_t)((a.tokens * a.turn_units + 255) / 256);
    const uint32_t pass_blocks = (uint32_t)((a.tokens * a.pass_units + 255) / 256);
    cfg.gridDim = dim3(a.turn_blocks + pass_blocks, (unsigned)((a.heads + a.chunk - 1) / a.chunk));
    cfg.blockDim = dim3(256);
    cfg.stream = st->s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = overlap_launches_enabled() ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (how == kUneven) return half ? cudaLaunchKernelEx(&cfg, rotary_uneven_kernel<T, FV, true>, a) : cudaLaunchKernelEx(&cfg, rotary_uneven_kernel<T, FV, false>, a);
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
    const bool vec = strides_ok(X) && strides_ok(Y) && d % fv == 0;
    bool in_place = X->ptr == Y->ptr;
    for (int k = 1; k < X->ndim; ++k) in_place = in_place && (X->shape[k] == 1 || X->stride[k] == Y->stride[k]);
    if (in_place && rot == 0) return B200_OK;
    // interleaved heads that turn in part go by whole vectors too: one kind of thread for all (16384 tokens of
    // 16 heads of 96 with 64 turned: 15 us, 18 with blocks apart, 24 with both kinds in a warp)
    const int how = !vec ? kByElement : half ? (rot / 2 % fv == 0 ? kVectors : in_place ? kByElement : kUneven) : rot == d ? kVectors : kUneven;
    if (a.tokens * (d / (how == kByElement ? 1 : fv)) / 256 > 0x7ffffff0) return fail(B200_TOO_LARGE, "rotary: too many tokens for one call");
    switch (X->dtype) {
        case B200_F16: B200_CUDA(run_rotary<__half>(st, a, half, how, in_place)); break;
        case B200_BF16: B200_CUDA(run_rotary<__nv_bfloat16>(st, a, half, how, in_place)); break;
        default: B200_CUDA(run_rotary<float>(st, a, half, how, in_place)); break;
    }
    return finish(st, "b200_rotary");
}
