// Shared by the row operators (layer norm, 8-bit checkpoints, rotary positions, quantised cache):
// rows of a column-major array as (pointer, row stride), vector accesses with conversion to
// binary32, and the 8-bit row codec.
#pragma once
#include "common.cuh"

namespace b200 {

// ---- rows ------------------------------------------------------------------------------------
// An array seen as `rows` rows of `d` neighbouring elements, `ld` elements apart: the first `lead`
// dimensions are one row (dense), the others count the rows and must collapse to one stride.
struct RowView {
    void*   p;
    int64_t rows, d, ld;
    int32_t dtype;
};

inline int32_t row_view(const b200_tensor* t, int lead, const char* name, RowView* out) {
    B200_TRY(check_tensor(t, name));
    if (lead > t->ndim) return fail(B200_INVALID_ARG, "%s: needs at least %d dimensions", name, lead);
    int64_t d = 1, rows = 1;
    for (int k = 0; k < lead; ++k) {
        if (t->shape[k] > 1 && t->stride[k] != d) return fail(B200_UNSUPPORTED, "%s: the elements of a row must be neighbours", name);
        d *= t->shape[k];
    }
    int64_t ld = 0;
    for (int k = lead; k < t->ndim; ++k) {
        if (t->shape[k] == 1) continue;
        if (rows == 1) ld = t->stride[k];
        else if (t->shape[k] > 0 && t->stride[k] != ld * rows)
            return fail(B200_UNSUPPORTED, "%s: the row dimensions must collapse to one stride", name);
        rows *= t->shape[k];
    }
    if (rows == 1) ld = d;
    if (ld < 0) return fail(B200_UNSUPPORTED, "%s: negative row stride", name);
    *out = RowView{t->ptr, rows, d, ld, t->dtype};
    return B200_OK;
}
// Rows of a destination must not overlap.
inline int32_t row_view_out(const b200_tensor* t, int lead, const char* name, RowView* out) {
    B200_TRY(row_view(t, lead, name, out));
    if (out->rows > 1 && out->ld < out->d) return fail(B200_INVALID_ARG, "%s: rows of a destination overlap", name);
    return B200_OK;
}
inline bool same_shape(const b200_tensor* a, const b200_tensor* b) {
    if (a->ndim != b->ndim) return false;
    for (int k = 0; k < a->ndim; ++k) if (a->shape[k] != b->shape[k]) return false;
    return true;
}
inline bool is_row_type(int32_t dt) { return dt == B200_F16 || dt == B200_BF16 || dt == B200_F32; }
// Every row starts on a multiple of `bytes`.
inline bool rows_aligned(const RowView& v, size_t bytes) {
    return reinterpret_cast<uintptr_t>(v.p) % bytes == 0 && (v.rows <= 1 || (size_t)v.ld * dtype_size(v.dtype) % bytes == 0);
}

// 8-bit form of an array: codes (Int8, or UInt8 holding e4m3) of the same shape, and one scale
// byte per 32 elements of the first dimension.
constexpr int kBlock = 32;
inline int64_t row_blocks(int64_t d) { return (d + kBlock - 1) / kBlock; }
inline int32_t check_codes(const b200_tensor* Q, const b200_tensor* S, const char* name) {
    B200_TRY(check_tensor(Q, name));
    B200_TRY(check_tensor(S, name));
    if (Q->dtype != B200_I8 && Q->dtype != B200_U8) return fail(B200_UNSUPPORTED, "%s: codes are Int8, or UInt8 for e4m3", name);
    if (S->dtype != B200_U8) return fail(B200_UNSUPPORTED, "%s: scales are UInt8", name);
    if (Q->ndim < 1 || S->ndim != Q->ndim || S->shape[0] != row_blocks(Q->shape[0]))
        return fail(B200_INVALID_ARG, "%s: the scales need one byte per %d elements of the first dimension", name, kBlock);
    for (int k = 1; k < Q->ndim; ++k)
        if (S->shape[k] != Q->shape[k]) return fail(B200_INVALID_ARG, "%s: codes and scales differ in shape", name);
    return B200_OK;
}

// Quotients of numbers below 2^31 by one divisor: q = (mulhi(n, m) + n) >> s (Granlund and
// Montgomery 1994).
struct FastDiv {
    uint32_t d, m, s;
    FastDiv() = default;
    explicit FastDiv(uint32_t div) : d(div ? div : 1), m(0), s(0) {
        while (s < 31 && (1u << s) < d) ++s;
        m = (uint32_t)(((uint64_t(1) << 32) * ((uint64_t(1) << s) - d)) / d + 1);
    }
#ifdef __CUDACC__
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
#endif
};

enum { kInt8 = 1, kE4M3 = 2 };          // formats as template arguments

#ifdef __CUDACC__
// ---- vectors of elements -------------------------------------------------------------------------
template <int BYTES> struct RawOfBytes;
template <> struct RawOfBytes<1> { using type = uint8_t; };
template <> struct RawOfBytes<2> { using type = uint16_t; };
template <> struct RawOfBytes<4> { using type = uint32_t; };
template <> struct RawOfBytes<8> { using type = uint2; };
template <> struct RawOfBytes<16> { using type = uint4; };
struct alignas(16) Raw32 { uint4 lo, hi; };
template <> struct RawOfBytes<32> { using type = Raw32; };
template <typename T, int V> using RawVec = typename RawOfBytes<(int)sizeof(T) * V>::type;

template <typename T, int V>
__device__ __forceinline__ RawVec<T, V> ld_raw(const T* p) { return __ldcs(reinterpret_cast<const RawVec<T, V>*>(p)); }
// (Plain loads for what is read again: a non-coherent load could be moved up past the wait for the
// kernel in front, grid_dependency_wait.)
template <typename T, int V>
__device__ __forceinline__ RawVec<T, V> ld_raw_cached(const T* p) { return *reinterpret_cast<const RawVec<T, V>*>(p); }
template <typename T, int V>
__device__ __forceinline__ void st_raw(T* p, RawVec<T, V> r) { __stcs(reinterpret_cast<RawVec<T, V>*>(p), r); }

// 32 bytes: one access where the address allows it (sm_100), else two.
__device__ __forceinline__ Raw32 ld_raw32(const void* p, bool aligned32) {
    Raw32 r;
    if (aligned32) {
        asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(r.lo.x), "=r"(r.lo.y), "=r"(r.lo.z), "=r"(r.lo.w), "=r"(r.hi.x), "=r"(r.hi.y), "=r"(r.hi.z), "=r"(r.hi.w) : "l"(p));
    } else {
        r.lo = __ldcs(reinterpret_cast<const uint4*>(p));
        r.hi = __ldcs(reinterpret_cast<const uint4*>(p) + 1);
    }
    return r;
}
__device__ __forceinline__ void st_raw32(void* p, const Raw32& r, bool aligned32) {
    if (aligned32) {
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                     ::"l"(p), "r"(r.lo.x), "r"(r.lo.y), "r"(r.lo.z), "r"(r.lo.w), "r"(r.hi.x), "r"(r.hi.y), "r"(r.hi.z), "r"(r.hi.w) : "memory");
    } else {
        __stcs(reinterpret_cast<uint4*>(p), r.lo);
        __stcs(reinterpret_cast<uint4*>(p) + 1, r.hi);
    }
}

// Element types by storage: two 16-bit floats share a word.
template <typename T> struct Elem;
template <> struct Elem<float> {
    static __device__ __forceinline__ float get(float x) { return x; }
    static __device__ __forceinline__ float put(float x) { return x; }
    static constexpr float kMax = 3.402823466e38f;
};
template <> struct Elem<__half> {
    static __device__ __forceinline__ float get(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half put(float x) { return __float2half_rn(x); }
    static __device__ __forceinline__ float2 get2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ uint32_t put2(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
    static constexpr float kMax = 65504.f;
};
template <> struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float get(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 put(float x) { return __float2bfloat16_rn(x); }
    static __device__ __forceinline__ float2 get2(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
    static __device__ __forceinline__ uint32_t put2(float a, float b) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
    static constexpr float kMax = 3.389531390e38f;
};

template <typename T, int V>
__device__ __forceinline__ void unpack(const RawVec<T, V>& r, float* v) {
    if constexpr (V == 1) {
        v[0] = Elem<T>::get(*reinterpret_cast<const T*>(&r));
    } else {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = __uint_as_float(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const float2 f = Elem<T>::get2(w[i]);
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        }
    }
}
template <typename T, int V>
__device__ __forceinline__ RawVec<T, V> pack(const float* v) {
    RawVec<T, V> r;
    if constexpr (V == 1) {
        *reinterpret_cast<T*>(&r) = Elem<T>::put(v[0]);
    } else {
        uint32_t* w = reinterpret_cast<uint32_t*>(&r);
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < V; ++i) w[i] = __float_as_uint(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) w[i] = Elem<T>::put2(v[2 * i], v[2 * i + 1]);
        }
    }
    return r;
}

// ---- pairs of binary32 ------------------------------------------------------------------------------
// sm_100 issues one instruction for two neighbouring lanes' worth of binary32 arithmetic; the row
// kernels spend their time on instructions once their loads are in flight, so they work in pairs.
using F2 = unsigned long long;
__device__ __forceinline__ F2 f2(float lo, float hi) { F2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi)); return r; }
__device__ __forceinline__ F2 f2(float both) { return f2(both, both); }
__device__ __forceinline__ float2 f2_parts(F2 v) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v)); return r; }
__device__ __forceinline__ float f2_total(F2 v) { const float2 r = f2_parts(v); return r.x + r.y; }
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) { F2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ F2 f2_mul(F2 a, F2 b) { F2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) { F2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
// Largest magnitude of three, NaN if there is one.
__device__ __forceinline__ float amax3(float a, float b, float c) { float r; asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }

template <typename T, int V>
__device__ __forceinline__ void unpack2(const RawVec<T, V>& r, F2* v) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        if constexpr (sizeof(T) == 4) {
            v[i] = f2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        } else {
            const float2 f = Elem<T>::get2(w[i]);
            v[i] = f2(f.x, f.y);
        }
    }
}
template <typename T, int V>
__device__ __forceinline__ RawVec<T, V> pack2(const F2* v) {
    RawVec<T, V> r;
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        const float2 f = f2_parts(v[i]);
        if constexpr (sizeof(T) == 4) { w[2 * i] = __float_as_uint(f.x); w[2 * i + 1] = __float_as_uint(f.y); }
        else w[i] = Elem<T>::put2(f.x, f.y);
    }
    return r;
}

// ---- 8-bit codec --------------------------------------------------------------------------------
// A block of 32 values shares the scale 2^(e-127): the smallest power of two, at least 2^-127, that
// brings the largest magnitude to 127 (Int8) or 448 (e4m3).  Value over scale is exact, so a code is
// rounded once, to nearest even, and every implementation gets the same bits.  A block that holds an
// infinity or a NaN has e = 255 and codes 0 and reads back as NaN.
//
// e from the bits of the largest magnitude: its exponent less that of the largest code, one more
// when its mantissa is above that of the largest code (127 = 1.984375 * 2^6, 448 = 1.75 * 2^8).
__device__ __forceinline__ uint32_t scale_byte(float amax, bool e4m3) {
    const uint32_t b = __float_as_uint(amax);
    if (b >= 0x7f800000u) return 255u;
    const int e = (int)((b + (e4m3 ? 0x7fffffu - 0x600000u : 0x7fffffu - 0x7e0000u)) >> 23) - (e4m3 ? 8 : 6);
    return (uint32_t)(e > 0 ? e : 0);
}
// 1 / scale; e is at most 249 here, so the exponent field stays normal.
__device__ __forceinline__ float inverse_scale(uint32_t e) { return __uint_as_float((254u - e) << 23); }
__device__ __forceinline__ float scale_value(uint32_t e) {
    return e == 0 ? __uint_as_float(0x00400000u) : e == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(e << 23);
}

// Largest magnitude (NaN if there is one) over the lanes that share a block; V values per lane.
template <int V>
__device__ __forceinline__ float block_amax(const float* v) {
    float m = fabsf(v[0]);
#pragma unroll
    for (int i = 1; i < V; ++i) m = jl_max(m, fabsf(v[i]));
#pragma unroll
    for (int o = kBlock / V / 2; o > 0; o /= 2) m = jl_max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}

// Adding 1.5 * 2^23 leaves the integer nearest to x (ties to even) in the low mantissa bits.
__device__ __forceinline__ uint32_t int8_code(float v, float inv) { return __float_as_uint(fmaf(v, inv, 12582912.f)); }
__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 e4m3_values(uint16_t w) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(w));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

template <int V>
__device__ __forceinline__ RawVec<uint8_t, V> encode(const float* v, uint32_t e, bool e4m3) {
    RawVec<uint8_t, V> r{};
    if (e == 255u) return r;
    const float inv = inverse_scale(e);
    if constexpr (V == 1) {
        r = (uint8_t)(e4m3 ? e4m3_pair(v[0] * inv, 0.f) : int8_code(v[0], inv));
    } else {
        uint32_t* w = reinterpret_cast<uint32_t*>(&r);
        if (e4m3) {
#pragma unroll
            for (int i = 0; i < V / 4; ++i)
                w[i] = e4m3_pair(v[4 * i] * inv, v[4 * i + 1] * inv) | e4m3_pair(v[4 * i + 2] * inv, v[4 * i + 3] * inv) << 16;
        } else {
#pragma unroll
            for (int i = 0; i < V / 4; ++i) {
                const uint32_t lo = __byte_perm(int8_code(v[4 * i], inv), int8_code(v[4 * i + 1], inv), 0x0040);
                const uint32_t hi = __byte_perm(int8_code(v[4 * i + 2], inv), int8_code(v[4 * i + 3], inv), 0x0040);
                w[i] = __byte_perm(lo, hi, 0x5410);
            }
        }
    }
    return r;
}

// Codes to binary32.  Int8: the byte with its sign bit flipped, as the low mantissa bits of 2^23.
template <int V>
__device__ __forceinline__ void decode(const RawVec<uint8_t, V>& r, uint32_t e, bool e4m3, float* v) {
    const float s = scale_value(e);
    if constexpr (V == 1) {
        v[0] = (e4m3 ? e4m3_values((uint16_t)r).x : (float)(int8_t)r) * s;
    } else {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            if (e4m3) {
                const float2 a = e4m3_values((uint16_t)(w[i] & 0xffffu)), b = e4m3_values((uint16_t)(w[i] >> 16));
                v[4 * i] = a.x * s; v[4 * i + 1] = a.y * s; v[4 * i + 2] = b.x * s; v[4 * i + 3] = b.y * s;
            } else {
                const uint32_t u = w[i] ^ 0x80808080u;
                v[4 * i]     = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440)) - 8388736.f) * s;
                v[4 * i + 1] = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441)) - 8388736.f) * s;
                v[4 * i + 2] = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7442)) - 8388736.f) * s;
                v[4 * i + 3] = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7443)) - 8388736.f) * s;
            }
        }
    }
}
// The same for pairs.
template <int V>
__device__ __forceinline__ float block_amax2(const F2* v, bool in) {
    const float2 a = f2_parts(v[0]);
    float m = amax3(a.x, a.y, 0.f);
#pragma unroll
    for (int i = 1; i < V / 2; ++i) { const float2 b = f2_parts(v[i]); m = amax3(m, b.x, b.y); }
    if (!in) m = 0.f;
#pragma unroll
    for (int o = kBlock / V / 2; o > 0; o /= 2) m = jl_max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}
template <int V>
__device__ __forceinline__ RawVec<uint8_t, V> encode2(const F2* v, uint32_t e, bool e4m3) {
    RawVec<uint8_t, V> r;
    const F2 inv = f2(inverse_scale(e));
    const uint32_t mask = e == 255u ? 0u : ~0u;           // no branch around the rest
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
    if (e4m3) {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const float2 a = f2_parts(f2_mul(v[2 * i], inv)), b = f2_parts(f2_mul(v[2 * i + 1], inv));
            w[i] = (e4m3_pair(a.x, a.y) | e4m3_pair(b.x, b.y) << 16) & mask;
        }
    } else {
        const F2 magic = f2(12582912.f);
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const float2 a = f2_parts(f2_fma(v[2 * i], inv, magic)), b = f2_parts(f2_fma(v[2 * i + 1], inv, magic));
            const uint32_t lo = __byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040);
            const uint32_t hi = __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040);
            w[i] = __byte_perm(lo, hi, 0x5410) & mask;
        }
    }
    return r;
}
// For e up to 200: the offset of the Int8 codes is folded into one multiply-add (2^23 2^73 overflows nothing).
template <int V>
__device__ __forceinline__ void decode2(const RawVec<uint8_t, V>& r, uint32_t e, bool e4m3, F2* v) {
    const float scale = scale_value(e);
    const F2 s = f2(scale);
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
    if (e4m3) {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const float2 a = e4m3_values((uint16_t)(w[i] & 0xffffu)), b = e4m3_values((uint16_t)(w[i] >> 16));
            v[2 * i] = f2_mul(f2(a.x, a.y), s);
            v[2 * i + 1] = f2_mul(f2(b.x, b.y), s);
        }
    } else {
        const F2 zero = f2(-8388736.f * scale);
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const uint32_t u = w[i] ^ 0x80808080u;
            v[2 * i] = f2_fma(f2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441))), s, zero);
            v[2 * i + 1] = f2_fma(f2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7442)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7443))), s, zero);
        }
    }
}
// A value near the largest of its type can have been rounded up past it: such blocks saturate.
// The code of largest magnitude (Int8 -128, which no encoder here writes, e4m3 448) times 2^(e-127) passes
// T's largest value only from this e on.
template <typename T>
__device__ __forceinline__ uint32_t saturating_from(bool e4m3) {
    return sizeof(T) == 2 && Elem<T>::kMax < 1e5f ? (e4m3 ? 135u : 136u) : (e4m3 ? 247u : 248u);
}
// Scales that are far from overflowing anything.
template <typename T>
__device__ __forceinline__ bool plain_scale(uint32_t e) { return e <= (sizeof(T) == 2 && Elem<T>::kMax < 1e5f ? 134u : 200u); }
template <typename T, int V>
__device__ __forceinline__ void decode_as(const RawVec<uint8_t, V>& r, uint32_t e, bool e4m3, float* v) {
    decode<V>(r, e, e4m3, v);
    if (e >= saturating_from<T>(e4m3) && e != 255u) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = v[i] > Elem<T>::kMax ? Elem<T>::kMax : v[i] < -Elem<T>::kMax ? -Elem<T>::kMax : v[i];     // NaN stays
    }
}

// ---- angles --------------------------------------------------------------------------------------
// Sine and cosine of a phase counted in 2^-64 turns.  Position times frequency is one wrapping
// 64-bit product: what a table's entry is off by (2^-65 turns, where it was rounded once) times the
// position is all that far positions lose, 4e-9 turns at 2^37.  The phase is taken to
// the nearest quarter turn and the rest, at most pi/4, goes through the Taylor series (terms left
// out: below 2e-9).
__device__ __forceinline__ void phase_sincos(uint64_t phase, float factor, float& sn, float& cs) {
    const uint32_t quarter = (uint32_t)((phase + (uint64_t(1) << 61)) >> 62);
    const int64_t rest = (int64_t)(phase - ((uint64_t)quarter << 62));                 // [-2^61, 2^61)
    const float a = (float)(int32_t)(rest >> 30) * 3.6572952e-10f;                     // 2 pi / 2^34
    const float z = a * a;
    float s = fmaf(z, 1.f / 362880.f, -1.f / 5040.f);
    s = fmaf(z, s, 1.f / 120.f);
    s = fmaf(z, s, -1.f / 6.f);
    s = fmaf(a * z, s, a) * factor;
    float c = fmaf(z, -1.f / 3628800.f, 1.f / 40320.f);
    c = fmaf(z, c, -1.f / 720.f);
    c = fmaf(z, c, 1.f / 24.f);
    c = fmaf(z, c, -0.5f);
    c = fmaf(z, c, 1.f) * factor;
    const bool swap = quarter & 1;
    sn = swap ? c : s;
    cs = swap ? s : c;
    if (quarter & 2) sn = -sn;
    if ((quarter + 1) & 2) cs = -cs;
}
__device__ __forceinline__ int64_t load_int(const void* p, bool wide, int64_t i) {
    return wide ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t)reinterpret_cast<const int32_t*>(p)[i];
}
#endif  // __CUDACC__

enum { kRotaryHalf = 0, kRotaryInterleaved = 1 };
inline bool is_index_type(int32_t dt) { return dt == B200_I32 || dt == B200_I64; }

}  // namespace b200
