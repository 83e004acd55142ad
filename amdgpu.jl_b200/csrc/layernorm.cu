// Layer norm along the leading dimensions and its gradient, with the normalised rows kept as they
// are, or in 8 bits (rowops.cuh) for the gradient.  It takes the place of a chain of mapreduce and
// broadcast calls over the same rows (src/kernels/mapreduce.jl:86-173, src/broadcast.jl:3-30).
//
//   forward   m = mean(x), r = 1/sqrt(mean((x-m)^2) + eps), h = (x-m) r, y = h gamma + beta
//   gradient  g = dy gamma, dx = r (g - mean(g) - h mean(g h)), dgamma = sum_rows dy h, dbeta = sum_rows dy
//
// Everything is held in binary32 and rounded once, on the store.
#include "rowops.cuh"

namespace b200 {

struct NormArgs {
    const void *x, *dy, *gamma, *beta;
    void *y;                            // forward: y; gradient: dx
    float *mean, *rstd;
    uint8_t *q, *s;                     // codes and scale bytes of the normalised rows
    float *partial;                     // gradient: [block][2][d] sums of dy*h and dy
    int64_t ldx, ldy, lddy, rows, d, blocks;
    // ring kernels: rows from one of a group's to its next, and that many rows of each array in elements
    int64_t step, x_step, y_step, dy_step, q_step, s_step;
    float eps;
    int32_t gamma_f32, e4m3, group;     // group: threads per row
    int32_t pitch, pitch_x, units2;     // rows of any alignment: bytes of a stage of the rings; two elements at a time
};

__device__ __forceinline__ float load_param(const void* p, bool f32, int32_t dtype, int64_t i) {
    if (f32) return reinterpret_cast<const float*>(p)[i];
    return dtype == B200_F16 ? __half2float(reinterpret_cast<const __half*>(p)[i])
                             : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}
template <typename T> constexpr int32_t dtype_of();
template <> constexpr int32_t dtype_of<float>() { return B200_F32; }
template <> constexpr int32_t dtype_of<__half>() { return B200_F16; }
template <> constexpr int32_t dtype_of<__nv_bfloat16>() { return B200_BF16; }

__device__ __forceinline__ float lane_sum(float v, int width) {
#pragma unroll
    for (int o = 16; o > 0; o /= 2) if (o < width) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// ---- rows through a ring in shared memory -----------------------------------------------------------
// Aligned rows of whole vectors.  `group` threads hold a row, E elements each; a block has as many groups
// as fit and every group walks over the rows with the grid's stride, STAGES - 1 rows ahead of its own work.
// A thread copies its own vectors (cp.async, 16 bytes) into its own places of the ring and reads only
// those, so the ring needs no barrier: a thread waits for its own copies.  Groups run on their own, with a
// hardware barrier each for their sums, so that some load while others compute and store.
//
// With the loads out of the way these kernels are held up by their instructions and by the latency of a
// row's sums (issue slots 38 to 48 % taken at 10 to 14 warps an SM), not by HBM: arithmetic goes in pairs
// (F2), a thread has as many columns as its registers hold, and nothing is predicated but the copies and
// stores (vectors beyond a row read as zeros).  One B200, 16384 x 4096 BFloat16: forward 48 us
// (5.5 TB/s), with the 8-bit rows written as well 63 us, gradient 69 us (5.8 TB/s), from the 8-bit rows
// 66 us; waiting for each row in turn the gradient takes 120 us.  A register spilled inside the loop costs
// more than a second pass over it (20 bytes: 69 -> 84 us).
//
// Rows that fill every thread of whole warps (d = group * E) lie warp by warp, so that a thread's steps
// through a row are known at compile time, and nothing is predicated: 8192 x 5120 BFloat16 forward with the
// 8-bit rows 41 us (44 without), gradient from them 50 us (56), 8192 x 6144 Float16 46 (55) and 55 (61) us,
// 8192 x 8192 gradient 79 (84) us; 16384 x 4096 forward with the 8-bit rows 63 (61) us.  The steps alone, for
// rows that leave threads empty: 16000 x 2624 forward with the 8-bit rows 45 us (47).

// How a row lies over its group: neighbouring vectors over all threads; over the threads of each warp, so
// that steps are known at compile time; the same with every thread filled, so that nothing is predicated.
enum { kOverGroup = 0, kOverWarps = 1, kFilled = 2 };
enum { kAsIs = 0 };                     // form of the rows kept for the gradient: as they are, kInt8, kE4M3

struct GroupBarrier {
    int id, threads;
    __device__ __forceinline__ void sync() const { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
};
// What a thread of a ring kernel knows about its place and its rows: row + i * step for i < mine.
struct RingPlace {
    int group, t, warps, warp, lane, width, mine, walk;
    int64_t row;
    GroupBarrier bar;
    __device__ __forceinline__ RingPlace(int G, int64_t rows, int64_t step) {
        const int per_block = blockDim.x / G;
        group = threadIdx.x / G;
        t = threadIdx.x % G;
        warps = G / 32; warp = t / 32; lane = t % 32;
        width = G < 32 ? G : 32;
        bar = GroupBarrier{group + 1, G};
        row = (int64_t)blockIdx.x * per_block + group;
        mine = row < rows ? (int)((rows - row + step - 1) / step) : 0;
        // exchanges take whole warps: groups that share one walk as often as its first, which has most rows
        walk = __shfl_sync(0xffffffffu, mine, 0);
    }
};
// Places for the warps' sums: zero beyond the group's warps, whole vectors for the reader.
constexpr int kShare = 16;
// Sum over a group.
__device__ __forceinline__ float group_sum(float v, const RingPlace& p, float* share) {
    v = lane_sum(v, p.width);
    if (p.warps <= 1) return v;
    if (p.lane == 0) share[p.warp] = v;
    p.bar.sync();
    const float4* q = reinterpret_cast<const float4*>(share);
    float4 a = q[0], b = q[1];
    v = ((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w));
    if (p.warps > 8) {
        a = q[2]; b = q[3];
        v += ((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w));
    }
    return v;
}
// Two sums at once: after the first exchange one half of the lanes carries each.
__device__ __forceinline__ float2 group_sum2(float a, float b, const RingPlace& p, float2* share) {
    if (p.width < 32) {
        a = lane_sum(a, p.width);
        return make_float2(a, lane_sum(b, p.width));
    }
    const bool upper = p.lane & 16;
    float v = (upper ? b : a) + __shfl_xor_sync(0xffffffffu, upper ? a : b, 16);
#pragma unroll
    for (int o = 8; o > 0; o /= 2) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (p.warps <= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, v, 16);
        return upper ? make_float2(other, v) : make_float2(v, other);
    }
    if ((p.lane & 15) == 0) reinterpret_cast<float*>(share + p.warp)[upper] = v;
    p.bar.sync();
    const ulonglong2* q = reinterpret_cast<const ulonglong2*>(share);
    const ulonglong2 u0 = q[0], u1 = q[1], u2 = q[2], u3 = q[3];
    F2 sum = f2_add(f2_add(f2_add(u0.x, u0.y), f2_add(u1.x, u1.y)), f2_add(f2_add(u2.x, u2.y), f2_add(u3.x, u3.y)));
    if (p.warps > 8) {
#pragma unroll
        for (int w = 4; w < 8; ++w) { const ulonglong2 u = q[w]; sum = f2_add(sum, f2_add(u.x, u.y)); }
    }
    return f2_parts(sum);
}
template <int BYTES>
__device__ __forceinline__ void ring_copy(void* dst, const void* src) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(src), "n"(BYTES) : "memory");
}
template <typename T, int V, int NV>
__device__ __forceinline__ void load_params2(const NormArgs& a, const void* p, int t, int step, int nvec, float missing, F2* out) {
    const bool aligned = (reinterpret_cast<uintptr_t>(p) & 15) == 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int vi = t + k * step;
#pragma unroll
        for (int i = 0; i < V / 2; ++i) out[k * V / 2 + i] = f2(missing);
        if (!p || vi >= nvec) continue;
        if (a.gamma_f32) {
#pragma unroll
            for (int i = 0; i < V / 4; ++i) {
                const float* f = reinterpret_cast<const float*>(p) + (int64_t)vi * V + 4 * i;
                float4 q;
                if (aligned) q = *reinterpret_cast<const float4*>(f);
                else q = make_float4(f[0], f[1], f[2], f[3]);
                out[k * V / 2 + 2 * i] = f2(q.x, q.y);
                out[k * V / 2 + 2 * i + 1] = f2(q.z, q.w);
            }
        } else {
            const T* f = reinterpret_cast<const T*>(p) + (int64_t)vi * V;
            if (aligned) {
                unpack2<T, V>(ld_raw_cached<T, V>(f), out + k * V / 2);
            } else {
#pragma unroll
                for (int i = 0; i < V / 2; ++i) out[k * V / 2 + i] = f2(Elem<T>::get(f[2 * i]), Elem<T>::get(f[2 * i + 1]));
            }
        }
    }
}

// Two passes over the row in registers: the mean first, then the squares about it.
template <typename T, int E, int STAGES, int THREADS, int KEEP, int FORM>
__global__ void __launch_bounds__(THREADS)
norm_forward_ring_kernel(NormArgs a) {
    constexpr int V = 16 / (int)sizeof(T), NV = E / V, SLOT = NV * THREADS;
    extern __shared__ uint4 ring[];                       // [stage][vector][thread]
    __shared__ __align__(16) float shares[THREADS / 64][4][kShare];
    for (int i = threadIdx.x; i < (int)(sizeof(shares) / 4); i += blockDim.x) (&shares[0][0][0])[i] = 0.f;
    __syncthreads();
    grid_dependency_wait();
    const RingPlace p(a.group, a.rows, a.step);
    const int S = FORM ? 32 : a.group, t = FORM ? p.warp * (32 * NV) + p.lane : p.t, nvec = (int)(a.d / V);
    bool in[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) in[k] = FORM == kFilled || t + k * S < nvec;
    const T* src = reinterpret_cast<const T*>(a.x) + p.row * a.ldx + (int64_t)t * V;      // next row to fetch
    T* dst = reinterpret_cast<T*>(a.y) + p.row * a.ldy + (int64_t)t * V;
    uint8_t* dst_q = a.q + p.row * a.d + t * V;
    uint8_t* dst_s = a.s + p.row * a.blocks + t / (kBlock / V);
    uint4* own = ring + threadIdx.x;
    int to_fetch = p.mine;
    auto fetch = [&](int slot) {
        if (to_fetch > 0) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (in[k]) ring_copy<16>(own + slot + k * THREADS, src + k * S * V);
        }
        --to_fetch;
        src += a.x_step;
        cp_async_commit();
    };
    // places that no copy fills: the vectors beyond the row read as zeros
#pragma unroll
    for (int s = 0; s < STAGES; ++s) {
#pragma unroll
        for (int k = 0; k < NV; ++k) if (!in[k]) own[s * SLOT + k * THREADS] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) fetch(s * SLOT);
    F2 gm[E / 2], bt[E / 2];
    load_params2<T, V, NV>(a, a.gamma, t, S, nvec, 1.f, gm);
    load_params2<T, V, NV>(a, a.beta, t, S, nvec, 0.f, bt);
    const float per_d = 1.f / (float)a.d;
    int slot = 0, free_slot = (STAGES - 1) * SLOT;
    float* share = &shares[p.warps > 1 ? p.group : 0][0][0];
    int64_t row = p.row;
    for (int it = 0; it < p.walk; ++it, row += a.step) {
        const bool live = FORM || it < p.mine;
        cp_async_wait<STAGES - 2>();
        F2 v[E / 2];
        F2 sum2 = f2(0.f);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            unpack2<T, V>(own[slot + k * THREADS], v + k * V / 2);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) sum2 = f2_add(sum2, v[k * V / 2 + i]);
        }
        fetch(free_slot);
        free_slot = slot;
        slot = slot == (STAGES - 1) * SLOT ? 0 : slot + SLOT;
        const float mean = group_sum(f2_total(sum2), p, share) * per_d;
        F2 m2 = f2(0.f);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const F2 minus = f2(in[k] ? -mean : 0.f);     // beyond the row: zeros stay zeros
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                F2& c = v[k * V / 2 + i];
                c = f2_add(c, minus);
                m2 = f2_fma(c, c, m2);
            }
        }
        const float var = group_sum(f2_total(m2), p, share + kShare) * per_d;
        share = (it & 1) ? share - 2 * kShare : share + 2 * kShare;
        const float rstd = 1.f / sqrtf(var + a.eps);
        if (live && p.t == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
        const F2 r2 = f2(rstd);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            F2* h = v + k * V / 2;
            F2 o[V / 2];
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                h[i] = f2_mul(h[i], r2);
                o[i] = f2_fma(h[i], gm[k * V / 2 + i], bt[k * V / 2 + i]);
            }
            if (live && in[k]) st_raw<T, V>(dst + k * S * V, pack2<T, V>(o));
            if constexpr (KEEP != kAsIs) {
                const uint32_t e = scale_byte(block_amax2<V>(h, live && in[k]), KEEP == kE4M3);
                if (live && in[k]) {
                    st_raw<uint8_t, V>(dst_q + k * S * V, encode2<V>(h, e, KEEP == kE4M3));
                    if (t % (kBlock / V) == 0) dst_s[k * (S / (kBlock / V))] = (uint8_t)e;
                }
            }
        }
        dst += a.y_step;
        if constexpr (KEEP != kAsIs) { dst_q += a.q_step; dst_s += a.s_step; }
    }
}

// dx needs the row again after its sums: g gamma and h stay in registers (HOLD), or the row is read out
// of the ring a second time and the registers are for the column sums of more columns.
template <typename T, int E, int STAGES, int THREADS, int KEPT, bool HOLD, int FORM>
__global__ void __launch_bounds__(THREADS)
norm_backward_ring_kernel(NormArgs a) {
    constexpr int V = 16 / (int)sizeof(T), NV = E / V, SLOT = NV * THREADS;
    extern __shared__ uint4 ring[];                       // dy: [stage][vector][thread], then x or codes alike
    __shared__ __align__(16) float2 shares[THREADS / 64][2][kShare];
    using Code = RawVec<uint8_t, V>;
    for (int i = threadIdx.x; i < (int)(sizeof(shares) / 8); i += blockDim.x) (&shares[0][0][0])[i] = make_float2(0.f, 0.f);
    __syncthreads();
    grid_dependency_wait();
    const RingPlace p(a.group, a.rows, a.step);
    const int S = FORM ? 32 : a.group, t = FORM ? p.warp * (32 * NV) + p.lane : p.t, nvec = (int)(a.d / V), per_block = blockDim.x / a.group;
    bool in[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) in[k] = FORM == kFilled || t + k * S < nvec;
    const T* src = reinterpret_cast<const T*>(a.dy) + p.row * a.lddy + (int64_t)t * V;    // next row to fetch
    const T* src_x = reinterpret_cast<const T*>(a.x) + p.row * a.ldx + (int64_t)t * V;
    const uint8_t* src_q = a.q + p.row * a.d + (int64_t)t * V;
    uint4* own = ring + threadIdx.x;
    uint4* own_x = ring + STAGES * SLOT + threadIdx.x;
    Code* own_q = reinterpret_cast<Code*>(ring + STAGES * SLOT) + threadIdx.x;
    auto fetch = [&](int slot, bool more) {
        if (more) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (in[k]) {
                    ring_copy<16>(own + slot + k * THREADS, src + k * S * V);
                    if constexpr (KEPT != kAsIs) ring_copy<V>(own_q + slot + k * THREADS, src_q + k * S * V);
                    else ring_copy<16>(own_x + slot + k * THREADS, src_x + k * S * V);
                }
            }
        }
        src += a.dy_step;
        if constexpr (KEPT != kAsIs) src_q += a.q_step; else src_x += a.x_step;
        cp_async_commit();
    };
    // places that no copy fills: the vectors beyond the row read as zeros
#pragma unroll
    for (int s = 0; s < STAGES; ++s) {
#pragma unroll
        for (int k = 0; k < NV; ++k) if (!in[k]) {
            own[s * SLOT + k * THREADS] = make_uint4(0, 0, 0, 0);
            if constexpr (KEPT != kAsIs) own_q[s * SLOT + k * THREADS] = Code{};
            else own_x[s * SLOT + k * THREADS] = make_uint4(0, 0, 0, 0);
        }
    }
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) fetch(s * SLOT, s < p.mine);
    // gamma lies in shared memory, [vector][quarter][thread], where threads' vectors lie side by side: the
    // registers are taken
    float4* gammas = reinterpret_cast<float4*>(reinterpret_cast<char*>(ring) + (size_t)STAGES * SLOT * (16 + (KEPT ? V : 16))) +
                     (FORM ? p.warp * (32 * E / 4) + p.lane : t);
    if (p.group == 0) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
#pragma unroll
            for (int j = 0; j < V / 4; ++j) {
                const int64_t c = (int64_t)(t + k * S) * V + 4 * j;
                float4 g = make_float4(1.f, 1.f, 1.f, 1.f);
                if (a.gamma && in[k])
                    g = make_float4(load_param(a.gamma, a.gamma_f32, dtype_of<T>(), c), load_param(a.gamma, a.gamma_f32, dtype_of<T>(), c + 1),
                                    load_param(a.gamma, a.gamma_f32, dtype_of<T>(), c + 2), load_param(a.gamma, a.gamma_f32, dtype_of<T>(), c + 3));
                gammas[(k * (V / 4) + j) * S] = g;
            }
        }
    }
    __syncthreads();
    F2 dg[E / 2], db[E / 2];
#pragma unroll
    for (int i = 0; i < E / 2; ++i) dg[i] = db[i] = f2(0.f);
    const float per_d = 1.f / (float)a.d;
    // what a row needs beside the ring is loaded one row ahead
    float rstd_next = 0.f, mean_next = 0.f;
    uint32_t scale[NV] = {};
    int row = (int)p.row;                                 // fewer than 2^31 rows: a pointer for each of these is two registers
    auto ahead = [&](int r, bool live) {
        if (live) {
            rstd_next = a.rstd[r];
            if constexpr (KEPT == kAsIs) mean_next = a.mean[r];
            else {
                const uint8_t* at = a.s + r * a.blocks + t / (kBlock / V);
#pragma unroll
                for (int k = 0; k < NV; ++k) if (in[k]) scale[k] = at[k * S / (kBlock / V)];
            }
        }
    };
    ahead(row, p.mine > 0);
    int slot = 0, free_slot = (STAGES - 1) * SLOT;
    float2* share = &shares[p.warps > 1 ? p.group : 0][0][0];
    for (int it = 0; it < p.walk; ++it, row += (int)a.step) {
        const bool live = it < p.mine;                    // whole warps: always; without the branch the loads below move about and spill
        const float rstd = rstd_next;
        const F2 r2 = f2(rstd), minus = f2(-mean_next);
        cp_async_wait<STAGES - 2>();
        auto load_dy = [&](int k, F2* g) { unpack2<T, V>(own[slot + k * THREADS], g); };
        auto load_h = [&](int k, F2* h) {
            if constexpr (KEPT != kAsIs) {
                decode2<V>(own_q[slot + k * THREADS], scale[k], KEPT == kE4M3, h);
            } else {
                unpack2<T, V>(own_x[slot + k * THREADS], h);
#pragma unroll
                for (int i = 0; i < V / 2; ++i) h[i] = f2_mul(f2_add(h[i], minus), r2);
            }
        };
        F2 s1 = f2(0.f), s2 = f2(0.f);
        F2 gs[HOLD ? E / 2 : V / 2], hs[HOLD ? E / 2 : V / 2];
        if (live) {                                       // false for groups that share a warp with a longer one
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                F2* g = gs + (HOLD ? k * V / 2 : 0);
                F2* h = hs + (HOLD ? k * V / 2 : 0);
                load_dy(k, g);
                load_h(k, h);
#pragma unroll
                for (int q = 0; q < V / 4; ++q) {
                    const ulonglong2 gm = *reinterpret_cast<const ulonglong2*>(gammas + (k * (V / 4) + q) * S);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int i = 2 * q + e, j = k * V / 2 + i;
                        dg[j] = f2_fma(g[i], h[i], dg[j]);
                        db[j] = f2_add(db[j], g[i]);
                        g[i] = f2_mul(g[i], e ? gm.y : gm.x);
                        s1 = f2_add(s1, g[i]);
                        s2 = f2_fma(g[i], h[i], s2);
                    }
                }
            }
        }
        if constexpr (HOLD) {
            ahead(row + (int)a.step, it + 1 < p.mine);
            fetch(free_slot, it + STAGES - 1 < p.mine);
        }
        const float2 s = group_sum2(f2_total(s1), f2_total(s2), p, share);
        share = (it & 1) ? share - kShare : share + kShare;
        if (a.y) {
            T* dst = reinterpret_cast<T*>(a.y) + row * a.ldy + t * V;
            const F2 c1 = f2(-s.x * per_d * rstd), c2 = f2(-s.y * per_d * rstd);
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                F2* g = gs + (HOLD ? k * V / 2 : 0);
                F2* h = hs + (HOLD ? k * V / 2 : 0);
                if constexpr (!HOLD) load_h(k, h);
                if constexpr (!HOLD) {
                    load_dy(k, g);
#pragma unroll
                    for (int q = 0; q < V / 4; ++q) {
                        const ulonglong2 gm = *reinterpret_cast<const ulonglong2*>(gammas + (k * (V / 4) + q) * S);
                        g[2 * q] = f2_mul(g[2 * q], gm.x);
                        g[2 * q + 1] = f2_mul(g[2 * q + 1], gm.y);
                    }
                }
                F2 o[V / 2];
#pragma unroll
                for (int i = 0; i < V / 2; ++i) o[i] = f2_fma(h[i], c2, f2_fma(g[i], r2, c1));
                if (live && in[k]) st_raw<T, V>(dst + k * S * V, pack2<T, V>(o));
            }
        }
        if constexpr (!HOLD) {
            ahead(row + (int)a.step, it + 1 < p.mine);
            fetch(free_slot, it + STAGES - 1 < p.mine);
        }
        free_slot = slot;
        slot = slot == (STAGES - 1) * SLOT ? 0 : slot + SLOT;
    }
    grid_dependency_release();
    if (!a.partial) return;
    // Column sums: the groups' side by side in the ring's place, [group][2][d], joined in the groups'
    // order, so that the order of the sum is fixed.
    float* column = reinterpret_cast<float*>(ring);
    const int d2 = 2 * (int)a.d;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        float* c = column + (int64_t)p.group * d2 + (t + k * S) * V;
        if (in[k]) {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {             // in pairs: quads would tie the loop's registers
                *reinterpret_cast<F2*>(c + 2 * i) = dg[k * V / 2 + i];
                *reinterpret_cast<F2*>(c + a.d + 2 * i) = db[k * V / 2 + i];
            }
        }
    }
    __syncthreads();
    ulonglong2* out = reinterpret_cast<ulonglong2*>(a.partial) + (int64_t)blockIdx.x * (d2 / 4);
    const ulonglong2* quads = reinterpret_cast<const ulonglong2*>(column);
#pragma unroll 2
    for (int q = threadIdx.x; q < d2 / 4; q += blockDim.x) {
        ulonglong2 sum = quads[q];
#pragma unroll 4
        for (int g = 1; g < per_block; ++g) {
            const ulonglong2 v = quads[g * (d2 / 4) + q];
            sum.x = f2_add(sum.x, v.x);
            sum.y = f2_add(sum.y, v.y);
        }
        out[q] = sum;
    }
}

// ---- rows of any alignment ------------------------------------------------------------------------
// The same for rows that start anywhere (odd widths, views): the aligned 16-byte pieces that cover a row go
// through the ring, and a thread picks its columns t, t + group, ... out of them one by one, so its gamma and
// its column sums stay its own whatever a row's offset.  The pieces are shared by a group: one more barrier
// per row.  Pieces that reach past the first or the last byte of the array are copied element by element.
// Instructions are what it takes its time for: a shared-memory load, a conversion and a store per element, and
// a row's fixed work, 27 a thread and element forward and 32 for the gradient (16384 x 4095 BFloat16; issue
// slots 60 and 54 % taken at 34 and 25 % of the warps, HBM at 30 and 39 %).  So a thread has fewer columns where
// rows are narrow, a block's scale is worked out by one lane and handed to the others, and whole warps skip
// the predicates.  Float32 rows have half the elements per byte and lose little: 16384 x 4095 forward 92 us,
// gradient 137 us (floors 82 and 123).  One B200, 16384 x 4095 BFloat16 (4096: in brackets): forward 90 us (48), with the
// 8-bit rows 151 us (63), gradient 118 us (69), from the 8-bit rows 124 us (66); 200000 x 101 Float16 68, 97,
// 78 and 82 us (16 columns per thread: 106, 204, 136 and 145 us).  Rows of up to 512 * 16 = 8192 columns; with
// a block per row that reads it three times out of L2, as longer ones still go, 16384 x 4095 takes 266 us forward
// and as long for the gradient.
constexpr int kAnyElems = 16;
constexpr int kAnyStages = 3;
constexpr int kAnyThreads = 512;

template <typename T>
struct PieceRing {
    const char *lo, *hi;                       // the array's first byte and the one behind its last
    char* buf;                                 // this group's first stage
    int pitch, bytes;                          // of a stage; of a row
    int64_t ld;
    __device__ __forceinline__ PieceRing(const void* p, int64_t row_elems, int64_t ld_elems, int64_t rows, char* smem, int pitch_)
        : lo(reinterpret_cast<const char*>(p)), hi(lo + ((rows - 1) * ld_elems + row_elems) * (int64_t)sizeof(T)), buf(smem), pitch(pitch_),
          bytes((int)(row_elems * sizeof(T))), ld(ld_elems * (int64_t)sizeof(T)) {}
    __device__ __forceinline__ int offset(int64_t row) const { return ((uint32_t)reinterpret_cast<uintptr_t>(lo) + (uint32_t)row * (uint32_t)ld) & 15; }
    __device__ __forceinline__ void fetch(int64_t row, int stage, int t, int G) const {
        const char* first = lo + row * ld;
        const char* from = first - offset(row);
        char* to = buf + stage * pitch;
        const int n = (offset(row) + bytes + 15) / 16;
        if (from >= lo && from + 16 * n <= hi) {              // all but the first and the last rows of an array
            for (int c = t; c < n; c += G) ring_copy<16>(to + 16 * c, from + 16 * c);
            return;
        }
        for (int c = t; c < n; c += G) {
            const char* src = from + 16 * c;
            if (src >= lo && src + 16 <= hi) {
                ring_copy<16>(to + 16 * c, src);
            } else {
                for (int j = 0; j < 16; j += (int)sizeof(T))
                    if (src + j >= first && src + j < first + bytes) *reinterpret_cast<T*>(to + 16 * c + j) = *reinterpret_cast<const T*>(src + j);
            }
        }
    }
    __device__ __forceinline__ const T* row(int64_t r, int stage) const { return reinterpret_cast<const T*>(buf + stage * pitch + offset(r)); }
};
inline int piece_pitch(int64_t row_bytes) { return (int)((row_bytes + 15) / 16 * 16 + 16); }

__device__ __forceinline__ void group_sync(const RingPlace& p) {
    if (p.warps > 1) p.bar.sync();
    else __syncwarp();
}

// A thread's columns: units of W neighbours, its warp's first unit + lane + 32 k for k < count (steps known
// at compile time: no registers for addresses); W is 2 where every row of 16-bit elements starts on 4 bytes.
// Two elements to a pair: those of a unit, or those of units 2j, 2j+1.
template <int W, int E>
struct AnyColumns {
    static constexpr int NU = E / W;
    int unit, count;
    bool full;                 // every lane of the warp has all its columns
    __device__ __forceinline__ AnyColumns(int t, int d) : unit(t / 32 * 32 * NU + t % 32) {
        const int units = d / W;
        count = unit < units ? min(NU, (units - unit + 31) / 32) : 0;
        full = __all_sync(0xffffffffu, count == NU);
    }
    __device__ __forceinline__ int column(int k) const { return (unit + 32 * k) * W; }
    // A warp's columns are kWarpBlocks blocks of 32.  Each block's scale is one lane's work: lane k for block k,
    // or, two columns to a unit, the 16 / NU lanes from k 16 / NU on of either half for the half's block of unit k.
    static constexpr int kWarpBlocks = E, kLanes = W == 1 ? 1 : 16 / NU;
    static __device__ __forceinline__ int block_of_lane() {
        const int lane = threadIdx.x % 32;
        return W == 1 ? lane % kWarpBlocks : 2 * (lane % 16 / kLanes) + lane / 16;
    }
    static __device__ __forceinline__ int lane_of_unit(int k) { return W == 1 ? k : (int)(threadIdx.x & 16) | kLanes * k; }
    // Largest magnitude, as bits, of this lane's block.
    __device__ __forceinline__ uint32_t block_most(const F2* v) const {
        const int lane = threadIdx.x % 32;
        uint32_t m[NU];
#pragma unroll
        for (int k = 0; k < NU; ++k) {
            float f[2];
            get(v, k, f);
            m[k] = __float_as_uint(f[0]) & 0x7fffffffu;
            if constexpr (W == 2) m[k] = max(m[k], __float_as_uint(f[1]) & 0x7fffffffu);
        }
        if constexpr (W == 1) {
            uint32_t most = 0;
#pragma unroll
            for (int k = 0; k < NU; ++k) {
                const uint32_t r = __reduce_max_sync(0xffffffffu, m[k]);
                if (lane % kWarpBlocks == k) most = r;
            }
            return most;
        } else {
            // every exchange halves the units a lane carries, until one is left
#pragma unroll
            for (int o = 8, n = NU / 2; o > 0; o /= 2, n /= 2) {
                if (n == 0) m[0] = max(m[0], __shfl_xor_sync(0xffffffffu, m[0], o));
#pragma unroll
                for (int k = 0; k < n; ++k) {
                    const bool upper = lane & o;
                    const uint32_t keep = upper ? m[k + n] : m[k], give = upper ? m[k] : m[k + n];
                    m[k] = max(keep, __shfl_xor_sync(0xffffffffu, give, o));
                }
            }
            return m[0];
        }
    }
    // The row's codes and scale bytes; PLAIN: all columns are there and all blocks are finite.
    template <bool PLAIN, bool E4M3>
    __device__ __forceinline__ void store_codes(uint8_t* q, const F2* v, float inv) const {
#pragma unroll
        for (int k = 0; k < NU; ++k) {
            const float s = __shfl_sync(0xffffffffu, inv, lane_of_unit(k));
            float f[2] = {0.f, 0.f};
            get(v, k, f);
            uint32_t c;
            if constexpr (E4M3) c = e4m3_pair(f[0] * s, f[1] * s);
            else if constexpr (W == 1) c = int8_code(f[0], s);
            else c = __byte_perm(int8_code(f[0], s), int8_code(f[1], s), 0x0040);
            if (!PLAIN && s == 0.f) c = 0;
            if (PLAIN || k < count) {
                if constexpr (W == 1) q[unit + 32 * k] = (uint8_t)c;
                else *reinterpret_cast<uint16_t*>(q + 2 * unit + 64 * k) = (uint16_t)c;
            }
        }
    }
    __device__ __forceinline__ void keep(uint8_t* q, uint8_t* sc, int warp, int blocks, bool e4m3, const F2* v) const {
        const uint32_t e = scale_byte(__uint_as_float(block_most(v)), e4m3);
        const int block = warp * kWarpBlocks + block_of_lane();
        if ((W == 1 ? threadIdx.x % 32 < E : threadIdx.x % kLanes == 0) && block < blocks) sc[block] = (uint8_t)e;
        const float inv = e == 255u ? 0.f : inverse_scale(e);
        if (__all_sync(0xffffffffu, full && e != 255u)) {
            if (e4m3) store_codes<true, true>(q, v, inv);
            else store_codes<true, false>(q, v, inv);
        } else {
            if (e4m3) store_codes<false, true>(q, v, inv);
            else store_codes<false, false>(q, v, inv);
        }
    }
    // The row out of its codes in shared memory, zeros beyond it; scale: of this lane's block.
    template <bool E4M3>
    __device__ __forceinline__ void restore(const uint8_t* x, float scale, F2* v) const {
#pragma unroll
        for (int k = 0; k < NU; k += 2 / W) {
            uint32_t c[2] = {0, 0};
            float s[2];
            s[0] = s[1] = __shfl_sync(0xffffffffu, scale, lane_of_unit(k));
            if constexpr (W == 1) {
                s[1] = __shfl_sync(0xffffffffu, scale, lane_of_unit(k + 1));
                if (full || k < count) c[0] = x[unit + 32 * k];
                if (full || k + 1 < count) c[1] = x[unit + 32 * k + 32];
            } else {
                uint32_t w = 0;
                if (full || k < count) w = *reinterpret_cast<const uint16_t*>(x + 2 * unit + 64 * k);
                c[0] = w & 0xff;
                c[1] = w >> 8;
            }
            if constexpr (E4M3) {
                const float2 f = e4m3_values((uint16_t)(c[0] | c[1] << 8));
                v[k * W / 2] = f2_mul(f2(f.x, f.y), f2(s[0], s[1]));
            } else {                                          // as in decode: the low mantissa bits of 2^23
                const F2 u = f2(__uint_as_float(c[0] ^ 0x4b000080u), __uint_as_float(c[1] ^ 0x4b000080u));
                v[k * W / 2] = f2_mul(f2_add(u, f2(-8388736.f)), f2(s[0], s[1]));
            }
        }
    }
    // pairs of a row in shared memory, zeros beyond the row
    template <typename T>
    __device__ __forceinline__ void load(const T* x, F2* v) const { full ? load_as<true>(x, v) : load_as<false>(x, v); }
    template <bool FULL, typename T>
    __device__ __forceinline__ void load_as(const T* x, F2* v) const {
#pragma unroll
        for (int k = 0; k < NU; ++k) {
            RawVec<T, W> r{};
            if (FULL || k < count) r = *reinterpret_cast<const RawVec<T, W>*>(x + unit * W + 32 * W * k);
            float f[2];
            unpack<T, W>(r, f);
            put(v, k, f);
        }
    }
    __device__ __forceinline__ void put(F2* v, int k, const float* f) const {
        if constexpr (W == 2) v[k] = f2(f[0], f[1]);
        else v[k / 2] = k & 1 ? f2(f2_parts(v[k / 2]).x, f[0]) : f2(f[0], 0.f);
    }
    __device__ __forceinline__ void get(const F2* v, int k, float* f) const {
        const float2 x = f2_parts(v[k * W / 2]);
        if constexpr (W == 2) { f[0] = x.x; f[1] = x.y; }
        else f[0] = k & 1 ? x.y : x.x;
    }
    template <typename T>
    __device__ __forceinline__ void store(T* y, const F2* v) const { full ? store_as<true>(y, v) : store_as<false>(y, v); }
    template <bool FULL, typename T>
    __device__ __forceinline__ void store_as(T* y, const F2* v) const {
#pragma unroll
        for (int k = 0; k < NU; ++k) {
            float f[2];
            get(v, k, f);
            if (FULL || k < count) *reinterpret_cast<RawVec<T, W>*>(y + unit * W + 32 * W * k) = pack<T, W>(f);
        }
    }
    // v - mean in the columns of the row; beyond it zeros stay zeros
    __device__ __forceinline__ void center(F2* v, float mean) const {
        const F2 minus = f2(-mean);
        if (full) {
#pragma unroll
            for (int j = 0; j < E / 2; ++j) v[j] = f2_add(v[j], minus);
        } else {
#pragma unroll
            for (int j = 0; j < E / 2; ++j)
                v[j] = f2_add(v[j], W == 2 ? f2(j < count ? -mean : 0.f) : f2(2 * j < count ? -mean : 0.f, 2 * j + 1 < count ? -mean : 0.f));
        }
    }
    template <typename T>
    __device__ __forceinline__ void params(const NormArgs& a, const void* p, float missing, F2* v) const {
#pragma unroll
        for (int k = 0; k < NU; ++k) {
            float f[2] = {missing, missing};
            if (p && k < count) {
#pragma unroll
                for (int i = 0; i < W; ++i) f[i] = load_param(p, a.gamma_f32, dtype_of<T>(), column(k) + i);
            }
            put(v, k, f);
        }
    }
};

template <typename T, int W, int E, int THREADS, bool KEEP>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 3 : 1)
norm_forward_any_kernel(NormArgs a) {
    extern __shared__ char pieces[];
    __shared__ __align__(16) float shares[THREADS / 64][4][kShare];
    for (int i = threadIdx.x; i < (int)(sizeof(shares) / 4); i += blockDim.x) (&shares[0][0][0])[i] = 0.f;
    __syncthreads();
    grid_dependency_wait();
    const RingPlace p(a.group, a.rows, a.step);
    const AnyColumns<W, E> mine(p.t, (int)a.d);
    const PieceRing<T> ring(a.x, a.d, a.ldx, a.rows, pieces + p.group * kAnyStages * a.pitch, a.pitch);
#pragma unroll
    for (int s = 0; s < kAnyStages - 1; ++s) {
        if (s < p.mine) ring.fetch(p.row + s * a.step, s, p.t, a.group);
        cp_async_commit();
    }
    F2 gm[E / 2], bt[E / 2];
    mine.template params<T>(a, a.gamma, 1.f, gm);
    mine.template params<T>(a, a.beta, 0.f, bt);
    const float per_d = 1.f / (float)a.d;
    float* share = &shares[p.warps > 1 ? p.group : 0][0][0];
    int stage = 0;
    int64_t row = p.row;
    for (int it = 0; it < p.mine; ++it, row += a.step) {
        cp_async_wait<kAnyStages - 2>();
        group_sync(p);
        F2 v[E / 2];
        mine.load(ring.row(row, stage), v);
        if (it + kAnyStages - 1 < p.mine) ring.fetch(row + (kAnyStages - 1) * a.step, stage == 0 ? kAnyStages - 1 : stage - 1, p.t, a.group);
        cp_async_commit();
        stage = stage + 1 == kAnyStages ? 0 : stage + 1;
        F2 sum = f2(0.f), m2 = f2(0.f);
#pragma unroll
        for (int j = 0; j < E / 2; ++j) sum = f2_add(sum, v[j]);
        const float mean = group_sum(f2_total(sum), p, share) * per_d;
        mine.center(v, mean);
#pragma unroll
        for (int j = 0; j < E / 2; ++j) m2 = f2_fma(v[j], v[j], m2);
        const float rstd = 1.f / sqrtf(fmaf(group_sum(f2_total(m2), p, share + kShare), per_d, a.eps));
        share = (it & 1) ? share - 2 * kShare : share + 2 * kShare;
        if (p.t == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
        const F2 r2 = f2(rstd);
        F2 o[E / 2];
#pragma unroll
        for (int j = 0; j < E / 2; ++j) {
            v[j] = f2_mul(v[j], r2);
            o[j] = f2_fma(v[j], gm[j], bt[j]);
        }
        mine.store(reinterpret_cast<T*>(a.y) + row * a.ldy, o);
        if constexpr (KEEP) {
            mine.keep(a.q + row * a.d, a.s + row * a.blocks, p.warp, (int)a.blocks, a.e4m3, v);
        }
    }
}

template <typename T, int W, int E, bool KEPT>
__global__ void __launch_bounds__(kAnyThreads)
norm_backward_any_kernel(NormArgs a) {
    extern __shared__ char pieces[];                      // [group][stage]: dy, then of all groups x or codes
    __shared__ __align__(16) float2 shares[kAnyThreads / 64][2][kShare];
    for (int i = threadIdx.x; i < (int)(sizeof(shares) / 8); i += blockDim.x) (&shares[0][0][0])[i] = make_float2(0.f, 0.f);
    __syncthreads();
    grid_dependency_wait();
    const RingPlace p(a.group, a.rows, a.step);
    const int G = a.group, d = (int)a.d, per_block = blockDim.x / G;
    const AnyColumns<W, E> mine(p.t, d);
    using S = typename std::conditional<KEPT, uint8_t, T>::type;
    char* second = pieces + per_block * kAnyStages * a.pitch;
    const PieceRing<T> ring(a.dy, a.d, a.lddy, a.rows, pieces + p.group * kAnyStages * a.pitch, a.pitch);
    const PieceRing<S> ring_x(KEPT ? (const void*)a.q : a.x, a.d, KEPT ? a.d : a.ldx, a.rows, second + p.group * kAnyStages * a.pitch_x, a.pitch_x);
#pragma unroll
    for (int s = 0; s < kAnyStages - 1; ++s) {
        if (s < p.mine) { ring.fetch(p.row + s * a.step, s, p.t, G); ring_x.fetch(p.row + s * a.step, s, p.t, G); }
        cp_async_commit();
    }
    F2 gm[E / 2], dg[E / 2], db[E / 2];
    mine.template params<T>(a, a.gamma, 1.f, gm);
#pragma unroll
    for (int j = 0; j < E / 2; ++j) dg[j] = db[j] = f2(0.f);
    const float per_d = 1.f / (float)a.d;
    float2* share = &shares[p.warps > 1 ? p.group : 0][0][0];
    int stage = 0, row = (int)p.row;
    // what a row needs beside the rings is loaded one row ahead
    const int block = p.warp * AnyColumns<W, E>::kWarpBlocks + AnyColumns<W, E>::block_of_lane();
    float rstd_next = 0.f, mean_next = 0.f;
    uint32_t scale_next = 0;
    auto ahead = [&](int r, bool live) {
        if (!live) return;
        rstd_next = a.rstd[r];
        if constexpr (!KEPT) mean_next = a.mean[r];
        else if (block < (int)a.blocks) scale_next = a.s[r * a.blocks + block];
    };
    ahead(row, p.mine > 0);
    for (int it = 0; it < p.mine; ++it, row += (int)a.step) {
        const float rstd = rstd_next, mean = mean_next;
        const uint32_t scale = scale_next;
        ahead(row + (int)a.step, it + 1 < p.mine);
        cp_async_wait<kAnyStages - 2>();
        group_sync(p);
        F2 g[E / 2], h[E / 2];
        mine.load(ring.row(row, stage), g);
        const S* x = ring_x.row(row, stage);
        if constexpr (KEPT) {
            if (a.e4m3) mine.template restore<true>(x, scale_value(scale), h);
            else mine.template restore<false>(x, scale_value(scale), h);
        } else {
            mine.load(x, h);
            const F2 r2 = f2(rstd);
            mine.center(h, mean);
#pragma unroll
            for (int j = 0; j < E / 2; ++j) h[j] = f2_mul(h[j], r2);
        }
        F2 s1 = f2(0.f), s2 = f2(0.f);
#pragma unroll
        for (int j = 0; j < E / 2; ++j) {
            dg[j] = f2_fma(g[j], h[j], dg[j]);
            db[j] = f2_add(db[j], g[j]);
            g[j] = f2_mul(g[j], gm[j]);
            s1 = f2_add(s1, g[j]);
            s2 = f2_fma(g[j], h[j], s2);
        }
        if (it + kAnyStages - 1 < p.mine) {
            const int next = row + (kAnyStages - 1) * (int)a.step, to = stage == 0 ? kAnyStages - 1 : stage - 1;
            ring.fetch(next, to, p.t, G);
            ring_x.fetch(next, to, p.t, G);
        }
        cp_async_commit();
        stage = stage + 1 == kAnyStages ? 0 : stage + 1;
        const float2 s = group_sum2(f2_total(s1), f2_total(s2), p, share);
        share = (it & 1) ? share - kShare : share + kShare;
        if (a.y) {
            const F2 c1 = f2(-s.x * per_d * rstd), c2 = f2(-s.y * per_d * rstd), r2 = f2(rstd);
#pragma unroll
            for (int j = 0; j < E / 2; ++j) g[j] = f2_fma(h[j], c2, f2_fma(g[j], r2, c1));
            mine.store(reinterpret_cast<T*>(a.y) + row * a.ldy, g);
        }
    }
    grid_dependency_release();
    if (!a.partial) return;
    // column sums as in the kernel above: groups side by side, joined in their order
    float* column = reinterpret_cast<float*>(pieces) + p.group * 2 * d;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < mine.NU; ++k) {
        float f[2];
        if (k < mine.count) {
            mine.get(dg, k, f);
#pragma unroll
            for (int i = 0; i < W; ++i) column[mine.column(k) + i] = f[i];
            mine.get(db, k, f);
#pragma unroll
            for (int i = 0; i < W; ++i) column[d + mine.column(k) + i] = f[i];
        }
    }
    __syncthreads();
    column = reinterpret_cast<float*>(pieces);
    float* out = a.partial + (int64_t)blockIdx.x * 2 * d;
    for (int c = threadIdx.x; c < 2 * d; c += blockDim.x) {
        float sum = column[c];
#pragma unroll 4
        for (int g = 1; g < per_block; ++g) sum += column[g * 2 * d + c];
        out[c] = sum;
    }
}

// Sums the partials (a few MB, out of L2): 4 W columns per block (W lanes of four), 1024 / W strands of partials, joined in a
// fixed order.  VEC: d is a multiple of 4, so four columns are one access.
template <bool VEC>
__global__ void __launch_bounds__(1024)
norm_fold_kernel(const float* partial, int64_t npartials, int64_t d, void* dgamma, void* dbeta, int32_t dtype) {
    constexpr int W = 16, STRANDS = 1024 / W;
    __shared__ float part[STRANDS][4 * W + 4];
    grid_dependency_wait();
    const int lane = threadIdx.x % W, strand = threadIdx.x / W;
    const int64_t c = ((int64_t)blockIdx.x * W + lane) * 4;  // over [dgamma | dbeta]
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    // a partial per SM: a strand's three loads are on their way together
    for (int64_t b = strand; b < npartials; b += STRANDS * 3) {
        float4 v[3];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (b + STRANDS * k >= npartials) continue;
            const float* at = partial + (b + STRANDS * k) * 2 * d + c;
            if (VEC) {
                if (c < 2 * d) v[k] = *reinterpret_cast<const float4*>(at);
            } else {
                if (c < 2 * d) v[k].x = at[0];
                if (c + 1 < 2 * d) v[k].y = at[1];
                if (c + 2 < 2 * d) v[k].z = at[2];
                if (c + 3 < 2 * d) v[k].w = at[3];
            }
        }
        sum[0] += v[0].x + v[1].x + v[2].x;
        sum[1] += v[0].y + v[1].y + v[2].y;
        sum[2] += v[0].z + v[1].z + v[2].z;
        sum[3] += v[0].w + v[1].w + v[2].w;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) part[strand][4 * lane + i] = sum[i];
    __syncthreads();
    // sixteen threads per column take four strands each
    const int column = threadIdx.x / 16, fourth = threadIdx.x % 16;
    float v = (part[fourth][column] + part[fourth + 16][column]) + (part[fourth + 32][column] + part[fourth + 48][column]);
    v = lane_sum(v, 16);
    const int64_t cc = (int64_t)blockIdx.x * 4 * W + column;
    if (fourth != 0 || cc >= 2 * d) return;
    void* out = cc < d ? dgamma : dbeta;
    if (!out) return;
    const int64_t i = cc < d ? cc : cc - d;
    if (dtype == B200_F32) reinterpret_cast<float*>(out)[i] = v;
    else if (dtype == B200_F16) reinterpret_cast<__half*>(out)[i] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
}

// ---- rows of any length ---------------------------------------------------------------------------
// One block per row, element accesses, the row read again for each pass (out of L2): misaligned or odd rows
// past 8192 columns, Float32 gradients past 8192, everything past 16384.  Four to twelve times the floor:
// 7456 x 9001 BFloat16 forward 353 us (41), gradient 446 us (61), 2048 x 32768 318 (41) and 443 us (61),
// with 8-bit rows 442 and 628 us (52 each); Float32 gradient 4096 x 16384 494 us (123), 5000 x 12288 434 us (113).
// 118 instructions a thread and element forward, issue slots 64 % taken, HBM at 8 %.
__device__ __forceinline__ float block_sum(float v, float* buf) {
    v = lane_sum(v, 32);
    __syncthreads();
    if (threadIdx.x % 32 == 0) buf[threadIdx.x / 32] = v;
    __syncthreads();
    v = threadIdx.x % 32 < blockDim.x / 32 ? buf[threadIdx.x % 32] : 0.f;
    return lane_sum(v, 32);
}

template <typename T>
__global__ void __launch_bounds__(1024)
norm_forward_long_kernel(NormArgs a) {
    __shared__ float buf[32];
    grid_dependency_wait();
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx;
        T* y = reinterpret_cast<T*>(a.y) + row * a.ldy;
        float sum = 0.f;
        for (int64_t i = threadIdx.x; i < a.d; i += blockDim.x) sum += Elem<T>::get(x[i]);
        const float mean = block_sum(sum, buf) / (float)a.d;
        float m2 = 0.f;
        for (int64_t i = threadIdx.x; i < a.d; i += blockDim.x) { const float c = Elem<T>::get(x[i]) - mean; m2 = fmaf(c, c, m2); }
        const float rstd = 1.f / sqrtf(block_sum(m2, buf) / (float)a.d + a.eps);
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
        for (int64_t b = 0; b < a.d; b += blockDim.x) {
            const int64_t i = b + threadIdx.x;
            float h = 0.f;
            if (i < a.d) {
                h = (Elem<T>::get(x[i]) - mean) * rstd;
                const float g = a.gamma ? load_param(a.gamma, a.gamma_f32, dtype_of<T>(), i) : 1.f;
                const float o = a.beta ? load_param(a.beta, a.gamma_f32, dtype_of<T>(), i) : 0.f;
                y[i] = Elem<T>::put(fmaf(h, g, o));
            }
            if (a.q) {
                const uint32_t e = scale_byte(block_amax<1>(&h), a.e4m3);
                if (i < a.d) {
                    a.q[row * a.d + i] = encode<1>(&h, e, a.e4m3);
                    if (i % kBlock == 0) a.s[row * a.blocks + i / kBlock] = (uint8_t)e;
                }
            }
        }
    }
}

template <typename T>
__device__ __forceinline__ float norm_hat(const NormArgs& a, int64_t row, int64_t i, float mean, float rstd) {
    if (a.q) {
        float h;
        decode<1>(a.q[row * a.d + i], a.s[row * a.blocks + i / kBlock], a.e4m3, &h);
        return h;
    }
    return (Elem<T>::get(reinterpret_cast<const T*>(a.x)[row * a.ldx + i]) - mean) * rstd;
}

template <typename T>
__global__ void __launch_bounds__(1024)
norm_backward_long_kernel(NormArgs a) {
    __shared__ float buf[32];
    grid_dependency_wait();
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* dy = reinterpret_cast<const T*>(a.dy) + row * a.lddy;
        T* dx = reinterpret_cast<T*>(a.y) + row * a.ldy;
        const float rstd = a.rstd[row], mean = a.q ? 0.f : a.mean[row];
        float s1 = 0.f, s2 = 0.f;
        for (int64_t i = threadIdx.x; i < a.d; i += blockDim.x) {
            const float g = Elem<T>::get(dy[i]) * (a.gamma ? load_param(a.gamma, a.gamma_f32, dtype_of<T>(), i) : 1.f);
            s1 += g;
            s2 = fmaf(g, norm_hat<T>(a, row, i, mean, rstd), s2);
        }
        const float c1 = block_sum(s1, buf) / (float)a.d, c2 = block_sum(s2, buf) / (float)a.d;
        for (int64_t i = threadIdx.x; i < a.d; i += blockDim.x) {
            const float g = Elem<T>::get(dy[i]) * (a.gamma ? load_param(a.gamma, a.gamma_f32, dtype_of<T>(), i) : 1.f);
            const float h = norm_hat<T>(a, row, i, mean, rstd);
            dx[i] = Elem<T>::put(rstd * (g - fmaf(h, c2, c1)));
        }
    }
}

// dgamma and dbeta of long rows: 32 columns and a strand of rows per block; runs in front of the
// kernel above, which may write over dy or x.
template <typename T>
__global__ void __launch_bounds__(256)
norm_columns_long_kernel(NormArgs a) {
    __shared__ float2 part[8][33];
    grid_dependency_wait();
    const int lane = threadIdx.x % 32, strand = threadIdx.x / 32;
    const int64_t i = (int64_t)blockIdx.x * 32 + lane;
    float dg = 0.f, db = 0.f;
    if (i < a.d) {
        for (int64_t row = (int64_t)blockIdx.y * 8 + strand; row < a.rows; row += (int64_t)gridDim.y * 8) {
            const float dy = Elem<T>::get(reinterpret_cast<const T*>(a.dy)[row * a.lddy + i]);
            dg = fmaf(dy, norm_hat<T>(a, row, i, a.q ? 0.f : a.mean[row], a.q ? 0.f : a.rstd[row]), dg);
            db += dy;
        }
    }
    part[strand][lane] = make_float2(dg, db);
    __syncthreads();
    if (strand != 0 || i >= a.d) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) { dg += part[k][lane].x; db += part[k][lane].y; }
    float* out = a.partial + (int64_t)blockIdx.y * 2 * a.d;
    out[i] = dg;
    out[a.d + i] = db;
}

// ---- host ---------------------------------------------------------------------------------------
// Threads per row for E elements each: a power of two below a warp (at least a whole 8-bit block's
// lanes), whole warps above.
static int ring_group(int64_t d, int e, int v) {
    const int64_t need = (d + e - 1) / e;
    if (need > 32) return (int)((need + 31) / 32 * 32);
    int g = v == 1 ? 32 : 8;
    while (g < need) g *= 2;
    return g;
}
static int norm_vector(const NormArgs& a, int32_t dtype, bool aligned) {
    const int v = dtype == B200_F32 ? 4 : 8;
    return aligned && a.d % v == 0 && a.rows <= 0x3fffffff ? v : 1;    // the ring kernels count rows in 32 bits
}
// f(constant): how a row lies over its group.
template <bool WARPS, typename F>
static auto by_form(const NormArgs& a, int e, F f) {
    if (a.group % 32 == 0) {
        if (a.d == (int64_t)a.group * e) return f(std::integral_constant<int, kFilled>{});
        if constexpr (WARPS) return f(std::integral_constant<int, kOverWarps>{});
    }
    return f(std::integral_constant<int, kOverGroup>{});
}
// Dynamic shared memory that with the static one may pass 48 KB has to be allowed once per kernel and device.
static cudaError_t allow_shared(const void* kernel, size_t bytes, int dev) {
    if (bytes <= 32 * 1024) return cudaSuccess;
    static std::mutex mu;
    static std::vector<std::pair<const void*, int>> done;
    std::lock_guard<std::mutex> lk(mu);
    for (const auto& d : done) if (d.first == kernel && d.second == dev) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 219 * 1024);
    if (e == cudaSuccess) done.emplace_back(kernel, dev);
    return e;
}

// Columns of a thread for rows of any alignment: fewer where a row is less than a warp's worth of them.
template <typename F>
static auto any_elements(int64_t d, F f) {
    if (d <= 32 * 4) return f(std::integral_constant<int, 4>{});
    if (d <= 32 * 8) return f(std::integral_constant<int, 8>{});
    return f(std::integral_constant<int, kAnyElems>{});
}

struct NormLaunch {
    b200_stream_t st;
    NormArgs a;
    unsigned threads = 0, grid = 0;
    size_t smem = 0;
    // Blocks for a kernel: all resident, each with the same number of rows up to one.
    template <typename K> cudaError_t plan(K kernel, int per_block, size_t bytes) {
        threads = (unsigned)(per_block * a.group);
        smem = bytes;
        const cudaError_t e = allow_shared(reinterpret_cast<const void*>(kernel), smem, st->dev);
        if (e != cudaSuccess) return e;
        grid = balanced_grid((a.rows + per_block - 1) / per_block, resident_blocks(kernel, (int)threads, smem, st->dev));
        return cudaSuccess;
    }
    template <typename K> cudaError_t go(K kernel) {
        a.step = (int64_t)grid * (threads / a.group);
        a.x_step = a.step * a.ldx; a.y_step = a.step * a.ldy; a.dy_step = a.step * a.lddy;
        a.q_step = a.step * a.d; a.s_step = a.step * a.blocks;
        return launch_overlapped(kernel, grid, threads, smem, st->s, a);
    }
};

template <typename T, int E, int STAGES, int THREADS>
static cudaError_t forward_ring(b200_stream_t st, const NormArgs& a) {
    NormLaunch l{st, a};
    int per = a.group >= 256 ? 1 : 256 / a.group;
    while (per > 1 && a.rows < (int64_t)per * sm_count(st->dev) && (per / 2) * a.group >= 32) per /= 2;      // few rows: an SM each
    const size_t bytes = (size_t)STAGES * (E * sizeof(T)) * THREADS;
    auto run = [&](auto kernel) { const cudaError_t e = l.plan(kernel, per, bytes); return e == cudaSuccess ? l.go(kernel) : e; };
    auto form = [&](auto full) {
        constexpr int FORM = decltype(full)::value;
        if (!a.q) return run(norm_forward_ring_kernel<T, E, STAGES, THREADS, kAsIs, FORM>);
        return a.e4m3 ? run(norm_forward_ring_kernel<T, E, STAGES, THREADS, kE4M3, FORM>) : run(norm_forward_ring_kernel<T, E, STAGES, THREADS, kInt8, FORM>);
    };
    return by_form<true>(a, E, form);
}
template <typename T>
static cudaError_t run_forward(b200_stream_t st, NormArgs a, int v) {
    if (v > 1) {
        a.group = ring_group(a.d, 32, v);
        if (a.group <= 256) return forward_ring<T, 32, 3, 256>(st, a);
        if (a.group <= 512) return forward_ring<T, 32, 3, 512>(st, a);
    } else if (a.rows <= 0x3fffffff) {
        a.group = ring_group(a.d, kAnyElems, 1);
        if (a.group <= kAnyThreads) {
            NormLaunch l{st, a};
            l.a.pitch = piece_pitch(a.d * (int64_t)sizeof(T));
            // blocks of 256 threads where a row needs no more: several to an SM
            const int per = a.group >= 256 ? 1 : 256 / a.group;
            const size_t bytes = (size_t)per * kAnyStages * l.a.pitch;
            auto run = [&](auto kernel) { const cudaError_t e = l.plan(kernel, per, bytes); return e == cudaSuccess ? l.go(kernel) : e; };
            auto width = [&](auto w) {
                constexpr int W = decltype(w)::value;
                return any_elements(a.d, [&](auto e) {
                    constexpr int E = decltype(e)::value;
                    if constexpr (E == kAnyElems) {
                        if (a.group > 256) return a.q ? run(norm_forward_any_kernel<T, W, E, 512, true>) : run(norm_forward_any_kernel<T, W, E, 512, false>);
                    }
                    return a.q ? run(norm_forward_any_kernel<T, W, E, 256, true>) : run(norm_forward_any_kernel<T, W, E, 256, false>);
                });
            };
            if constexpr (sizeof(T) == 2) { if (a.units2) return width(std::integral_constant<int, 2>{}); }
            return width(std::integral_constant<int, 1>{});
        }
    }
    return launch_overlapped(norm_forward_long_kernel<T>, balanced_grid(a.rows, (int64_t)sm_count(st->dev) * 2), 1024u, 0, st->s, a);
}

// Gradient: plans first (the number of blocks sizes the workspace), then launches.
template <typename T, int E, int STAGES, int THREADS, int KEPT, bool HOLD, typename F>
static int32_t backward_ring(NormLaunch& l, F space) {
    constexpr int V = 16 / (int)sizeof(T);
    const int per = THREADS / l.a.group;
    size_t bytes = (size_t)STAGES * (E / V) * (16 + (KEPT ? V : 16)) * THREADS + (size_t)E * l.a.group * sizeof(float);
    const size_t columns = (size_t)per * 2 * l.a.d * sizeof(float);
    if (bytes < columns) bytes = columns;
    auto run = [&](auto kernel) -> int32_t {
        B200_CUDA(l.plan(kernel, per, bytes));
        B200_TRY(space((int64_t)l.grid));
        B200_CUDA(l.go(kernel));
        return B200_OK;
    };
    // with 32 columns a thread's registers are all taken, and predicates over fixed steps cost more than the
    // steps (16000 x 2624 BFloat16 54 -> 58 us)
    return by_form<E == 16>(l.a, E, [&](auto form) { return run(norm_backward_ring_kernel<T, E, STAGES, THREADS, KEPT, HOLD, decltype(form)::value>); });
}

// Workspace of one call.  Outside a capture it is the stream's scratch; inside one the graph gets an
// allocation of its own, so that graphs captured on one stream can be replayed side by side.
struct NormSpace {
    b200_stream_t st;
    void* temp = nullptr;
    int32_t get(size_t bytes, float** out) {
        cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
        B200_CUDA(cudaStreamIsCapturing(st->s, &cap));
        void* p = nullptr;
        if (cap == cudaStreamCaptureStatusNone) B200_TRY(scratch(st, bytes, &p));
        else { B200_TRY(b200_malloc_async(&temp, bytes, st)); p = temp; }
        *out = reinterpret_cast<float*>(p);
        return B200_OK;
    }
    int32_t release() { return temp ? b200_free_async(temp, st) : B200_OK; }
};

template <typename T>
static int32_t run_backward(b200_stream_t st, NormArgs a, int v, void* dgamma, void* dbeta, int32_t ptype) {
    constexpr bool k16 = sizeof(T) == 2;
    const bool columns = dgamma || dbeta;
    NormSpace space{st};
    NormLaunch l{st, a};
    int64_t blocks = 0;
    // room for the partials of `n` blocks
    auto room = [&](int64_t n) -> int32_t {
        blocks = n;
        return columns ? space.get((size_t)n * 2 * a.d * sizeof(float), &l.a.partial) : B200_OK;
    };
    const int g16 = ring_group(a.d, 16, v), g32 = ring_group(a.d, 32, v);
    // 32 columns per thread where that holds more rows side by side on an SM than 16 do: fewer
    // instructions per element (16384 x 4096 BFloat16: 69 us, with 16 columns 80; 8192 x 8192: 93 and 84,
    // one row per SM either way).  Up to 2048 columns only where they fill the threads (16384 x 2048 out
    // of 8 bits 38 us, with 16 columns 42; 16384 x 1536, which they do not fill, 39 and 33).
    const bool wide = k16 && v > 1 && g32 <= 384 && (g16 > 512 || ((a.d > 2048 || a.d % 1024 == 0) && 384 / g32 > 512 / g16));
    if (wide) {
        l.a.group = g32;
        if constexpr (k16) {
            if (a.q && a.e4m3) B200_TRY((backward_ring<T, 32, 4, 384, kE4M3, true>(l, room)));
            else if (a.q) B200_TRY((backward_ring<T, 32, 4, 384, kInt8, true>(l, room)));
            else B200_TRY((backward_ring<T, 32, 3, 384, kAsIs, true>(l, room)));
        }
    } else if (v > 1 && g16 <= 512) {
        l.a.group = g16;
        if (a.q && a.e4m3) B200_TRY((backward_ring<T, 16, k16 ? 4 : 3, 512, kE4M3, true>(l, room)));
        else if (a.q) B200_TRY((backward_ring<T, 16, k16 ? 4 : 3, 512, kInt8, true>(l, room)));
        else B200_TRY((backward_ring<T, 16, k16 ? 4 : 2, 512, kAsIs, true>(l, room)));
    } else if (v > 1 && k16 && g32 <= 512) {
        l.a.group = g32;
        if constexpr (k16) {
            if (a.q && a.e4m3) B200_TRY((backward_ring<T, 32, 2, 512, kE4M3, false>(l, room)));
            else if (a.q) B200_TRY((backward_ring<T, 32, 2, 512, kInt8, false>(l, room)));
            else B200_TRY((backward_ring<T, 32, 2, 512, kAsIs, false>(l, room)));
        }
    } else if (v == 1 && a.rows <= 0x3fffffff && ring_group(a.d, kAnyElems, 1) <= kAnyThreads) {
        l.a.group = ring_group(a.d, kAnyElems, 1);
        l.a.pitch = piece_pitch(a.d * (int64_t)sizeof(T));
        l.a.pitch_x = piece_pitch(a.q ? a.d : a.d * (int64_t)sizeof(T));
        const int per = kAnyThreads / l.a.group;
        size_t bytes = (size_t)per * kAnyStages * (l.a.pitch + l.a.pitch_x);
        if (bytes < (size_t)per * 2 * a.d * sizeof(float)) bytes = (size_t)per * 2 * a.d * sizeof(float);
        auto run = [&](auto kernel) -> int32_t {
            B200_CUDA(l.plan(kernel, per, bytes));
            B200_TRY(room(l.grid));
            B200_CUDA(l.go(kernel));
            return B200_OK;
        };
        B200_TRY(any_elements(a.d, [&](auto e) -> int32_t {
            constexpr int E = decltype(e)::value;
            if constexpr (k16) {
                if (a.units2) return a.q ? run(norm_backward_any_kernel<T, 2, E, true>) : run(norm_backward_any_kernel<T, 2, E, false>);
            }
            return a.q ? run(norm_backward_any_kernel<T, 1, E, true>) : run(norm_backward_any_kernel<T, 1, E, false>);
        }));
    } else {
        const int64_t tiles = (a.d + 31) / 32;
        int64_t n = (int64_t)sm_count(st->dev) * 8 / tiles;
        if (n > (a.rows + 7) / 8) n = (a.rows + 7) / 8;
        if (n < 1) n = 1;
        B200_TRY(room(n));
        if (columns) norm_columns_long_kernel<T><<<dim3((unsigned)tiles, (unsigned)n), 256, 0, st->s>>>(l.a);
        if (a.y) B200_CUDA(launch_overlapped(norm_backward_long_kernel<T>, balanced_grid(a.rows, (int64_t)sm_count(st->dev) * 2), 1024u, 0, st->s, l.a));
    }
    if (columns) {
        B200_CUDA(launch_overlapped(a.d % 4 == 0 ? norm_fold_kernel<true> : norm_fold_kernel<false>, (unsigned)((2 * a.d + 63) / 64), 1024u, 0, st->s, (const float*)l.a.partial, blocks, a.d, dgamma, dbeta, ptype));
        B200_TRY(space.release());
    }
    return B200_OK;
}

static int32_t check_params(const b200_tensor* p, const char* name, const RowView& x, int32_t* ptype) {
    if (!p) return B200_OK;
    B200_TRY(check_tensor(p, name));
    if (tensor_numel(p) != x.d) return fail(B200_INVALID_ARG, "%s: needs one value per element of a row", name);
    if (!tensor_is_contiguous(p)) return fail(B200_UNSUPPORTED, "%s: must be dense", name);
    if (p->dtype != B200_F32 && p->dtype != x.dtype) return fail(B200_UNSUPPORTED, "%s: must be Float32 or of the rows' type", name);
    if (*ptype >= 0 && *ptype != p->dtype) return fail(B200_INVALID_ARG, "%s: the parameters and their gradients must have one element type", name);
    *ptype = p->dtype;
    return B200_OK;
}
static int32_t check_row_values(const b200_tensor* t, const char* name, int64_t rows) {
    B200_TRY(check_tensor(t, name));
    if (t->dtype != B200_F32) return fail(B200_UNSUPPORTED, "%s: must be Float32", name);
    if (tensor_numel(t) != rows) return fail(B200_INVALID_ARG, "%s: needs one value per row", name);
    if (!tensor_is_contiguous(t)) return fail(B200_UNSUPPORTED, "%s: must be dense", name);
    return B200_OK;
}
// Codes of rows: dense, one scale byte per 32 elements of a row; a row is the first dimension.
static int32_t check_row_codes(const b200_tensor* Q, const b200_tensor* S, const RowView& x, int lead, const char* name) {
    B200_TRY(check_codes(Q, S, name));
    if (lead != 1) return fail(B200_UNSUPPORTED, "%s: rows kept in 8 bits are normalised along the first dimension", name);
    if (Q->shape[0] != x.d || tensor_numel(Q) != x.d * x.rows) return fail(B200_INVALID_ARG, "%s: differs in shape from the rows", name);
    if (!tensor_is_contiguous(Q) || !tensor_is_contiguous(S)) return fail(B200_UNSUPPORTED, "%s: must be dense", name);
    return B200_OK;
}

}  // namespace b200

using namespace b200;

extern "C" int32_t b200_layernorm(b200_stream_t st, const b200_tensor* Y, const b200_tensor* X, int32_t lead, const b200_tensor* gamma,
                                  const b200_tensor* beta, double eps, const b200_tensor* mean, const b200_tensor* rstd,
                                  const b200_tensor* Q, const b200_tensor* S) {
    RowView x, y;
    if (lead < 1) return fail(B200_INVALID_ARG, "layernorm: at least one dimension is normalised");
    B200_TRY(row_view(X, lead, "layernorm source", &x));
    B200_TRY(row_view_out(Y, lead, "layernorm destination", &y));
    if (!same_shape(X, Y)) return fail(B200_INVALID_ARG, "layernorm: source and destination differ in shape");
    if (X->dtype != Y->dtype) return fail(B200_INVALID_ARG, "layernorm: source and destination differ in element type");
    if (!is_row_type(x.dtype)) return fail(B200_UNSUPPORTED, "layernorm: Float16, BFloat16 or Float32 rows");
    if (!(eps >= 0)) return fail(B200_INVALID_ARG, "layernorm: eps must not be negative");
    int32_t ptype = -1;
    B200_TRY(check_params(gamma, "layernorm gamma", x, &ptype));
    B200_TRY(check_params(beta, "layernorm beta", x, &ptype));
    if (mean) B200_TRY(check_row_values(mean, "layernorm mean", x.rows));
    if (rstd) B200_TRY(check_row_values(rstd, "layernorm rstd", x.rows));
    if ((Q != nullptr) != (S != nullptr)) return fail(B200_INVALID_ARG, "layernorm: codes and scales belong together");
    if (Q) B200_TRY(check_row_codes(Q, S, x, lead, "layernorm checkpoint"));
    if (x.d > 0x7fffffff) return fail(B200_TOO_LARGE, "layernorm: rows of at most 2^31-1 elements");
    B200_TRY(enter(st));
    StreamGuard guard(st);
    if (x.rows == 0) return B200_OK;
    if (x.d == 0) {          // moments over no elements
        for (const b200_tensor* t : {mean, rstd})
            if (t) B200_TRY(b200_memset_async(t->ptr, 0x7fc00000, 4, (size_t)x.rows, st));
        return finish(st, "b200_layernorm");
    }
    NormArgs a{};
    a.x = x.p; a.ldx = x.ld; a.y = y.p; a.ldy = y.ld; a.rows = x.rows; a.d = x.d; a.eps = (float)eps;
    a.gamma = gamma ? gamma->ptr : nullptr;
    a.beta = beta ? beta->ptr : nullptr;
    a.gamma_f32 = ptype == B200_F32;
    a.mean = mean ? (float*)mean->ptr : nullptr;
    a.rstd = rstd ? (float*)rstd->ptr : nullptr;
    if (Q) { a.q = (uint8_t*)Q->ptr; a.s = (uint8_t*)S->ptr; a.e4m3 = Q->dtype == B200_U8; a.blocks = row_blocks(x.d); }
    const int full = x.dtype == B200_F32 ? 4 : 8;
    a.units2 = x.dtype != B200_F32 && x.d % 2 == 0 && rows_aligned(x, 4) && rows_aligned(y, 4) && (!Q || reinterpret_cast<uintptr_t>(a.q) % 2 == 0);
    const int v = norm_vector(a, x.dtype, rows_aligned(x, 16) && rows_aligned(y, 16) && (!Q || reinterpret_cast<uintptr_t>(a.q) % full == 0));
    switch (x.dtype) {
        case B200_F16: B200_CUDA(run_forward<__half>(st, a, v)); break;
        case B200_BF16: B200_CUDA(run_forward<__nv_bfloat16>(st, a, v)); break;
        default: B200_CUDA(run_forward<float>(st, a, v)); break;
    }
    return finish(st, "b200_layernorm");
}

extern "C" int32_t b200_layernorm_backward(b200_stream_t st, const b200_tensor* dX, const b200_tensor* dgamma, const b200_tensor* dbeta,
                                           const b200_tensor* dY, int32_t lead, const b200_tensor* X, const b200_tensor* Q,
                                           const b200_tensor* S, const b200_tensor* gamma, const b200_tensor* mean,
                                           const b200_tensor* rstd) {
    RowView dy, dx{}, x{};
    if (lead < 1) return fail(B200_INVALID_ARG, "layernorm gradient: at least one dimension is normalised");
    B200_TRY(row_view(dY, lead, "layernorm gradient", &dy));
    if (!is_row_type(dy.dtype)) return fail(B200_UNSUPPORTED, "layernorm gradient: Float16, BFloat16 or Float32 rows");
    if (!dX && !dgamma && !dbeta) return fail(B200_INVALID_ARG, "layernorm gradient: no gradient is asked for");
    if (dX) {
        B200_TRY(row_view_out(dX, lead, "layernorm gradient destination", &dx));
        if (!same_shape(dX, dY) || dX->dtype != dY->dtype) return fail(B200_INVALID_ARG, "layernorm gradient: dX and dY differ");
    }
    if ((X != nullptr) == (Q != nullptr) || (Q != nullptr) != (S != nullptr))
        return fail(B200_INVALID_ARG, "layernorm gradient: needs the source or its codes and scales, one of the two");
    int32_t ptype = -1;
    B200_TRY(check_params(gamma, "layernorm gamma", dy, &ptype));
    B200_TRY(check_params(dgamma, "layernorm dgamma", dy, &ptype));
    B200_TRY(check_params(dbeta, "layernorm dbeta", dy, &ptype));
    if (!rstd) return fail(B200_INVALID_ARG, "layernorm gradient: needs rstd");
    B200_TRY(check_row_values(rstd, "layernorm rstd", dy.rows));
    if (X) {
        B200_TRY(row_view(X, lead, "layernorm source", &x));
        if (!same_shape(X, dY) || X->dtype != dY->dtype) return fail(B200_INVALID_ARG, "layernorm gradient: source and dY differ");
        if (!mean) return fail(B200_INVALID_ARG, "layernorm gradient: needs the mean of the source's rows");
        B200_TRY(check_row_values(mean, "layernorm mean", dy.rows));
    } else {
        B200_TRY(check_row_codes(Q, S, dy, lead, "layernorm checkpoint"));
    }
    if (dy.d > 0x7fffffff) return fail(B200_TOO_LARGE, "layernorm: rows of at most 2^31-1 elements");
    B200_TRY(enter(st));
    StreamGuard guard(st);
    if (dy.d == 0) return B200_OK;
    if (dy.rows == 0) {      // sums over no rows
        if (dgamma) B200_TRY(b200_memset_async(dgamma->ptr, 0, (int32_t)dtype_size(ptype), (size_t)dy.d, st));
        if (dbeta) B200_TRY(b200_memset_async(dbeta->ptr, 0, (int32_t)dtype_size(ptype), (size_t)dy.d, st));
        return finish(st, "b200_layernorm_backward");
    }
    NormArgs a{};
    a.dy = dy.p; a.lddy = dy.ld; a.y = dX ? dx.p : nullptr; a.ldy = dx.ld; a.x = X ? x.p : nullptr; a.ldx = x.ld;
    a.rows = dy.rows; a.d = dy.d;
    a.gamma = gamma ? gamma->ptr : nullptr;
    a.gamma_f32 = ptype == B200_F32;
    a.mean = X ? (float*)mean->ptr : nullptr;
    a.rstd = (float*)rstd->ptr;
    if (Q) { a.q = (uint8_t*)Q->ptr; a.s = (uint8_t*)S->ptr; a.e4m3 = Q->dtype == B200_U8; a.blocks = row_blocks(dy.d); }
    const int full = dy.dtype == B200_F32 ? 4 : 8;
    a.units2 = dy.dtype != B200_F32 && dy.d % 2 == 0 && rows_aligned(dy, 4) && (!dX || rows_aligned(dx, 4)) && (!X || rows_aligned(x, 4)) &&
               (!Q || reinterpret_cast<uintptr_t>(a.q) % 2 == 0);
    const int v = norm_vector(a, dy.dtype, rows_aligned(dy, 16) && (!dX || rows_aligned(dx, 16)) && (!X || rows_aligned(x, 16)) &&
                                               (!Q || reinterpret_cast<uintptr_t>(a.q) % full == 0));
    void* dg = dgamma ? dgamma->ptr : nullptr;
    void* db = dbeta ? dbeta->ptr : nullptr;
    switch (dy.dtype) {
        case B200_F16: B200_TRY(run_backward<__half>(st, a, v, dg, db, ptype)); break;
        case B200_BF16: B200_TRY(run_backward<__nv_bfloat16>(st, a, v, dg, db, ptype)); break;
        default: B200_TRY(run_backward<float>(st, a, v, dg, db, ptype)); break;
    }
    return finish(st, "b200_layernorm_backward");
}
