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

constexpr int kNormThreads = 256;
constexpr int kNormElems = 16;          // elements of a row per thread
constexpr int kNormMaxGroup = 512;      // threads per row

struct NormArgs {
    const void *x, *dy, *gamma, *beta;
    void *y;                            // forward: y; gradient: dx
    float *mean, *rstd;
    uint8_t *q, *s;                     // codes and scale bytes of the normalised rows
    float *partial;                     // gradient: [block][2][d] sums of dy*h and dy
    int64_t ldx, ldy, lddy, rows, d, blocks;
    float eps;
    int32_t gamma_f32, e4m3, group;     // group: threads per row, a power of two
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

// ---- rows in registers --------------------------------------------------------------------------
// `group` threads hold one row, NV vectors of V elements each, so a row is read once; a block of
// kNormThreads (or one group, if that is larger) works on several rows side by side and walks over
// the rows with the grid's stride.  gamma and beta stay in registers.
//
// Moments in one exchange: every warp takes the mean of its share and the squares about that mean;
// the shares combine as M2 = sum M2_w + n_w (mean_w - mean)^2 (Chan, Golub and LeVeque 1983), which
// loses nothing when the mean is large against the spread.
template <typename T, int V, int NV, bool KEEP>
__global__ void __launch_bounds__(kNormMaxGroup)
norm_forward_kernel(NormArgs a) {
    __shared__ float2 share[2][kNormMaxGroup / 32];
    grid_dependency_wait();
    const int G = a.group, group = threadIdx.x / G, t = threadIdx.x % G;
    const int per_block = blockDim.x / G, warps = G / 32, warp = t / 32;
    const int width = G < 32 ? G : 32;
    const int nvec = (int)(a.d / V);
    const T* x = reinterpret_cast<const T*>(a.x);
    T* y = reinterpret_cast<T*>(a.y);

    float gm[NV * V], bt[NV * V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int vi = t + k * G;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            gm[k * V + i] = a.gamma && vi < nvec ? load_param(a.gamma, a.gamma_f32, dtype_of<T>(), (int64_t)vi * V + i) : 1.f;
            bt[k * V + i] = a.beta && vi < nvec ? load_param(a.beta, a.gamma_f32, dtype_of<T>(), (int64_t)vi * V + i) : 0.f;
        }
    }
    // elements of this warp's share of a row
    int count = 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int left = nvec - (k * G + warp * 32);
        count += (left < 0 ? 0 : left > width ? width : left) * V;
    }
    int parity = 0;
    for (int64_t base = (int64_t)blockIdx.x * per_block; base < a.rows; base += (int64_t)gridDim.x * per_block) {
        const int64_t row = base + group;
        const bool live = row < a.rows;
        float v[NV * V];
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int vi = t + k * G;
            RawVec<T, V> r{};
            if (live && vi < nvec) r = ld_raw<T, V>(x + row * a.ldx + (int64_t)vi * V);
            unpack<T, V>(r, v + k * V);
        }
#pragma unroll
        for (int i = 0; i < NV * V; ++i) sum += v[i];
        sum = lane_sum(sum, width);
        float mean = count ? sum / (float)count : 0.f, m2 = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (t + k * G < nvec) {
#pragma unroll
                for (int i = 0; i < V; ++i) { const float c = v[k * V + i] - mean; m2 = fmaf(c, c, m2); }
            }
        }
        m2 = lane_sum(m2, width);
        if (warps > 1) {
            // a group has whole warps here and is the block or a power-of-two part of it
            float2* sh = share[parity] + group * warps;
            if ((t & 31) == 0) sh[warp] = make_float2(sum, m2);
            __syncthreads();
            parity ^= 1;
            float total = 0.f;
            for (int w = 0; w < warps; ++w) total += sh[w].x;
            mean = total / (float)a.d;
            m2 = 0.f;
            for (int w = 0; w < warps; ++w) {
                int n = 0;
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    const int left = nvec - (k * G + w * 32);
                    n += (left < 0 ? 0 : left > 32 ? 32 : left) * V;
                }
                if (n) { const float c = sh[w].x / (float)n - mean; m2 += sh[w].y + (float)n * c * c; }
            }
        }
        const float rstd = 1.f / sqrtf(m2 / (float)a.d + a.eps);
        if (live && t == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int vi = t + k * G;
            const bool in = live && vi < nvec;
            float o[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[k * V + i] = in ? (v[k * V + i] - mean) * rstd : 0.f;
                o[i] = fmaf(v[k * V + i], gm[k * V + i], bt[k * V + i]);
            }
            if (in) st_raw<T, V>(y + row * a.ldy + (int64_t)vi * V, pack<T, V>(o));
            if constexpr (KEEP) {
                const uint32_t e = scale_byte(block_amax<V>(v + k * V), a.e4m3);
                if (in) {
                    st_raw<uint8_t, V>(a.q + row * a.d + (int64_t)vi * V, encode<V>(v + k * V, e, a.e4m3));
                    if (vi % (kBlock / V) == 0) a.s[row * a.blocks + vi / (kBlock / V)] = (uint8_t)e;
                }
            }
        }
    }
}

template <typename T, int V, int NV, bool KEPT>
__global__ void __launch_bounds__(kNormMaxGroup)
norm_backward_kernel(NormArgs a) {
    __shared__ float2 share[2][kNormMaxGroup / 32];
    extern __shared__ float column[];   // [2][d] when several rows share the block
    grid_dependency_wait();
    const int G = a.group, group = threadIdx.x / G, t = threadIdx.x % G;
    const int per_block = blockDim.x / G, warps = G / 32, warp = t / 32;
    const int width = G < 32 ? G : 32;
    const int nvec = (int)(a.d / V);
    const T* x = reinterpret_cast<const T*>(a.x);
    const T* dy = reinterpret_cast<const T*>(a.dy);
    T* dx = reinterpret_cast<T*>(a.y);

    float gm[NV * V], dg[NV * V], db[NV * V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int vi = t + k * G;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            gm[k * V + i] = a.gamma && vi < nvec ? load_param(a.gamma, a.gamma_f32, dtype_of<T>(), (int64_t)vi * V + i) : 1.f;
            dg[k * V + i] = db[k * V + i] = 0.f;
        }
    }
    int parity = 0;
    for (int64_t base = (int64_t)blockIdx.x * per_block; base < a.rows; base += (int64_t)gridDim.x * per_block) {
        const int64_t row = base + group;
        const bool live = row < a.rows;
        const float rstd = live ? a.rstd[row] : 0.f;
        const float mean = !KEPT && live ? a.mean[row] : 0.f;
        float h[NV * V], g[NV * V];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int vi = t + k * G;
            const bool in = live && vi < nvec;
            RawVec<T, V> r{};
            if (in) r = ld_raw<T, V>(dy + row * a.lddy + (int64_t)vi * V);
            unpack<T, V>(r, g + k * V);
            if constexpr (KEPT) {
                RawVec<uint8_t, V> c{};
                uint32_t e = 0;
                if (in) {
                    c = ld_raw<uint8_t, V>(a.q + row * a.d + (int64_t)vi * V);
                    e = a.s[row * a.blocks + vi / (kBlock / V)];
                }
                decode<V>(c, e, a.e4m3, h + k * V);
            } else {
                r = RawVec<T, V>{};
                if (in) r = ld_raw<T, V>(x + row * a.ldx + (int64_t)vi * V);
                unpack<T, V>(r, h + k * V);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int j = k * V + i;
                if constexpr (!KEPT) h[j] = in ? (h[j] - mean) * rstd : 0.f;
                if (!in) h[j] = 0.f;
                dg[j] = fmaf(g[j], h[j], dg[j]);
                db[j] += g[j];
                g[j] *= gm[j];
                s1 += g[j];
                s2 = fmaf(g[j], h[j], s2);
            }
        }
        s1 = lane_sum(s1, width);
        s2 = lane_sum(s2, width);
        if (warps > 1) {
            float2* sh = share[parity] + group * warps;
            if ((t & 31) == 0) sh[warp] = make_float2(s1, s2);
            __syncthreads();
            parity ^= 1;
            s1 = s2 = 0.f;
            for (int w = 0; w < warps; ++w) { s1 += sh[w].x; s2 += sh[w].y; }
        }
        const float c1 = s1 / (float)a.d, c2 = s2 / (float)a.d;
        if (dx) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int vi = t + k * G;
                float o[V];
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = rstd * (g[k * V + i] - fmaf(h[k * V + i], c2, c1));
                if (live && vi < nvec) st_raw<T, V>(dx + row * a.ldy + (int64_t)vi * V, pack<T, V>(o));
            }
        }
    }
    if (!a.partial) return;
    float* out = a.partial + (int64_t)blockIdx.x * 2 * a.d;
    // rows of one block, group after group, so that the order of the sum is fixed
    for (int gi = 0; gi < per_block; ++gi) {
        if (gi == group) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int vi = t + k * G;
                if (vi < nvec) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const int64_t c = (int64_t)vi * V + i;
                        float u = dg[k * V + i], w = db[k * V + i];
                        if (gi > 0) { u += column[c]; w += column[a.d + c]; }
                        if (gi + 1 < per_block) { column[c] = u; column[a.d + c] = w; }
                        else { out[c] = u; out[a.d + c] = w; }
                    }
                }
            }
        }
        if (per_block > 1) __syncthreads();
    }
}

// Sums the blocks' partials: 32 columns per block, eight strands of blocks, joined in a fixed order.
__global__ void __launch_bounds__(256)
norm_fold_kernel(const float* partial, int64_t nblocks, int64_t d, void* dgamma, void* dbeta, int32_t dtype) {
    __shared__ float part[8][33];
    grid_dependency_wait();
    const int lane = threadIdx.x % 32, strand = threadIdx.x / 32;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;      // over [dgamma | dbeta]
    float sum = 0.f;
    if (c < 2 * d) for (int64_t b = strand; b < nblocks; b += 8) sum += partial[b * 2 * d + c];
    part[strand][lane] = sum;
    __syncthreads();
    if (strand != 0 || c >= 2 * d) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) sum += part[k][lane];
    void* out = c < d ? dgamma : dbeta;
    if (!out) return;
    const int64_t i = c < d ? c : c - d;
    if (dtype == B200_F32) reinterpret_cast<float*>(out)[i] = sum;
    else if (dtype == B200_F16) reinterpret_cast<__half*>(out)[i] = __float2half_rn(sum);
    else reinterpret_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(sum);
}

// ---- rows of any length ---------------------------------------------------------------------------
// One block per row, element accesses, the row read again for each pass (out of L2).
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
// Threads per row: 16 elements each; at least a whole 8-bit block's lanes.
static int norm_group(int64_t d, int v) {
    int g = v == 1 ? 32 : 8;
    while ((int64_t)g * kNormElems < d) g *= 2;
    return g;
}
static int norm_vector(const NormArgs& a, int32_t dtype, bool aligned) {
    const int v = dtype == B200_F32 ? 4 : 8;
    return aligned && a.d % v == 0 ? v : 1;
}

template <typename T, int V, int NV>
static cudaError_t launch_forward(b200_stream_t st, const NormArgs& a, int threads) {
    const int64_t tiles = (a.rows + threads / a.group - 1) / (threads / a.group);
    auto go = [&](auto kernel) {
        return launch_overlapped(kernel, balanced_grid(tiles, resident_blocks(kernel, threads, 0, st->dev)), (unsigned)threads, 0, st->s, a);
    };
    return a.q ? go(norm_forward_kernel<T, V, NV, true>) : go(norm_forward_kernel<T, V, NV, false>);
}
template <typename T>
static cudaError_t run_forward(b200_stream_t st, NormArgs a, int v) {
    constexpr int FV = 16 / (int)sizeof(T);
    a.group = norm_group(a.d, v);
    if (a.group > kNormMaxGroup)
        return launch_overlapped(norm_forward_long_kernel<T>, balanced_grid(a.rows, (int64_t)sm_count(st->dev) * 2), 1024u, 0, st->s, a);
    const int threads = a.group > kNormThreads ? a.group : kNormThreads;
    return v == 1 ? launch_forward<T, 1, kNormElems>(st, a, threads) : launch_forward<T, FV, kNormElems / FV>(st, a, threads);
}

template <typename T>
struct NormBackward {
    static constexpr int FV = 16 / (int)sizeof(T);
    b200_stream_t st;
    NormArgs a;
    int v, threads = 0;
    unsigned grid = 0;
    size_t smem = 0;

    template <typename K> void plan(K kernel) {
        threads = a.group > kNormThreads ? a.group : kNormThreads;
        const int per = threads / a.group;
        smem = per > 1 ? 2 * a.d * sizeof(float) : 0;
        grid = balanced_grid((a.rows + per - 1) / per, resident_blocks(kernel, threads, smem, st->dev));
    }
    template <typename F> cudaError_t with_kernel(F f) {
        if (v == 1) return a.q ? f(norm_backward_kernel<T, 1, kNormElems, true>) : f(norm_backward_kernel<T, 1, kNormElems, false>);
        return a.q ? f(norm_backward_kernel<T, FV, kNormElems / FV, true>) : f(norm_backward_kernel<T, FV, kNormElems / FV, false>);
    }
};

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
    const bool columns = dgamma || dbeta;
    NormSpace space{st};
    a.group = norm_group(a.d, v);
    int64_t blocks;
    if (a.group <= kNormMaxGroup) {
        NormBackward<T> b{st, a, v};
        b.with_kernel([&](auto k) { b.plan(k); return cudaSuccess; });
        blocks = b.grid;
        if (columns) B200_TRY(space.get((size_t)blocks * 2 * a.d * sizeof(float), &b.a.partial));
        a.partial = b.a.partial;
        B200_CUDA(b.with_kernel([&](auto k) { return launch_overlapped(k, b.grid, (unsigned)b.threads, b.smem, st->s, b.a); }));
    } else {
        const int64_t tiles = (a.d + 31) / 32;
        blocks = (int64_t)sm_count(st->dev) * 8 / tiles;
        if (blocks > (a.rows + 7) / 8) blocks = (a.rows + 7) / 8;
        if (blocks < 1) blocks = 1;
        if (columns) {
            B200_TRY(space.get((size_t)blocks * 2 * a.d * sizeof(float), &a.partial));
            norm_columns_long_kernel<T><<<dim3((unsigned)tiles, (unsigned)blocks), 256, 0, st->s>>>(a);
        }
        if (a.y) B200_CUDA(launch_overlapped(norm_backward_long_kernel<T>, balanced_grid(a.rows, (int64_t)sm_count(st->dev) * 2), 1024u, 0, st->s, a));
    }
    if (columns) {
        B200_CUDA(launch_overlapped(norm_fold_kernel, (unsigned)((2 * a.d + 31) / 32), 256u, 0, st->s, (const float*)a.partial, blocks, a.d, dgamma, dbeta, ptype));
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
    if (x.rows == 0 || x.d == 0) return B200_OK;
    NormArgs a{};
    a.x = x.p; a.ldx = x.ld; a.y = y.p; a.ldy = y.ld; a.rows = x.rows; a.d = x.d; a.eps = (float)eps;
    a.gamma = gamma ? gamma->ptr : nullptr;
    a.beta = beta ? beta->ptr : nullptr;
    a.gamma_f32 = ptype == B200_F32;
    a.mean = mean ? (float*)mean->ptr : nullptr;
    a.rstd = rstd ? (float*)rstd->ptr : nullptr;
    if (Q) { a.q = (uint8_t*)Q->ptr; a.s = (uint8_t*)S->ptr; a.e4m3 = Q->dtype == B200_U8; a.blocks = row_blocks(x.d); }
    const int full = x.dtype == B200_F32 ? 4 : 8;
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
