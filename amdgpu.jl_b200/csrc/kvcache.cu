// Key/value cache held in 8 bits, in pages: new tokens are written (keys turned to their positions on
// the way) and contexts are read back.  Scatter and gather of whole rows beside the element gather and
// compaction of src/kernels/indexing.jl:8-36.
//
// A cache is four arrays: codes (head size, heads, page size, pages) and scale bytes (blocks of 32 of
// a head, heads, page size, pages), for keys and for values.  Slots and pages are 1-based; slot s is
// place (s-1) mod page size of page (s-1) div page size + 1.
#include "rowops.cuh"

namespace b200 {

struct CacheSide {                              // keys or values
    const void* x;                              // tokens: (head size, heads, tokens)
    void* out;                                  // read back: (head size, heads, places, sequences)
    uint8_t *q, *s;
    int64_t xh, xt, oh, ol, ob;                 // element strides of tokens and of the read-back array
    int64_t qh, qp, qn, sh, sp, sn;             // strides of codes and scale bytes: head, place, page
    int32_t d, units;                           // units: vectors per token
    FastDiv per_head;                           // vectors per head
};
struct CacheArgs {
    CacheSide k, v;
    const void *slots, *pos, *pages, *lengths;
    const uint64_t* table;
    uint32_t* owner;                            // per slot: highest token that claims it, plus one
    int32_t* err;
    int64_t tokens, nslots, npages, pl, pb, most, places, seqs;   // pl, pb: strides of the page table
    int64_t islots, ipos, ilengths;                               // their strides
    int32_t heads, page, rot, half, slots_wide, pos_wide, pages_wide, lengths_wide, e4m3, group;
    int32_t tile, parts, abreast, wide;                           // reading: tokens of a block, blocks of a token, tokens side by side
    FastDiv per_page, per_token;
    float factor;
};

// Tokens above this many settle two claims on one slot through a table instead of by looking through
// the later slots.  The table has a word for every slot of the cache, whatever the call writes: 4 bytes a
// slot of scratch, which the stream keeps (inside a capture: of an allocation of the graph's own).
constexpr int64_t kScanTokens = 2048;

// Twice per call: first the words of the call's own slots are cleared (a cache may have many more), then claimed.
template <bool CLEAR>
__global__ void __launch_bounds__(256)
cache_claim_kernel(CacheArgs a) {
    grid_dependency_wait();
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= a.tokens) return;
    const int64_t slot = load_int(a.slots, a.slots_wide, t * a.islots);
    if (slot < 1 || slot > a.nslots) return;
    if constexpr (CLEAR) a.owner[slot - 1] = 0;
    else atomicMax(a.owner + slot - 1, (uint32_t)t + 1u);
}

// V elements at `p`: 32 bytes are one access where `wide` says that they are aligned.
template <typename T, int V>
__device__ __forceinline__ RawVec<T, V> load_row(const T* p, bool wide) {
    if constexpr (sizeof(T) * V == 32) return ld_raw32(p, wide);
    else return ld_raw_cached<T, V>(p);
}
template <typename T, int V>
__device__ __forceinline__ void unpack_any(const RawVec<T, V>& r, F2* v) {
    if constexpr (V == 1) { float x; unpack<T, 1>(r, &x); v[0] = f2(x, 0.f); }
    else unpack2<T, V>(r, v);
}

// One vector of a token: which side, head and place in it.
struct CacheUnit { bool key, in; int h, i; };
template <int V>
__device__ __forceinline__ CacheUnit cache_unit(const CacheArgs& a, int u) {
    CacheUnit c;
    c.key = u < a.k.units;
    if (!c.key) u -= a.k.units;
    const CacheSide& side = c.key ? a.k : a.v;
    const bool some = u < side.units;
    c.h = some ? (int)side.per_head.div((uint32_t)u) : 0;
    c.i = some ? (u - c.h * (int)side.per_head.d) * V : 0;
    c.in = some && c.i < side.d;
    return c;
}

// How keys turn on the way: vector against vector (half layout), within a vector (interleaved), or, where
// pairs do not lie so, element by element against partners that are read one by one.
enum { kNoTurn = 0, kTurnHalf = 1, kTurnInterleaved = 2, kTurnUneven = 3 };

// Place of pair i's cosine and sine: the pairs of a thread's vector lie apart, those of neighbouring threads
// side by side (no bank is asked for twice).
template <int V, int TURN>
__device__ __forceinline__ int turn_at(int i, int half) {
    constexpr int PER = V == 1 || TURN == kTurnUneven ? 1 : TURN == kTurnHalf ? V : V / 2;
    return PER == 1 ? i : (i % PER) * (half / PER) + i / PER;
}

// `group` threads (whole warps) per token; the 32/V lanes of a block of 32 are neighbours.  A thread's first
// vectors are on their way while the slot is looked at and the angles are worked out.  Bound by latency
// and instruction issue: a token waits for its slot, then for its angles; working out both at once and fetching
// vectors ahead came out the same.  One B200, BFloat16 to e4m3, 8 heads of 128: 8192 tokens 17 us with the
// claims settled (51 MB: 8 us), 32768 tokens 58 us (3.5 TB/s), 44 us without turning.
template <typename T, int V, int F, int TURN>
__global__ void __launch_bounds__(256, TURN == kTurnHalf ? 5 : 1)
cache_write_kernel(CacheArgs a) {
    constexpr int P = V == 1 ? 1 : V / 2;
    extern __shared__ float2 turns[];            // [tokens of the block][rot / 2] cosine, sine
    __shared__ int lost[8];
    __shared__ int2 where[8];                    // page and place of a token's slot; page -1: nowhere
    grid_dependency_wait();
    const int G = a.group, group = threadIdx.x / G, lane = threadIdx.x % G;
    const uint32_t t = blockIdx.x * (256 / G) + group;
    const bool live = t < a.tokens;
    float2* turn = turns + group * (a.rot / 2);
    const int half = a.rot / 2;
    RawVec<T, V> own{}, other{};
    auto load = [&](const CacheUnit& c) {
        if (!c.in || !live) return;
        const CacheSide& side = c.key ? a.k : a.v;
        const T* x = reinterpret_cast<const T*>(side.x) + (int64_t)t * side.xt + c.h * side.xh + c.i;
        own = load_row<T, V>(x, a.wide);
        if (TURN != kNoTurn && c.key && c.i < a.rot) {
            if constexpr (TURN == kTurnHalf) other = load_row<T, V>(x + (c.i < half ? half : -half), a.wide);
            else if constexpr (V == 1) other = load_row<T, 1>(x + (c.i & 1 ? -1 : 1), false);
            else if constexpr (TURN == kTurnUneven) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int i = c.i + j;
                    if (i < a.rot) reinterpret_cast<T*>(&other)[j] = x[j + (a.half ? (i < half ? half : -half) : i & 1 ? -1 : 1)];
                }
            }
        }
    };
    CacheUnit c = cache_unit<V>(a, lane);
    load(c);
    if (lane == 0) {
        int2 w = make_int2(-1, 0);
        lost[group] = 0;
        if (live) {
            const int64_t slot = load_int(a.slots, a.slots_wide, t * a.islots);
            if (slot >= 1 && slot <= a.nslots) {
                const int64_t page = a.nslots < (int64_t)1 << 31 ? (int64_t)a.per_page.div((uint32_t)(slot - 1)) : (slot - 1) / a.page;
                w = make_int2((int)page, (int)(slot - 1 - page * a.page));
                if (a.owner && a.owner[slot - 1] != t + 1u) w.x = -1;
            } else if (slot != 0) {
                latch_error(a.err, B200_INVALID_ARG);
            }
        }
        where[group] = w;
    }
    if (G > 32) __syncthreads();
    else __syncwarp();
    const int2 w = where[group];
    if (w.x >= 0) {
        // of several tokens with one slot the last is kept, as if they were written in turn
        if (!a.owner && t + 1 < a.tokens) {
            const int64_t slot = load_int(a.slots, a.slots_wide, t * a.islots);
            for (int64_t j = t + 1 + lane; j < a.tokens; j += G)
                if (load_int(a.slots, a.slots_wide, j * a.islots) == slot) lost[group] = 1;
        }
        if constexpr (TURN != kNoTurn) {
            const uint64_t pos = (uint64_t)load_int(a.pos, a.pos_wide, t * a.ipos);
            for (int i = lane; i < half; i += G) {
                float s, cs;
                phase_sincos(pos * a.table[i], a.factor, s, cs);
                turn[turn_at<V, TURN>(i, half)] = make_float2(cs, s);
            }
        }
    }
    if (G > 32) __syncthreads();
    else __syncwarp();
    const bool write = w.x >= 0 && !lost[group];
    for (int base = 0;;) {
        const CacheSide& side = c.key ? a.k : a.v;
        F2 v[P], p[P];
        unpack_any<T, V>(own, v);
        if (TURN != kNoTurn && c.in && c.key && c.i < a.rot) {
            unpack_any<T, V>(other, p);
            if constexpr (TURN == kTurnUneven) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int i = c.i + j;
                    if (i >= a.rot) continue;
                    const bool first = a.half ? i < half : !(i & 1);
                    const float2 w = turn[a.half ? (first ? i : i - half) : i / 2];
                    float2 x = f2_parts(v[j / 2]);
                    const float2 y = f2_parts(p[j / 2]);
                    float& z = j & 1 ? x.y : x.x;
                    z = fmaf(z, w.x, (j & 1 ? y.y : y.x) * (first ? -w.y : w.y));
                    v[j / 2] = f2(x.x, x.y);
                }
            } else if constexpr (TURN == kTurnHalf) {
                const bool low = c.i < half;
                const float2* w = turn + (low ? c.i : c.i - half) / V;
                const int step = half / V;
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    const float2 w0 = w[2 * j * step], w1 = V == 1 ? w0 : w[(2 * j + 1) * step];
                    v[j] = f2_fma(v[j], f2(w0.x, w1.x), f2_mul(p[j], low ? f2(-w0.y, -w1.y) : f2(w0.y, w1.y)));
                }
            } else if constexpr (V == 1) {
                const float2 w = turn[c.i / 2], x = f2_parts(v[0]), y = f2_parts(p[0]);
                v[0] = f2(fmaf(x.x, w.x, (c.i & 1 ? y.x : -y.x) * w.y), 0.f);
            } else {
#pragma unroll
                for (int j = 0; j < P; ++j) {
                    const float2 w = turn[c.i / V + j * (half / P)], x = f2_parts(v[j]);
                    v[j] = f2_fma(v[j], f2(w.x), f2_mul(f2(x.y, x.x), f2(-w.y, w.y)));
                }
            }
        }
        const bool in = c.in && write;
        uint8_t* q = side.q + (int64_t)w.x * (int32_t)side.qn + (int64_t)w.y * (int32_t)side.qp + c.h * side.qh + c.i;
        uint32_t e;
        if constexpr (V == 1) {
            float x = c.in ? f2_parts(v[0]).x : 0.f;
            e = scale_byte(block_amax<1>(&x), F == kE4M3);
            if (in) *q = encode<1>(&x, e, F == kE4M3);
        } else {
            e = scale_byte(block_amax2<V>(v, c.in), F == kE4M3);
            if (in) *reinterpret_cast<RawVec<uint8_t, V>*>(q) = encode2<V>(v, e, F == kE4M3);
        }
        if (in && c.i % kBlock == 0)
            side.s[(int64_t)w.x * (int32_t)side.sn + (int64_t)w.y * (int32_t)side.sp + c.h * side.sh + c.i / kBlock] = (uint8_t)e;
        base += G;
        if (base >= a.k.units + a.v.units) break;
        c = cache_unit<V>(a, base + lane);
        own = other = RawVec<T, V>{};
        load(c);
    }
}

// A thread keeps its vector of a token - side, head and place are worked out once - and walks over the
// tokens of the block's tile, kReadUnroll at a time: their pages are looked up together, then their codes
// are loaded together.  Bound by HBM.  One B200, 8 contexts of up to 16384 tokens of 8 heads of 128, e4m3 to
// BFloat16: 80 us (6.0 TB/s of codes read and rows written), with a thread per vector and token 137 us.
constexpr int kReadUnroll = 4;

template <typename T, int V, int F>
__global__ void __launch_bounds__(256)
cache_read_kernel(CacheArgs a) {
    grid_dependency_wait();
    const int per_token = a.k.units + a.v.units;
    const int64_t cap = min(a.places, a.most * a.page);
    const int tile = (int)(blockIdx.x / a.parts), abreast = a.abreast;
    int u = (int)(blockIdx.x % a.parts) * 256 + threadIdx.x, t0 = 0;      // parts: of a token with more than 256 vectors
    if (a.parts == 1) { t0 = (int)a.per_token.div((uint32_t)u); u -= t0 * per_token; }
    const bool idle = u >= per_token;
    const bool key = u < a.k.units;
    if (!key) u -= a.k.units;
    const CacheSide& side = key ? a.k : a.v;
    const int h = idle ? 0 : (int)side.per_head.div((uint32_t)u);
    const int i = idle ? 0 : (u - h * (int)side.per_head.d) * V;
    const uint8_t *q = side.q + h * side.qh + i, *sc = side.s + h * side.sh + i / kBlock;
    const int32_t qn = (int32_t)side.qn, qp = (int32_t)side.qp, sn = (int32_t)side.sn, sp = (int32_t)side.sp, ol = (int32_t)side.ol;
    for (int64_t b = blockIdx.y; b < a.seqs; b += gridDim.y) {
        int64_t length = load_int(a.lengths, a.lengths_wide, b * a.ilengths);
        if (length < 0 || length > cap) {
            if (blockIdx.x == 0 && threadIdx.x == 0) latch_error(a.err, B200_INVALID_ARG);
            length = length < 0 ? 0 : cap;
        }
        const int first = tile * a.tile, last = (int)min((int64_t)first + a.tile, length);
        if (idle) continue;
        T* out = reinterpret_cast<T*>(side.out) + b * side.ob + h * side.oh + i;
        for (int l = first + t0; l < last; l += abreast * kReadUnroll) {
            int64_t page[kReadUnroll];
            int place[kReadUnroll];
#pragma unroll
            for (int k = 0; k < kReadUnroll; ++k) {
                const int lk = l + k * abreast;
                page[k] = -1;
                if (lk >= last) continue;
                const uint32_t pi = a.per_page.div((uint32_t)lk);
                place[k] = (int)((uint32_t)lk - pi * a.per_page.d);
                page[k] = load_int(a.pages, a.pages_wide, (int64_t)pi * a.pl + b * a.pb) - 1;
                if (page[k] < 0 || page[k] >= a.npages) { latch_error(a.err, B200_INVALID_ARG); page[k] = -1; }
            }
            RawVec<uint8_t, V> r[kReadUnroll];
            uint32_t e[kReadUnroll];
#pragma unroll
            for (int k = 0; k < kReadUnroll; ++k) {
                if (page[k] < 0) continue;
                const int32_t pg = (int32_t)page[k];
                e[k] = sc[(int64_t)pg * sn + (int64_t)place[k] * sp];
                r[k] = ld_raw<uint8_t, V>(q + (int64_t)pg * qn + (int64_t)place[k] * qp);
            }
#pragma unroll
            for (int k = 0; k < kReadUnroll; ++k) {
                if (page[k] < 0) continue;
                T* to = out + (int64_t)(l + k * abreast) * ol;
                if constexpr (V == 1) {
                    float v;
                    decode_as<T, 1>(r[k], e[k], F == kE4M3, &v);
                    st_raw<T, 1>(to, pack<T, 1>(&v));
                } else {
                    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r[k]);
                    RawVec<T, V> o;
                    uint32_t* po = reinterpret_cast<uint32_t*>(&o);
                    if (plain_scale<T>(e[k])) {
#pragma unroll
                        for (int j = 0; j < V / 4; ++j) {
                            F2 v[2];
                            decode2<4>(w[j], e[k], F == kE4M3, v);
                            *reinterpret_cast<RawVec<T, 4>*>(po + (int)sizeof(T) * j) = pack2<T, 4>(v);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < V / 4; ++j) {
                            float x[4];
                            decode_as<T, 4>(w[j], e[k], F == kE4M3, x);
                            *reinterpret_cast<RawVec<T, 4>*>(po + (int)sizeof(T) * j) = pack<T, 4>(x);
                        }
                    }
                    if constexpr (sizeof(T) * V == 32) st_raw32(to, o, a.wide);
                    else st_raw<T, V>(to, o);
                }
            }
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------
static int32_t cache_side(const b200_tensor* Q, const b200_tensor* S, const char* name, CacheSide* c) {
    B200_TRY(check_codes(Q, S, name));
    if (Q->ndim != 4) return fail(B200_INVALID_ARG, "%s: codes are (head size, heads, page size, pages)", name);
    if ((Q->shape[0] > 1 && Q->stride[0] != 1) || (S->shape[0] > 1 && S->stride[0] != 1))
        return fail(B200_UNSUPPORTED, "%s: the elements of a head must be neighbours", name);
    c->q = (uint8_t*)Q->ptr; c->s = (uint8_t*)S->ptr;
    c->d = (int32_t)Q->shape[0];
    c->qh = Q->stride[1]; c->qp = Q->stride[2]; c->qn = Q->stride[3];
    c->sh = S->stride[1]; c->sp = S->stride[2]; c->sn = S->stride[3];
    return B200_OK;
}
// The kernels take strides in 32 bits (and offsets in 64).
static bool far(int64_t stride) { return stride > 0x7fffffff || stride < -0x7fffffff; }
static int32_t cache_pair(const b200_tensor* KQ, const b200_tensor* KS, const b200_tensor* VQ, const b200_tensor* VS, CacheArgs* a) {
    B200_TRY(cache_side(KQ, KS, "cache keys", &a->k));
    B200_TRY(cache_side(VQ, VS, "cache values", &a->v));
    for (int k = 1; k < 4; ++k)
        if (KQ->shape[k] != VQ->shape[k]) return fail(B200_INVALID_ARG, "cache: keys and values differ in heads, page size or pages");
    if (KQ->dtype != VQ->dtype) return fail(B200_INVALID_ARG, "cache: keys and values differ in format");
    if (KQ->shape[0] > 8192 || VQ->shape[0] > 8192 || KQ->shape[1] > 65536 || KQ->shape[2] > 0x3fffffff)
        return fail(B200_TOO_LARGE, "cache: heads of at most 8192 elements, 65536 heads, pages of at most 2^30-1 places");
    for (const b200_tensor* t : {KQ, KS, VQ, VS})
        if (far(t->stride[2]) || far(t->stride[3])) return fail(B200_TOO_LARGE, "cache: pages more than 2^31 bytes apart");
    if (KQ->shape[3] > 0x7fffffff) return fail(B200_TOO_LARGE, "cache: at most 2^31-1 pages");
    a->heads = (int32_t)KQ->shape[1];
    a->page = (int32_t)KQ->shape[2];
    a->npages = KQ->shape[3];
    a->nslots = KQ->shape[2] * KQ->shape[3];
    a->e4m3 = KQ->dtype == B200_U8;
    return B200_OK;
}
static int32_t cache_rows(const b200_tensor* t, const b200_tensor* Q, int ndim, const char* name, int32_t* dtype) {
    B200_TRY(check_tensor(t, name));
    if (t->ndim != ndim || t->shape[0] != Q->shape[0] || t->shape[1] != Q->shape[1])
        return fail(B200_INVALID_ARG, "%s: differs in head size or heads from the cache", name);
    if (!is_row_type(t->dtype)) return fail(B200_UNSUPPORTED, "%s: Float16, BFloat16 or Float32", name);
    if (*dtype >= 0 && *dtype != t->dtype) return fail(B200_INVALID_ARG, "%s: keys and values differ in element type", name);
    if (t->shape[0] > 1 && t->stride[0] != 1) return fail(B200_UNSUPPORTED, "%s: the elements of a head must be neighbours", name);
    *dtype = t->dtype;
    return B200_OK;
}
static int32_t index_vector(const b200_tensor* t, const char* name, int64_t n, const void** p, int64_t* stride, int32_t* wide) {
    B200_TRY(check_tensor(t, name));
    if (!is_index_type(t->dtype)) return fail(B200_UNSUPPORTED, "%s: must be Int32 or Int64", name);
    if (t->ndim != 1 || t->shape[0] != n) return fail(B200_INVALID_ARG, "%s: needs %lld entries", name, (long long)n);
    *p = t->ptr; *stride = t->stride[0]; *wide = t->dtype == B200_I64;
    return B200_OK;
}
static bool multiple_strides(const b200_tensor* t, int64_t v, size_t bytes) {
    for (int k = 1; k < t->ndim; ++k) if (t->shape[k] > 1 && t->stride[k] % v) return false;
    return reinterpret_cast<uintptr_t>(t->ptr) % bytes == 0;
}
static int32_t no_overlap(const b200_tensor* t, const char* name) {
    if (tensor_numel(t) == 0) return B200_OK;
    for (int k = 1; k < t->ndim; ++k)
        if (t->shape[k] > 1 && t->stride[k] < t->shape[0] && t->stride[k] > -t->shape[0]) return fail(B200_INVALID_ARG, "%s: heads overlap", name);
    return B200_OK;
}

template <typename F>
static cudaError_t by_row_type(int32_t dtype, int v, F f) {
    auto width = [&](auto t) {
        constexpr int FV = 32 / (int)sizeof(t);
        return v == 1 ? f(t, std::integral_constant<int, 1>{}) : v == FV ? f(t, std::integral_constant<int, FV>{}) : f(t, std::integral_constant<int, FV / 2>{});
    };
    return dtype == B200_F16 ? width(__half{}) : dtype == B200_BF16 ? width(__nv_bfloat16{}) : width(float{});
}

}  // namespace b200

using namespace b200;

extern "C" int32_t b200_cache_write(b200_stream_t st, const b200_tensor* KQ, const b200_tensor* KS, const b200_tensor* VQ,
                                    const b200_tensor* VS, const b200_tensor* K, const b200_tensor* V, const b200_tensor* slots,
                                    const b200_tensor* positions, const b200_tensor* table, int32_t layout, double factor) {
    CacheArgs a{};
    B200_TRY(cache_pair(KQ, KS, VQ, VS, &a));
    for (const b200_tensor* t : {KQ, KS}) B200_TRY(no_overlap(t, "cache keys"));
    for (const b200_tensor* t : {VQ, VS}) B200_TRY(no_overlap(t, "cache values"));
    int32_t dtype = -1;
    B200_TRY(cache_rows(K, KQ, 3, "cache write keys", &dtype));
    B200_TRY(cache_rows(V, VQ, 3, "cache write values", &dtype));
    if (K->shape[2] != V->shape[2]) return fail(B200_INVALID_ARG, "cache write: keys and values differ in tokens");
    a.tokens = K->shape[2];
    B200_TRY(index_vector(slots, "cache write slots", a.tokens, &a.slots, &a.islots, &a.slots_wide));
    if ((positions != nullptr) != (table != nullptr)) return fail(B200_INVALID_ARG, "cache write: positions and their table belong together");
    if (table) {
        if (layout != kRotaryHalf && layout != kRotaryInterleaved) return fail(B200_UNSUPPORTED, "cache write: layout half (0) or interleaved (1)");
        B200_TRY(check_tensor(table, "rotary table"));
        if (table->dtype != B200_U64 || !tensor_is_contiguous(table)) return fail(B200_UNSUPPORTED, "cache write: the table must be dense UInt64");
        if (2 * tensor_numel(table) > K->shape[0]) return fail(B200_INVALID_ARG, "cache write: the table turns more elements than a head has");
        B200_TRY(index_vector(positions, "cache write positions", a.tokens, &a.pos, &a.ipos, &a.pos_wide));
        a.rot = (int32_t)(2 * tensor_numel(table));
        a.table = reinterpret_cast<const uint64_t*>(table->ptr);
        a.half = layout == kRotaryHalf;
        a.factor = (float)factor;
    }
    B200_TRY(enter(st));
    StreamGuard guard(st);
    if (a.tokens == 0 || a.heads == 0 || (a.k.d == 0 && a.v.d == 0)) return B200_OK;
    if (a.tokens > 0x7ffffff0) return fail(B200_TOO_LARGE, "cache write: at most 2^31-16 tokens");
    if (a.page == 0) a.page = 1;                                    // no slot is valid then
    a.k.x = K->ptr; a.k.xh = K->stride[1]; a.k.xt = K->stride[2];
    a.v.x = V->ptr; a.v.xh = V->stride[1]; a.v.xt = V->stride[2];
    a.err = device_error_word(st->dev);
    auto fits = [&](int w) {
        return a.k.d % w == 0 && a.v.d % w == 0 && multiple_strides(K, w, 16) && multiple_strides(V, w, 16) &&
               multiple_strides(KQ, w, (size_t)w) && multiple_strides(VQ, w, (size_t)w);
    };
    auto even = [&](int w) { return (a.half ? a.rot / 2 : a.rot) % w == 0; };
    const int full = dtype == B200_F32 ? 8 : 16;
    const int v = fits(full) && even(full) ? full : fits(full / 2) ? full / 2 : 1;
    const bool uneven = v > 1 && !even(v);
    a.wide = multiple_strides(K, full, 32) && multiple_strides(V, full, 32) && (!a.half || a.rot / 2 % full == 0);
    a.per_page = FastDiv((uint32_t)a.page);
    for (CacheSide* s : {&a.k, &a.v}) {
        const int per = (int)(row_blocks(s->d) * (kBlock / v));
        s->units = per * a.heads;
        s->per_head = FastDiv((uint32_t)per);
    }
    // few tokens: a thread per vector; many: four vectors to a thread, so that there are fewer to look at slots and
    // angles and a token mostly is one warp, with no barrier (32768 tokens of 8 heads of 128: 60 us, one
    // vector each 84)
    const int units = a.k.units + a.v.units, per_thread = a.tokens > kScanTokens ? 4 : 1;
    a.group = 32;
    auto angles = [&] { return (size_t)(256 / a.group) * (a.rot / 2) * sizeof(float2); };
    while (a.group < 256 && (a.group * per_thread < units || angles() > 32 * 1024)) a.group *= 2;
    const int per_block = 256 / a.group;
    void* temp = nullptr;
    if (a.tokens > kScanTokens && a.nslots > 0) {
        cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
        B200_CUDA(cudaStreamIsCapturing(st->s, &cap));
        void* p = nullptr;
        // a graph gets a table of its own (graphs captured on one stream may run side by side)
        if (cap == cudaStreamCaptureStatusNone) B200_TRY(scratch(st, (size_t)a.nslots * 4, &p));
        else { B200_TRY(b200_malloc_async(&temp, (size_t)a.nslots * 4, st)); p = temp; }
        a.owner = reinterpret_cast<uint32_t*>(p);
        B200_CUDA(launch_overlapped(cache_claim_kernel<true>, (unsigned)((a.tokens + 255) / 256), 256u, 0, st->s, a));
        B200_CUDA(launch_overlapped(cache_claim_kernel<false>, (unsigned)((a.tokens + 255) / 256), 256u, 0, st->s, a));
    }
    const size_t smem = angles();
    const unsigned grid = (unsigned)((a.tokens + per_block - 1) / per_block);
    B200_CUDA(by_row_type(dtype, v, [&](auto t, auto w) {
        using T = decltype(t);
        constexpr int W = decltype(w)::value;
        auto turn = [&](auto f) {
            constexpr int F = decltype(f)::value;
            if constexpr (W == 16 / (int)sizeof(T)) {
                if (uneven) return launch_overlapped(cache_write_kernel<T, W, F, kTurnUneven>, grid, 256u, smem, st->s, a);
            }
            return a.rot == 0 ? launch_overlapped(cache_write_kernel<T, W, F, kNoTurn>, grid, 256u, smem, st->s, a)
                   : a.half   ? launch_overlapped(cache_write_kernel<T, W, F, kTurnHalf>, grid, 256u, smem, st->s, a)
                              : launch_overlapped(cache_write_kernel<T, W, F, kTurnInterleaved>, grid, 256u, smem, st->s, a);
        };
        return a.e4m3 ? turn(std::integral_constant<int, kE4M3>{}) : turn(std::integral_constant<int, kInt8>{});
    }));
    if (temp) B200_TRY(b200_free_async(temp, st));
    return finish(st, "b200_cache_write");
}

extern "C" int32_t b200_cache_read(b200_stream_t st, const b200_tensor* K, const b200_tensor* V, const b200_tensor* KQ, const b200_tensor* KS,
                                   const b200_tensor* VQ, const b200_tensor* VS, const b200_tensor* pages, const b200_tensor* lengths) {
    CacheArgs a{};
    B200_TRY(cache_pair(KQ, KS, VQ, VS, &a));
    int32_t dtype = -1;
    B200_TRY(cache_rows(K, KQ, 4, "cache read keys", &dtype));
    B200_TRY(cache_rows(V, VQ, 4, "cache read values", &dtype));
    B200_TRY(no_overlap(K, "cache read keys"));
    B200_TRY(no_overlap(V, "cache read values"));
    if (K->shape[2] != V->shape[2] || K->shape[3] != V->shape[3]) return fail(B200_INVALID_ARG, "cache read: keys and values differ in places or sequences");
    a.places = K->shape[2];
    a.seqs = K->shape[3];
    if (far(K->stride[2]) || far(V->stride[2]) || a.places > 0x3fffffff)
        return fail(B200_TOO_LARGE, "cache read: at most 2^30 places, tokens at most 2^31 elements apart");
    B200_TRY(check_tensor(pages, "cache read pages"));
    if (!is_index_type(pages->dtype)) return fail(B200_UNSUPPORTED, "cache read: pages must be Int32 or Int64");
    if (pages->ndim != 2 || pages->shape[1] != a.seqs) return fail(B200_INVALID_ARG, "cache read: the page table is (pages of a sequence, sequences)");
    a.pages = pages->ptr; a.pl = pages->stride[0]; a.pb = pages->stride[1]; a.most = pages->shape[0]; a.pages_wide = pages->dtype == B200_I64;
    B200_TRY(index_vector(lengths, "cache read lengths", a.seqs, &a.lengths, &a.ilengths, &a.lengths_wide));
    B200_TRY(enter(st));
    StreamGuard guard(st);
    if (a.seqs == 0 || a.heads == 0 || (a.k.d == 0 && a.v.d == 0)) return B200_OK;
    if (a.page == 0) { a.page = 1; a.most = 0; }                    // no place holds a token
    a.k.out = K->ptr; a.k.oh = K->stride[1]; a.k.ol = K->stride[2]; a.k.ob = K->stride[3];
    a.v.out = V->ptr; a.v.oh = V->stride[1]; a.v.ol = V->stride[2]; a.v.ob = V->stride[3];
    a.err = device_error_word(st->dev);
    auto fits = [&](int w) {
        return a.k.d % w == 0 && a.v.d % w == 0 && multiple_strides(K, w, 16) && multiple_strides(V, w, 16) &&
               multiple_strides(KQ, w, (size_t)w) && multiple_strides(VQ, w, (size_t)w);
    };
    const int full = dtype == B200_F32 ? 8 : 16, v = fits(full) ? full : fits(full / 2) ? full / 2 : 1;
    a.wide = multiple_strides(K, full, 32) && multiple_strides(V, full, 32);
    a.per_page = FastDiv((uint32_t)a.page);
    for (CacheSide* s : {&a.k, &a.v}) {
        s->units = s->d / v * a.heads;
        s->per_head = FastDiv((uint32_t)(s->d / v));
    }
    const int per_token = a.k.units + a.v.units;
    a.per_token = FastDiv((uint32_t)per_token);
    a.parts = (per_token + 255) / 256;
    a.abreast = a.parts > 1 ? 1 : 256 / per_token;
    a.tile = a.abreast * kReadUnroll * 2;
    int64_t bx = (a.places + a.tile - 1) / a.tile * a.parts;
    if (bx < 1) bx = 1;                                             // one block at least looks at the lengths
    if (bx > 0x7fffffff) return fail(B200_TOO_LARGE, "cache read: too many places for one call");
    const dim3 grid((unsigned)bx, (unsigned)(a.seqs < 65535 ? a.seqs : 65535));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)(a.parts > 1 ? 256 : a.abreast * per_token));
    cfg.stream = st->s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = overlap_launches_enabled() ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    B200_CUDA(by_row_type(dtype, v, [&](auto t, auto w) {
        using T = decltype(t);
        constexpr int W = decltype(w)::value;
        return a.e4m3 ? cudaLaunchKernelEx(&cfg, cache_read_kernel<T, W, kE4M3>, a) : cudaLaunchKernelEx(&cfg, cache_read_kernel<T, W, kInt8>, a);
    }));
    return finish(st, "b200_cache_read");
}
