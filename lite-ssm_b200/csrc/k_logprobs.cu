// k_logprobs.cu — log probabilities of given tokens, entropy and top alternatives of rows of
// logits, and their gradient.
//
//   m = max_j x_j, s = sum_j e^(x_j - m), u = sum_j e^(x_j - m) (x_j - m)
//   lse = m + log s     logp = (x_t - m) - log s     entropy = log s - u / s
//   top: the K largest x_j, of equal ones the lower index first, as (x_j - m) - log s
//   d(logp)/dx_j = [j = t] - p_j     d(entropy)/dx_j = -p_j (log p_j + entropy)
//
// An entry of -inf has p = 0 and no share of the entropy. A row that holds nothing but -inf has
// lse = logp = top values = -inf, entropy 0 and gradient 0. A NaN or +inf entry makes every
// value of its row NaN (the ids rank NaN as -inf).
#include <cooperative_groups.h>

#include "device_util.cuh"
#include "lssm_internal.h"

namespace lssm {

namespace cg = cooperative_groups;

namespace {

constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32;
constexpr int LP_GROUP = 4;          // 16-byte loads a thread has in flight
constexpr int LP_CAND = 1024;        // candidates for the top entries that a CTA holds
constexpr int LP_CLUSTER_MAX = 8;
constexpr uint32_t FULL = 0xffffffffu;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
// An element's exponential is taken against a reference that follows the thread's running maximum,
// but only in steps of at least this much: the sums then hold at most 2^(1.44 * 8) times as much.
constexpr float REF_STEP = 8.0f;

// Orders values as whole numbers: NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t order_key(float v) {
    v = v != v ? -INFINITY : v + 0.0f;
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
// Larger value first, of equal ones the lower index: no two indices have the same.
__device__ __forceinline__ uint64_t rank_key(uint32_t key, uint32_t i) { return (uint64_t)key << 32 | (~i); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// Two fp32 lanes in one instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    return (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// A row as 16-byte chunks at 16-byte addresses; chunk 0 may begin before the row and the last
// chunk end behind it: those elements are not read and stand for -inf.
template <typename T>
struct Row {
    static constexpr int VEC = 16 / sizeof(T);
    const T* x;              // element 0
    int32_t lead;            // elements of chunk 0 before element 0
    uint32_t V, chunks;

    __device__ Row(const void* logits, uint64_t first, uint32_t vocab) {
        x = static_cast<const T*>(logits) + first;
        lead = (int32_t)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
        V = vocab;
        chunks = (uint32_t)(((uint64_t)vocab + lead + VEC - 1) / VEC);
    }
    __device__ __forceinline__ int64_t index(uint32_t c) const { return (int64_t)c * VEC - lead; }
    static __device__ __forceinline__ T lowest() {
        if constexpr (sizeof(T) == 4) return -INFINITY;
        else { const uint16_t b = std::is_same<T, __half>::value ? 0xFC00 : 0xFF80; T v; memcpy(&v, &b, 2); return v; }
    }
    __device__ __forceinline__ uint4 chunk(uint32_t c) const {
        const int64_t e = index(c);
        uint4 r;
        if (e >= 0 && e + VEC <= (int64_t)V) {
            r = __ldg(reinterpret_cast<const uint4*>(x + e));
        } else {
            T t[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) t[i] = e + i >= 0 && e + i < (int64_t)V ? x[e + i] : lowest();
            memcpy(&r, t, 16);
        }
        return r;
    }
    static __device__ __forceinline__ uint4 nothing() {
        T t[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) t[i] = lowest();
        uint4 r;
        memcpy(&r, t, 16);
        return r;
    }
};

__device__ __forceinline__ float2 to_float2(uint32_t w, __half) {
    __half2 h;
    memcpy(&h, &w, 4);
    return __half22float2(h);
}
__device__ __forceinline__ float2 to_float2(uint32_t w, __nv_bfloat16) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

// The largest of a chunk's elements; a NaN counts only where there is nothing else.
__device__ __forceinline__ float chunk_max(uint4 c, __half) {
    __half2 h[4];
    memcpy(h, &c, 16);
    const float2 f = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(f.x, f.y);
}
__device__ __forceinline__ float chunk_max(uint4 c, __nv_bfloat16) {
    __nv_bfloat162 h[4];
    memcpy(h, &c, 16);
    const float2 f = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(f.x, f.y);
}
__device__ __forceinline__ float chunk_max(uint4 c, float) {
    return fmaxf(fmaxf(__uint_as_float(c.x), __uint_as_float(c.y)), fmaxf(__uint_as_float(c.z), __uint_as_float(c.w)));
}
template <typename T>
__device__ __forceinline__ void chunk_values(uint4 c, float (&v)[16 / sizeof(T)]) {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(w[i]);
        else { const float2 f = to_float2(w[i], T()); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
    }
}

// Running sums of one thread: with z = (x - ref) log2 e, s = sum 2^z and u = sum 2^z z, two lanes
// each. For fp16, whose range allows it, z is one fma against refL = ref log2 e as rounded; `slip`
// gives back what that rounding moved.
template <typename T>
struct Sums {
    float ref = -INFINITY, refL = 0.0f;
    uint64_t s2 = 0, u2 = 0;

    __device__ __forceinline__ float slip() const {
        return std::is_same<T, __half>::value && ref > -INFINITY ? fmaf(-ref, LOG2E, refL) : 0.0f;
    }
    // The same sums against another reference: every exponent grows by d.
    static __device__ __forceinline__ void shift(float d, float& s, float& u) {
        const float f = ex2(d);
        u = f > 0.0f ? f * fmaf(s, d, u) : 0.0f;
        s = f * s;
    }
    __device__ __forceinline__ void follow(float gm) {
        if (!(gm > ref + REF_STEP)) return;
        float2 s = unpack2(s2), u = unpack2(u2);
        if (ref > -INFINITY) {
            const float newL = gm * LOG2E;
            const float d = std::is_same<T, __half>::value ? refL - newL : (ref - gm) * LOG2E;
            shift(d, s.x, u.x);
            shift(d, s.y, u.y);
        }
        ref = gm;
        refL = gm * LOG2E;
        s2 = pack2(s.x, s.y);
        u2 = pack2(u.x, u.y);
    }
    __device__ __forceinline__ void add(float z0, float z1) {
        const uint64_t e = pack2(ex2(z0), ex2(z1));
        s2 = add2(s2, e);
        u2 = fma2(e, pack2(z0, z1), u2);
    }
    __device__ __forceinline__ void chunk(uint4 c) {
        const uint32_t w[4] = {c.x, c.y, c.z, c.w};
        if constexpr (std::is_same<T, __half>::value) {
            const uint64_t l2 = pack2(LOG2E, LOG2E), r2 = pack2(-refL, -refL);
            if (ref > -60000.0f) {
                // -inf becomes the lowest finite value: its exponential is 0 too, but times z it is 0, not NaN
                const __half2 low = __half2half2(__ushort_as_half(0xFBFF));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    __half2 h;
                    memcpy(&h, &w[i], 4);
                    const float2 f = __half22float2(__hmax2_nan(h, low));
                    const float2 z = unpack2(fma2(pack2(f.x, f.y), l2, r2));
                    add(z.x, z.y);
                }
            } else {
                // nothing but -inf and values near the lowest so far: they have to be told apart
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = to_float2(w[i], T());
                    const float2 z = unpack2(fma2(pack2(f.x, f.y), l2, r2));
                    add(max_or_nan(z.x, -300.0f), max_or_nan(z.y, -300.0f));
                }
            }
        } else {
            const float r = ref > -INFINITY ? ref : 0.0f;
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int i = 0; i < 4; i += 2)
                    add(max_or_nan((__uint_as_float(w[i]) - r) * LOG2E, -300.0f),
                        max_or_nan((__uint_as_float(w[i + 1]) - r) * LOG2E, -300.0f));
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = to_float2(w[i], T());
                    add(max_or_nan((f.x - r) * LOG2E, -300.0f), max_or_nan((f.y - r) * LOG2E, -300.0f));
                }
            }
        }
    }
};

struct LpShared {
    uint64_t cand[LP_CAND + LSSM_TOP_K_MAX];
    uint64_t list[LSSM_TOP_K_MAX];                    // the CTA's top entries, in order (0: none)
    uint64_t all[LP_CLUSTER_MAX * LSSM_TOP_K_MAX];    // the cluster's (first CTA)
    float m, s, u;                                    // the CTA's sums against its maximum
    float red[3][LP_WARPS];
    uint32_t maxima[LP_WARPS * 4];
    uint32_t count, nsel, wsum[LP_WARPS];
    uint8_t sel[LP_THREADS];
};

// The CTA's largest K entries of chunks [c0, c1) into sh.list. `tkey`: this thread's largest (order_key).
//
// A value that at least K entries reach: the K-th largest of the four largest thread maxima of
// every warp. Only threads whose maximum reaches it can hold one of the top K, so only their chunks
// (about K / 256 of the slice, still in L2) are read again. The entries that reach the bound are
// counted, stored and ranked against one another by value and index.
template <typename T>
__device__ void cta_top(const Row<T>& row, uint32_t c0, uint32_t c1, uint32_t tkey, uint32_t K, LpShared& sh) {
    constexpr int VEC = 16 / sizeof(T);
    const uint32_t tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    uint32_t mine = tkey;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const uint32_t top = __reduce_max_sync(FULL, mine);
        if (lane == 0) sh.maxima[wid * 4 + r] = top;
        if ((int)lane == __ffs(__ballot_sync(FULL, mine == top)) - 1) mine = 0;
    }
    if (tid == 0) { sh.count = 0; sh.nsel = 0; }
    if (tid < LSSM_TOP_K_MAX) sh.list[tid] = 0;
    __syncthreads();
    // the K-th largest of the 32: the one with K - 1 before it
    const uint32_t v = sh.maxima[lane];
    uint32_t before = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const uint32_t o = sh.maxima[i];
        before += o > v || (o == v && i < (int)lane);
    }
    const uint32_t bound = __shfl_sync(FULL, v, __ffs(__ballot_sync(FULL, before == K - 1)) - 1);
    const bool chosen = tkey >= bound;
    const uint32_t votes = __ballot_sync(FULL, chosen);
    uint32_t at = 0;
    if (lane == 0 && votes) at = atomicAdd(&sh.nsel, __popc(votes));
    at = __shfl_sync(FULL, at, 0) + __popc(votes & ((1u << lane) - 1));
    if (chosen) sh.sel[at] = (uint8_t)tid;
    __syncthreads();
    const uint32_t per = (c1 - c0 + LP_THREADS - 1) / LP_THREADS, items = sh.nsel * per;
    const float bv = key_value(bound);
    auto collect = [&](bool ties) {
        for (uint32_t q = tid; q < items; q += LP_THREADS) {
            const uint32_t c = c0 + sh.sel[q / per] + (q % per) * LP_THREADS;
            if (c >= c1) continue;
            const uint4 raw = row.chunk(c);
            const float cm = chunk_max(raw, T());
            if (ties ? cm < bv : !(cm > bv)) continue;
            float x[VEC];
            chunk_values<T>(raw, x);
            const int64_t e = row.index(c);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const uint32_t k = order_key(x[i]);
                if (k < bound || (k == bound && !ties) || e + i < 0 || e + i >= (int64_t)row.V) continue;
                const uint32_t p = atomicAdd(&sh.count, 1u);
                if (p < LP_CAND) sh.cand[p] = rank_key(k, (uint32_t)(e + i));
            }
        }
    };
    const bool level = sh.nsel > LP_THREADS / 4;   // many threads reach the bound: a masked or constant row
    if (!level) collect(true);
    __syncthreads();
    uint32_t n = sh.count;
    if (level || n > LP_CAND) {
        // Many equal to the bound (masked or constant rows): those above it first, then of the
        // equal ones as many as are missing, in the order of their index.
        __syncthreads();
        if (tid == 0) sh.count = 0;
        __syncthreads();
        collect(false);
        __syncthreads();
        n = sh.count;
        if (n <= LP_CAND) {
            uint32_t have = n;
            for (uint32_t c = c0; c < c1 && have < K; c += LP_THREADS) {
                const uint32_t mc = c + tid;
                uint32_t hit = 0;
                int64_t e = 0;
                if (mc < c1) {
                    float x[VEC];
                    chunk_values<T>(row.chunk(mc), x);
                    e = row.index(mc);
#pragma unroll
                    for (int i = 0; i < VEC; ++i)
                        if (order_key(x[i]) == bound && e + i >= 0 && e + i < (int64_t)row.V) hit |= 1u << i;
                }
                const uint32_t cnt = __popc(hit);
                uint32_t inc = cnt;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t w = __shfl_up_sync(FULL, inc, o);
                    if ((int)lane >= o) inc += w;
                }
                if (lane == 31) sh.wsum[wid] = inc;
                __syncthreads();
                uint32_t pos = have + inc - cnt, total = 0;
                for (int w = 0; w < LP_WARPS; ++w) {
                    if (w < (int)wid) pos += sh.wsum[w];
                    total += sh.wsum[w];
                }
                for (; hit && pos < K; hit &= hit - 1, ++pos)
                    sh.cand[pos] = rank_key(bound, (uint32_t)(e + __ffs(hit) - 1));
                have = have + total < K ? have + total : K;
                __syncthreads();
            }
            n = have;
        } else {
            // More entries above the bound than there is room for (a pattern that puts the large ones
            // into a few threads' chunks): one entry after the other.
            uint64_t last = ~0ull;
            for (uint32_t k = 0; k < K; ++k) {
                uint64_t best = 0;
                for (uint32_t c = c0 + tid; c < c1; c += LP_THREADS) {
                    float x[VEC];
                    chunk_values<T>(row.chunk(c), x);
                    const int64_t e = row.index(c);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const uint64_t r = rank_key(order_key(x[i]), (uint32_t)(e + i));
                        if (e + i >= 0 && e + i < (int64_t)row.V && r < last && r > best) best = r;
                    }
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const uint64_t w = __shfl_xor_sync(FULL, best, o);
                    best = w > best ? w : best;
                }
                __syncthreads();
                if (lane == 0) sh.all[wid] = best;
                __syncthreads();
                last = sh.all[0];
                for (int w = 1; w < LP_WARPS; ++w) last = sh.all[w] > last ? sh.all[w] : last;
                if (tid == 0) sh.cand[k] = last;
            }
            n = K;
        }
        __syncthreads();
    }
    for (uint32_t i = tid; i < n; i += LP_THREADS) {
        const uint64_t k = sh.cand[i];
        uint32_t r = 0;
        for (uint32_t j = 0; j < n; ++j) r += sh.cand[j] > k;
        if (r < K) sh.list[r] = k;
    }
}

// One CTA, or a cluster of them over slices of the vocabulary, per row; one pass over the logits.
template <typename T>
__global__ void __launch_bounds__(LP_THREADS) k_logprobs(LogprobsArgs a, uint32_t nc) {
    __shared__ LpShared sh;
    const uint32_t tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const uint32_t r = blockIdx.x / nc, part = blockIdx.x % nc;
    const Row<T> row(a.logits, (uint64_t)r * a.row_stride, a.vocab);
    const uint32_t per = (row.chunks + nc - 1) / nc;
    const uint32_t c0 = min(row.chunks, part * per), c1 = min(row.chunks, c0 + per);
    uint32_t target = LSSM_NO_TOKEN;
    float xt = 0.0f;
    if (part == 0 && tid == 0 && a.logp) {
        target = a.targets[r];
        if (target < a.vocab) xt = load_any(row.x, target, a.dtype);
    }
    Sums<T> sum;
    float tmax = -INFINITY;
    auto group = [&](const uint4 (&w)[LP_GROUP]) {
        float gm = chunk_max(w[0], T());
#pragma unroll
        for (int g = 1; g < LP_GROUP; ++g) gm = fmaxf(gm, chunk_max(w[g], T()));
        tmax = fmaxf(tmax, gm);
        sum.follow(gm);
#pragma unroll
        for (int g = 0; g < LP_GROUP; ++g) sum.chunk(w[g]);
    };
    // whole groups of whole chunks first: chunks [inner, outer) lie inside the row
    const uint32_t inner = max(c0, row.lead ? 1u : 0u), outer = min(c1, (row.V + row.lead) / Row<T>::VEC);
    constexpr uint32_t STRIDE = LP_THREADS * LP_GROUP;
    uint32_t c = c0 + tid;
    if (c < inner) {
        const uint4 w[LP_GROUP] = {row.chunk(c), Row<T>::nothing(), Row<T>::nothing(), Row<T>::nothing()};
        group(w);
        c += LP_THREADS;
    }
    const uint4* at = reinterpret_cast<const uint4*>(row.x - row.lead) + c;
    for (; c + 3 * LP_THREADS < outer; c += STRIDE, at += STRIDE) {
        uint4 w[LP_GROUP];
#pragma unroll
        for (int g = 0; g < LP_GROUP; ++g) w[g] = __ldg(at + g * LP_THREADS);
        group(w);
    }
    if (c < c1) {
        uint4 w[LP_GROUP];
#pragma unroll
        for (int g = 0; g < LP_GROUP; ++g)
            w[g] = c + g * LP_THREADS < c1 ? row.chunk(c + g * LP_THREADS) : Row<T>::nothing();
        group(w);
    }
    // the CTA's sums against its maximum
    float m = warp_max(tmax);
    if (lane == 0) sh.red[0][wid] = m;
    __syncthreads();
    m = sh.red[0][0];
#pragma unroll
    for (int w = 1; w < LP_WARPS; ++w) m = fmaxf(m, sh.red[0][w]);
    float2 s2 = unpack2(sum.s2), u2 = unpack2(sum.u2);
    float s = s2.x + s2.y, u = u2.x + u2.y;
    if (sum.ref > -INFINITY && m < INFINITY) Sums<T>::shift((sum.ref - m) * LOG2E + sum.slip(), s, u);
    s = warp_sum(s);
    u = warp_sum(u);
    __syncthreads();
    if (lane == 0) { sh.red[1][wid] = s; sh.red[2][wid] = u; }
    if (a.top_k) cta_top(row, c0, c1, order_key(tmax), a.top_k, sh);
    __syncthreads();
    s = u = 0.0f;
#pragma unroll
    for (int w = 0; w < LP_WARPS; ++w) { s += sh.red[1][w]; u += sh.red[2][w]; }
    const uint32_t K = a.top_k;
    const uint64_t* lists = sh.list;
    if (nc > 1) {
        // the slices' sums and lists meet in the first CTA of the cluster
        cg::cluster_group cl = cg::this_cluster();
        if (tid == 0) { sh.m = m; sh.s = s; sh.u = u; }
        cl.sync();
        if (part == 0) {
            float mm = m;
            for (uint32_t p = 1; p < nc; ++p) mm = fmaxf(mm, *cl.map_shared_rank(&sh.m, p));
            float ss = 0.0f, uu = 0.0f;
            for (uint32_t p = 0; p < nc; ++p) {
                const float pm = *cl.map_shared_rank(&sh.m, p);
                float ps = *cl.map_shared_rank(&sh.s, p), pu = *cl.map_shared_rank(&sh.u, p);
                if (pm > -INFINITY && mm < INFINITY) Sums<T>::shift((pm - mm) * LOG2E, ps, pu);
                ss += ps;
                uu += pu;
            }
            m = mm; s = ss; u = uu;
            for (uint32_t i = tid; i < nc * K; i += LP_THREADS) sh.all[i] = *cl.map_shared_rank(&sh.list[i % K], i / K);
        }
        cl.sync();
        if (part != 0) return;
        lists = sh.all;
    }
    const bool none = m == -INFINITY && !(s != s);
    const float ls = m == INFINITY ? __int_as_float(0x7FC00000) : logf(s);
    if (tid == 0) {
        if (a.lse) a.lse[r] = none ? -INFINITY : m + ls;
        if (a.entropy) a.entropy[r] = none ? 0.0f : ls - LN2 * (u / s);
        if (a.logp) {
            float v = 0.0f;
            if (target != LSSM_NO_TOKEN)
                v = target >= a.vocab ? __int_as_float(0x7FC00000) : none ? -INFINITY : (xt - m) - ls;
            a.logp[r] = v;
        }
    }
    for (uint32_t i = tid; i < nc * K; i += LP_THREADS) {
        const uint64_t k = lists[i];
        if (!k) continue;
        // its place: the entries before it in its own list and in every other (each in order)
        uint32_t place = i % K;
        for (uint32_t p = 0; p < nc && place < K; ++p) {
            if (p == i / K) continue;
            uint32_t lo = 0, hi = K;
            while (lo < hi) {
                const uint32_t mid = (lo + hi) / 2;
                if (lists[p * K + mid] > k) lo = mid + 1; else hi = mid;
            }
            place += lo;
        }
        if (place < K) {
            a.top_ids[(uint64_t)r * K + place] = ~(uint32_t)k;
            a.top_logp[(uint64_t)r * K + place] = none ? -INFINITY : (key_value((uint32_t)(k >> 32)) - m) - ls;
        }
    }
}

__global__ void __launch_bounds__(LP_THREADS) k_logprobs_grad(LogprobsGradArgs a) {
    const uint32_t r = blockIdx.x, V = a.vocab;
    const uint64_t xb = (uint64_t)r * a.row_stride, gb = (uint64_t)r * a.grad_stride;
    const float lse = a.lse[r], H = a.g_entropy ? a.entropy[r] : 0.0f;
    const uint32_t t = a.targets ? a.targets[r] : LSSM_NO_TOKEN;
    const bool none = lse == -INFINITY, given = t != LSSM_NO_TOKEN;
    float g = a.g_logp && given ? a.g_logp[r] : 0.0f;
    const float h = a.g_entropy ? a.g_entropy[r] : 0.0f;
    if (given && t >= V) g = __int_as_float(0x7FC00000);
    for (uint32_t i = threadIdx.x; i < V; i += LP_THREADS) {
        float d = 0.0f;
        if (!none) {
            const float lp = load_any(a.logits, xb + i, a.dtype) - lse, p = expf(lp);
            d = (i == t ? g : 0.0f) - g * p;
            if (a.g_entropy && p != 0.0f) d -= h * p * (lp + H);
        }
        store_any(a.dlogits, gb + i, a.grad_dtype, d);
    }
}

}  // namespace

cudaError_t launch_logprobs(const LogprobsArgs& a, cudaStream_t s) {
    if (!a.rows) return cudaSuccess;
    // Few rows: a cluster of CTAs a row, until every SM has two CTAs or a thread less than one chunk.
    uint32_t nc = 1;
    while (nc < LP_CLUSTER_MAX && (uint64_t)a.rows * nc < 296 && a.vocab / (8 * LP_THREADS * nc) >= 1) nc *= 2;
    if ((uint64_t)a.rows * nc > 0x7FFFFFFFull) nc = 1;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {nc, 1, 1};
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = {a.rows * nc, 1, 1};
    cfg.blockDim = {LP_THREADS, 1, 1};
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaError_t e;
    if (a.dtype == LSSM_DT_F16) e = cudaLaunchKernelEx(&cfg, k_logprobs<__half>, a, nc);
    else if (a.dtype == LSSM_DT_BF16) e = cudaLaunchKernelEx(&cfg, k_logprobs<__nv_bfloat16>, a, nc);
    else e = cudaLaunchKernelEx(&cfg, k_logprobs<float>, a, nc);
    if (e != cudaSuccess) return e;
    return cudaGetLastError();
}

cudaError_t launch_logprobs_grad(const LogprobsGradArgs& a, cudaStream_t s) {
    if (!a.rows) return cudaSuccess;
    k_logprobs_grad<<<a.rows, LP_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace lssm
