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

constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32, LP_TOPS = 32 / LP_WARPS;
constexpr int LP_AHEAD = 2048;       // 16-byte chunks of a later row that a CTA asks L2 for
constexpr int LP_GROUP = 4;          // 16-byte loads that a thread has on their way while it works on as many
constexpr int LP_CTAS = 4;           // CTAs an SM holds
constexpr int LP_CAND = 1024;        // candidates for the top entries that a CTA holds
constexpr int LP_HITS = 256;         // chunks that may hold one
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
// Two fp32 lanes in one instruction, as the two halves of a 64-bit register.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
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
    // Chunks [inner, outer) lie inside the row.
    __device__ __forceinline__ uint32_t inner() const { return lead ? 1u : 0u; }
    __device__ __forceinline__ uint32_t outer() const { return (V + lead) / VEC; }
    __device__ __forceinline__ const uint4* base() const { return reinterpret_cast<const uint4*>(x - lead); }
    __device__ __forceinline__ int64_t index(uint32_t c) const { return (int64_t)c * VEC - lead; }
    static __device__ __forceinline__ T lowest() {
        if constexpr (sizeof(T) == 4) return -INFINITY;
        else { const uint16_t b = std::is_same<T, __half>::value ? 0xFC00 : 0xFF80; T v; memcpy(&v, &b, 2); return v; }
    }
    __device__ __forceinline__ uint4 chunk(uint32_t c) const {
        uint4 r;
        if (c >= inner() && c < outer()) {
            r = __ldg(base() + c);
        } else {
            const int64_t e = index(c);
            T t[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) t[i] = e + i >= 0 && e + i < (int64_t)V ? x[e + i] : lowest();
            memcpy(&r, t, 16);
        }
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

// The largest element of n chunks; a NaN counts only where there is nothing else.
template <typename T, int n>
__device__ __forceinline__ float chunks_max(const uint4 (&c)[n]) {
    if constexpr (sizeof(T) == 4) {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < n; ++i)
            m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(c[i].x), __uint_as_float(c[i].y)),
                               fmaxf(__uint_as_float(c[i].z), __uint_as_float(c[i].w))));
        return m;
    } else {
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        T2 h[4 * n];
        memcpy(h, c, sizeof(h));
#pragma unroll
        for (int w = 2 * n; w; w /= 2)
#pragma unroll
            for (int i = 0; i < w; ++i) h[i] = __hmax2(h[i], h[i + w]);
        uint32_t b;
        memcpy(&b, &h[0], 4);
        const float2 f = to_float2(b, T());
        return fmaxf(f.x, f.y);
    }
}
template <typename T>
__device__ __forceinline__ float chunk_max(uint4 c, T) {
    const uint4 one[1] = {c};
    return chunks_max<T, 1>(one);
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

__device__ __forceinline__ float load_one(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float load_one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_one(const float* p) { return *p; }

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
    __device__ __forceinline__ void add(uint64_t z) {
        const float2 f = unpack2(z);
        const uint64_t e = pack2(ex2(f.x), ex2(f.y));
        s2 = add2(s2, e);
        u2 = fma2(e, z, u2);
    }
    // n chunks whose largest element is gm
    template <int n>
    __device__ __forceinline__ void chunks(const uint4 (&c)[n], float gm) {
        follow(gm);
        uint32_t w[4 * n];
        memcpy(w, c, sizeof(w));
        if constexpr (std::is_same<T, __half>::value) {
            const uint64_t l2 = pack2(LOG2E, LOG2E), r2 = pack2(-refL, -refL);
            if (ref > -60000.0f) {
                // -inf becomes the lowest finite value: its exponential is 0 too, but times z it is 0, not NaN
                const __half2 low = __half2half2(__ushort_as_half(0xFBFF));
#pragma unroll
                for (int i = 0; i < 4 * n; ++i) {
                    __half2 h;
                    memcpy(&h, &w[i], 4);
                    const float2 f = __half22float2(__hmax2_nan(h, low));
                    add(fma2(pack2(f.x, f.y), l2, r2));
                }
            } else {
                // nothing but -inf and values near the lowest so far: they have to be told apart
#pragma unroll
                for (int i = 0; i < 4 * n; ++i) {
                    const float2 f = to_float2(w[i], T());
                    const float2 z = unpack2(fma2(pack2(f.x, f.y), l2, r2));
                    add(pack2(max_or_nan(z.x, -300.0f), max_or_nan(z.y, -300.0f)));
                }
            }
        } else {
            const float r = ref > -INFINITY ? ref : 0.0f;
            const uint64_t l2 = pack2(LOG2E, LOG2E), zero = pack2(-0.0f, -0.0f), r2 = pack2(-r, -r);
#pragma unroll
            for (int i = 0; i < 4 * n; i += sizeof(T) / 2) {
                float2 f;
                if constexpr (sizeof(T) == 4) f = make_float2(__uint_as_float(w[i]), __uint_as_float(w[i + 1]));
                else f = to_float2(w[i], T());
                const float2 z = unpack2(fma2(add2(pack2(f.x, f.y), r2), l2, zero));
                add(pack2(max_or_nan(z.x, -300.0f), max_or_nan(z.y, -300.0f)));
            }
        }
    }
};

struct LpShared {
    uint64_t cand[LP_CAND + LSSM_TOP_K_MAX];
    uint4 hit[LP_HITS];                               // chunks that hold an entry at or above the bound
    uint32_t hit_at[LP_HITS];
    // what the CTAs of a cluster send to the first one: sums against their maxima, and their top entries in
    // order, 0 behind the last
    float m[LP_CLUSTER_MAX], s[LP_CLUSTER_MAX], u[LP_CLUSTER_MAX];
    uint64_t list[LP_CLUSTER_MAX][LSSM_TOP_K_MAX];
    float red[2][LP_WARPS];
    alignas(16) uint32_t maxima[32];                  // the LP_TOPS largest thread maxima of every warp (order_key)
    uint32_t count, nhits, nsel, bound, wsum[LP_WARPS];
    uint64_t wbest[LP_WARPS];
    uint8_t sel[LP_THREADS];
};

// The first warp: of K of the 32 warp maxima the least, the largest K up to an order among values within 32
// steps of one another (for which every entry is made different by its place in the last bits).
__device__ __forceinline__ void find_bound(uint32_t K, LpShared& sh) {
    const uint32_t lane = threadIdx.x & 31, v = sh.maxima[lane], vr = (v & ~31u) | lane;
    uint32_t before = 0;
#pragma unroll
    for (uint32_t i = 0; i < 32; i += 4) {
        const uint4 o = *reinterpret_cast<const uint4*>(&sh.maxima[i]);
        before += (((o.x & ~31u) | i) > vr) + (((o.y & ~31u) | (i + 1)) > vr) + (((o.z & ~31u) | (i + 2)) > vr) +
                  (((o.w & ~31u) | (i + 3)) > vr);
    }
    const uint32_t least = __reduce_min_sync(FULL, before < K ? v : ~0u);
    if (lane == 0) sh.bound = least;
}

// The CTA's largest K entries of chunks [c0, c1), in order, into `list`. `tkey`: this thread's largest entry.
//
// sh.bound is a value that at least K entries reach. Only threads whose maximum reaches it can hold one of the
// top K, so only their chunks (about K / 256 of the slice, still in L2) are read again, and of those that reach
// it the elements. What reaches the bound is ranked by value and index. Thread t has chunks c0 + t, + LP_THREADS,
// ... (`dealt`: lane l of warp w has chunk c0 + l * LP_WARPS + w).
template <typename T>
__device__ __forceinline__ void cta_top(const Row<T>& row, uint32_t c0, uint32_t c1, uint32_t tkey, uint32_t K, LpShared& sh,
                                        bool dealt, uint64_t* list) {
    constexpr int VEC = 16 / sizeof(T);
    const uint32_t tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const uint32_t bound = sh.bound;
    uint32_t nsel = 0;
    // the threads that may hold an entry at or above the bound (ties), or one above it
    auto choose = [&](bool ties) {
        const bool chosen = ties ? tkey >= bound : tkey > bound;
        const uint32_t votes = __ballot_sync(FULL, chosen);
        uint32_t at = 0;
        if (lane == 0 && votes) at = atomicAdd(&sh.nsel, __popc(votes));
        at = __shfl_sync(FULL, at, 0) + __popc(votes & ((1u << lane) - 1));
        if (chosen) sh.sel[at] = (uint8_t)(dealt ? lane * LP_WARPS + wid : tid);
        __syncthreads();
        nsel = sh.nsel;
    };
    choose(true);
    const float bv = key_value(bound);
    const bool level = nsel > LP_THREADS / 4;   // many threads reach the bound: a masked or constant row
    auto collect = [&](bool ties) {
        // a warp takes four chosen threads at a time, a lane one of their chunks
        for (uint32_t i = wid * 4; i < nsel; i += LP_WARPS * 4)
            for (uint32_t k0 = 0; c0 + k0 < c1; k0 += 32 * LP_THREADS) {
                const uint32_t k = k0 + lane * LP_THREADS;
                uint4 w[4];
                uint32_t c[4], m[4];
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    c[g] = i + g < nsel ? min(c1, c0 + k + sh.sel[i + g]) : c1;
                    if (c[g] < c1) w[g] = row.chunk(c[g]);
                }
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float cm = c[g] < c1 ? chunk_max(w[g], T()) : -INFINITY;
                    const bool is = c[g] < c1 && !(ties ? cm < bv : cm <= bv);
                    m[g] = __ballot_sync(FULL, is);
                }
                const uint32_t total = __popc(m[0]) + __popc(m[1]) + __popc(m[2]) + __popc(m[3]);
                if (!total) continue;
                uint32_t p = 0;
                if (lane == 0) p = atomicAdd(&sh.nhits, total);
                p = __shfl_sync(FULL, p, 0);
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const uint32_t q = p + __popc(m[g] & ((1u << lane) - 1));
                    if ((m[g] >> lane & 1) && q < LP_HITS) { sh.hit[q] = w[g]; sh.hit_at[q] = c[g]; }
                    p += __popc(m[g]);
                }
            }
        __syncthreads();
        const uint32_t nh = min(sh.nhits, (uint32_t)LP_HITS);
        for (uint32_t q = tid; q < nh * VEC; q += LP_THREADS) {
            const int64_t e = row.index(sh.hit_at[q / VEC]) + q % VEC;
            const uint32_t k = order_key(load_one(reinterpret_cast<const T*>(sh.hit) + q));
            if (k < bound || (k == bound && !ties) || e < 0 || e >= (int64_t)row.V) continue;
            const uint32_t p = atomicAdd(&sh.count, 1u);
            if (p < LP_CAND) sh.cand[p] = rank_key(k, (uint32_t)e);
        }
        __syncthreads();
    };
    if (!level) collect(true);
    uint32_t n = sh.count;
    if (level || sh.nhits > LP_HITS || n > LP_CAND) {
        // Many equal to the bound: those above it first, then of the equal ones as many as are missing,
        // in the order of their index.
        __syncthreads();
        if (tid == 0) { sh.count = 0; sh.nhits = 0; sh.nsel = 0; }
        __syncthreads();
        choose(false);
        collect(false);
        n = sh.count;
        if (sh.nhits <= LP_HITS && n <= LP_CAND) {
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
                if (lane == 0) sh.wbest[wid] = best;
                __syncthreads();
                last = sh.wbest[0];
                for (int w = 1; w < LP_WARPS; ++w) last = sh.wbest[w] > last ? sh.wbest[w] : last;
                if (tid == 0) sh.cand[k] = last;
            }
            n = K;
        }
        __syncthreads();
    }
    // eight threads a candidate count those before it
    for (uint32_t i = tid / 8; i < (n + 3) / 4 * 4; i += LP_THREADS / 8) {
        const uint64_t k = i < n ? sh.cand[i] : ~0ull;
        uint32_t r = 0;
#pragma unroll 4
        for (uint32_t j = tid % 8; j < n; j += 8) r += sh.cand[j] > k;
        r += __shfl_xor_sync(FULL, r, 1);
        r += __shfl_xor_sync(FULL, r, 2);
        r += __shfl_xor_sync(FULL, r, 4);
        if (tid % 8 == 0 && i < n && r < K) list[r] = k;
    }
    if (tid >= n && tid < LSSM_TOP_K_MAX) list[tid] = 0;
}

// One CTA, or a cluster of nc over slices of the vocabulary, per row; one pass over the logits.
//
// The pass: a thread keeps s and u against its own lagging reference, and its largest entry; the threads' sums meet
// against the row's maximum m with e^(x - ref) = e^(x - m) e^(m - ref), where u moves by s (ref - m) too. The row is
// read once from HBM; cta_top's second look at a few chunks finds them in L2. Nothing between the kernel's phases
// goes through memory, so there is no workspace and no second launch.
//
// Why so: 256 threads x 2 groups of 4 x 16 bytes on their way, 4 CTAs an SM, put 128 KB of loads on an SM; the
// registers (64 a thread, and 16 bytes a thread spilled with fp16) allow no more. fp16 entries are worked on two a time (f32x2), with one ex2 each.
// What bounds it, at 2048 x 50288 fp16 with 20 alternatives: 47.1-49.1 us = 4.2-4.4 TB/s, 64-67 % of a copy's rate.
// Without alternatives 38.4 us, as a pass that only reads in this loop takes 37: the selection after a CTA's pass (barriers and
// second reads, a third of its cycles) leaves HBM idle where the other CTAs of the SM are in it too, and 2048 rows are
// 3.5 waves. 333 x 32001 fp32, 8 alternatives: 14.4 us; 64 x 256000 fp16, 5 of them: 14.4 us; one row of 50288: 8.2 us,
// latency of a launch, of reads one after the other and of barriers.
// Measured and not kept: a ring of bulk or 16-byte asynchronous copies in shared memory (54-56 us: the second trip
// through shared memory costs issue slots), 128 threads a CTA (56), CTAs that start at different places (49 where 50
// was), CTAs that walk over rows with the next row's first chunks copied ahead (107: spills), the last wave's rows
// split over clusters (51).
template <typename T>
__global__ void __launch_bounds__(LP_THREADS, LP_CTAS) k_logprobs(LogprobsArgs a, uint32_t nc) {
    __shared__ LpShared sh;
    const uint32_t tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const uint32_t r = blockIdx.x / nc, part = blockIdx.x % nc;
    const Row<T> row(a.logits, (uint64_t)r * a.row_stride, a.vocab);
    const uint32_t per = (row.chunks + nc - 1) / nc;
    const uint32_t c0 = min(row.chunks, part * per), c1 = min(row.chunks, c0 + per);
    if (nc > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // this CTA runs
    uint32_t target = LSSM_NO_TOKEN;
    if (part == 0 && tid == LP_THREADS - 32 && a.logp) target = a.targets[r];
    Sums<T> sum;
    float tmax = -INFINITY;
    // This thread's chunks c0 + tid, + LP_THREADS, ...: groups of LP_GROUP that lie inside the row, the next one
    // loaded before this one is worked on, and one by one what is left of the slice's ends.
    const uint32_t inner = row.inner(), outer = min(c1, row.outer());
    constexpr uint32_t STRIDE = LP_THREADS * LP_GROUP;
    // a slice with less than a chunk a thread is dealt to the warps in turn, so that all of them have maxima
    const bool dealt = c1 - c0 < LP_THREADS;
    uint32_t c = c0 + (dealt ? lane * LP_WARPS + wid : tid);
    const bool head = c < inner;
    if (head) c += LP_THREADS;
    uint32_t groups = c < outer ? (outer - c + LP_THREADS - 1) / LP_THREADS / LP_GROUP : 0;
    const uint4* at = row.base() + c;
    auto load = [&](uint4 (&d)[LP_GROUP]) {
#pragma unroll
        for (int g = 0; g < LP_GROUP; ++g) d[g] = __ldg(at + g * LP_THREADS);
        at += STRIDE;
    };
    auto work = [&](const uint4 (&d)[LP_GROUP]) {
        const float gm = chunks_max<T>(d);
        tmax = fmaxf(tmax, gm);
        sum.chunks(d, gm);
    };
    auto single = [&](uint4 d) {
        const uint4 one[1] = {d};
        const float gm = chunks_max<T>(one);
        tmax = fmaxf(tmax, gm);
        sum.chunks(one, gm);
    };
    uint4 w[LP_GROUP], next[LP_GROUP];
    if (groups) load(w);
    const uint32_t rest = c + groups * STRIDE;   // at most LP_GROUP chunks
#pragma unroll
    for (int g = 0; g < LP_GROUP; ++g)
        if (rest + g * LP_THREADS < c1) next[g] = row.chunk(rest + g * LP_THREADS);
    if (head) single(row.chunk(c - LP_THREADS));
#pragma unroll
    for (int g = 0; g < LP_GROUP; ++g)
        if (rest + g * LP_THREADS < c1) single(next[g]);
    while (groups) {
        if (--groups) load(next);
        work(w);
        if (!groups) break;
        if (--groups) load(w);
        work(next);
    }
    // HBM has nothing to do for this CTA from here on: the beginning of the row one full GPU of CTAs ahead goes to L2
    // (2048 x 50288 fp16, 20 alternatives: 50.5 us without, 49.3 with 16 KB, 47.2 with 32, 47.7 with 64, 51.1 with 128;
    // none 41.1, 39.7, 38.4, 39.3; 2048 x 32001 fp32 55.3, 53.4, 52.4, 51.9; 1024 x 100000 47.2, 47.2, 47.4, 49.3; 4096 x
    // 32000 63.3, 61.6, 61.5, 61.5; rows of 256000, and no more rows than CTAs: the same with and without).
    const uint64_t later = (uint64_t)r + (uint32_t)(a.sm_count * LP_CTAS);
    if (nc == 1 && tid == 0 && later < a.rows) {
        const Row<T> next_row(a.logits, later * a.row_stride, a.vocab);
        const uint32_t n = min(next_row.outer() - next_row.inner(), (uint32_t)LP_AHEAD);
        if (next_row.outer() > next_row.inner())
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;"
                         ::"l"(__cvta_generic_to_global(next_row.base() + next_row.inner())), "r"(n * 16) : "memory");
    }
    float xt = 0.0f;
    if (target < a.vocab) xt = load_one(row.x + target);
    // the largest thread maxima of every warp, the CTA's maximum, and the sums against it
    const uint32_t tkey = order_key(tmax), K = a.top_k;
    uint32_t mine = tkey;
#pragma unroll
    for (int q = 0; q < LP_TOPS; ++q) {
        const uint32_t top = __reduce_max_sync(FULL, mine);
        if (lane == 0) sh.maxima[wid * LP_TOPS + q] = top;
        if ((int)lane == __ffs(__ballot_sync(FULL, mine == top)) - 1) mine = 0;
    }
    if (tid == 0) { sh.count = 0; sh.nhits = 0; sh.nsel = 0; }
    __syncthreads();
    float m = key_value(__reduce_max_sync(FULL, sh.maxima[lane]));
    if (K && wid == 0) find_bound(K, sh);
    float2 s2 = unpack2(sum.s2), u2 = unpack2(sum.u2);
    float s = s2.x + s2.y, u = u2.x + u2.y;
    if (sum.ref > -INFINITY && m < INFINITY) Sums<T>::shift((sum.ref - m) * LOG2E + sum.slip(), s, u);
    s = warp_sum(s);
    u = warp_sum(u);
    if (lane == 0) { sh.red[0][wid] = s; sh.red[1][wid] = u; }
    __syncthreads();
    s = u = 0.0f;
#pragma unroll
    for (int w = 0; w < LP_WARPS; ++w) { s += sh.red[0][w]; u += sh.red[1][w]; }
    if (K) cta_top(row, c0, c1, tkey, K, sh, dealt, sh.list[part]);
    __syncthreads();
    if (nc > 1) {
        // the slices' sums and lists meet in the first CTA of the cluster, whose CTAs all run by now
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        if (part != 0 && tid < 32) {
            cg::cluster_group cl = cg::this_cluster();
            if (tid < K) *cl.map_shared_rank(&sh.list[part][tid], 0) = sh.list[part][tid];
            if (tid == 0) {
                *cl.map_shared_rank(&sh.m[part], 0) = m;
                *cl.map_shared_rank(&sh.s[part], 0) = s;
                *cl.map_shared_rank(&sh.u[part], 0) = u;
            }
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        if (part != 0) return;
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        const float pm = lane == 0 ? m : lane < nc ? sh.m[lane] : -INFINITY;
        float ps = lane == 0 ? s : lane < nc ? sh.s[lane] : 0.0f, pu = lane == 0 ? u : lane < nc ? sh.u[lane] : 0.0f;
        m = warp_max(pm);
        if (pm > -INFINITY && m < INFINITY) Sums<T>::shift((pm - m) * LOG2E, ps, pu);
        s = warp_sum(ps);
        u = warp_sum(pu);
    }
    const bool none = m == -INFINITY && !(s != s);
    const float ls = m == INFINITY ? __int_as_float(0x7FC00000) : logf(s);
    if (tid == LP_THREADS - 32) {   // a warp that has no alternative to write where there is one list
        if (a.lse) a.lse[r] = none ? -INFINITY : m + ls;
        if (a.entropy) a.entropy[r] = none ? 0.0f : ls - LN2 * (u / s);
        if (a.logp) {
            float v = 0.0f;
            if (target != LSSM_NO_TOKEN)
                v = target >= a.vocab ? __int_as_float(0x7FC00000) : none ? -INFINITY : (xt - m) - ls;
            a.logp[r] = v;
        }
    }
    for (uint32_t l = wid; l < nc && lane < K; l += LP_WARPS) {
        // entry `lane` of list `l`; its place: the entries before it, in its own list and in the others
        const uint64_t k = sh.list[l][lane];
        uint32_t place = lane;
        if (nc > 1) {
            uint32_t lo[LP_CLUSTER_MAX] = {};
#pragma unroll
            for (uint32_t step = 16; step; step >>= 1)
#pragma unroll
                for (uint32_t q = 0; q < LP_CLUSTER_MAX; ++q)
                    if (lo[q] + step <= K && sh.list[q][lo[q] + step - 1] > k) lo[q] += step;
#pragma unroll
            for (uint32_t q = 0; q < LP_CLUSTER_MAX; ++q) {
                if (lo[q] < K && sh.list[q][lo[q]] > k) ++lo[q];
                if (q < nc && q != l) place += lo[q];
            }
        }
        if (k && place < K) {
            a.top_ids[(uint64_t)r * K + place] = ~(uint32_t)k;
            a.top_logp[(uint64_t)r * K + place] = none ? -INFINITY : (key_value((uint32_t)(k >> 32)) - m) - ls;
        }
    }
}

// What a row's elements have in common, for d_j = g [j = t] - p_j (g + h (log p_j + H)).
struct GradRow {
    float lse, g, h, H;
    uint32_t t;
    bool none;
    __device__ GradRow(const LogprobsGradArgs& a, uint32_t r) {
        lse = a.lse[r];
        t = a.targets ? a.targets[r] : LSSM_NO_TOKEN;
        h = a.g_entropy ? a.g_entropy[r] : 0.0f;
        H = a.g_entropy ? a.entropy[r] : 0.0f;
        const bool outside = t != LSSM_NO_TOKEN && t >= a.vocab;
        none = lse == -INFINITY && !outside;
        g = a.g_logp && t != LSSM_NO_TOKEN ? a.g_logp[r] : 0.0f;
        if (outside) g = __int_as_float(0x7FC00000);
    }
    template <bool ENTROPY>
    __device__ __forceinline__ float operator()(float x, uint32_t j) const {
        const float lp = x - lse, p = ex2(lp * LOG2E);
        // p = 0 ends a masked entry, whose log p may be -inf: what is left is -p g, 0, or NaN for a target outside
        const float d = ENTROPY && p != 0.0f ? -p * fmaf(h, lp + H, g) : -p * g;
        return none ? 0.0f : j == t ? d + g : d;
    }
};

template <typename G> __device__ __forceinline__ void store_one(G* p, float v);
template <> __device__ __forceinline__ void store_one(__half* p, float v) { *p = __float2half_rn(v); }
template <> __device__ __forceinline__ void store_one(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ void store_one(float* p, float v) { *p = v; }

// The elements of one chunk in stores of 16 bytes (8 where they make no more), whose address has to allow it.
template <typename G, int n>
constexpr uint32_t STORE = n * sizeof(G) >= 16 ? 16 : 8;
template <typename G, int n>
__device__ __forceinline__ void store_chunk(G* p, const float (&v)[n]) {
    uint32_t w[n * sizeof(G) / 4];
#pragma unroll
    for (int i = 0; i < (int)(n * sizeof(G) / 4); ++i) {
        if constexpr (sizeof(G) == 4) w[i] = __float_as_uint(v[i]);
        else if constexpr (std::is_same<G, __half>::value) { const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]); memcpy(&w[i], &h, 4); }
        else { const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]); memcpy(&w[i], &h, 4); }
    }
    if constexpr (STORE<G, n> == 8) __stcs(reinterpret_cast<uint2*>(p), make_uint2(w[0], w[1]));
    else
#pragma unroll
        for (int i = 0; i < (int)(n * sizeof(G) / 16); ++i)
            __stcs(reinterpret_cast<uint4*>(p) + i, make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
}

// Elementwise: one read, one write. A CTA takes GRAD_CHUNKS chunks a thread of one row (a chunk is 16 bytes of
// logits); all of them are loaded before the first is worked on. Where the chunks' places in the output are not
// aligned for wide stores, a warp exchanges its 32 chunks through shared memory, so that a store instruction
// writes 32 neighbours.
// Bound by HBM: 2048 x 50288 fp16 to fp16 69.6-73.1 us = 5.6-5.9 TB/s, 86-90 % of a copy's rate (the same with a third fewer
// instructions, in pairs of entries: not kept); 257 x 32001 bf16 to fp32 with the entropy's term, rows at odd addresses,
// 12.6 us = 3.9 TB/s (35 us with stores of one element, before the exchange), where a launch's ends weigh more.
constexpr int GRAD_CHUNKS = 4;
template <typename T, typename G, bool ENTROPY>
__global__ void __launch_bounds__(LP_THREADS) k_logprobs_grad(LogprobsGradArgs a, uint32_t parts) {
    constexpr int VEC = 16 / sizeof(T);
    const uint32_t r = blockIdx.x / parts, part = blockIdx.x % parts;
    const Row<T> row(a.logits, (uint64_t)r * a.row_stride, a.vocab);
    G* out = static_cast<G*>(a.dlogits) + (uint64_t)r * a.grad_stride;
    const uint32_t c0 = part * (LP_THREADS * GRAD_CHUNKS) + threadIdx.x;
    uint4 w[GRAD_CHUNKS];
#pragma unroll
    for (int i = 0; i < GRAD_CHUNKS; ++i) {
        const uint32_t c = c0 + i * LP_THREADS;
        if (c >= row.inner() && c < row.outer()) w[i] = __ldcs(row.base() + c);
    }
    const GradRow grad(a, r);
    __shared__ float swap[LP_WARPS][32 * (VEC + 1)];   // a chunk to VEC + 1 words: no bank twice
    const uint32_t lane = threadIdx.x & 31;
    const bool wide = reinterpret_cast<uintptr_t>(out + row.index(row.inner())) % STORE<G, VEC> == 0;
#pragma unroll
    for (int i = 0; i < GRAD_CHUNKS; ++i) {
        const uint32_t c = c0 + i * LP_THREADS;
        const bool inside = c >= row.inner() && c < row.outer();
        const int64_t e = row.index(c);
        float d[VEC];
        if (inside) {
            float x[VEC];
            chunk_values<T>(w[i], x);
#pragma unroll
            for (int j = 0; j < VEC; ++j) d[j] = grad.template operator()<ENTROPY>(x[j], (uint32_t)e + j);
        }
        if (wide && inside) {
            store_chunk<G, VEC>(out + e, d);
        } else if (!wide && __all_sync(FULL, inside)) {
            float* mine = swap[threadIdx.x / 32];
#pragma unroll
            for (int j = 0; j < VEC; ++j) mine[lane * (VEC + 1) + j] = d[j];
            __syncwarp();
#pragma unroll
            for (uint32_t q = lane; q < 32 * VEC; q += 32) store_one(out + e - lane * VEC + q, mine[q / VEC * (VEC + 1) + q % VEC]);
            __syncwarp();
        } else if (c < row.chunks) {
            for (int j = 0; j < VEC; ++j)
                if (e + j >= 0 && e + j < (int64_t)row.V)
                    store_one(out + e + j, grad.template operator()<ENTROPY>(load_one(row.x + e + j), (uint32_t)(e + j)));
        }
    }
}

template <typename T, typename G>
cudaError_t launch_grad(const LogprobsGradArgs& a, cudaStream_t s) {
    constexpr uint32_t VEC = 16 / sizeof(T), SPAN = LP_THREADS * GRAD_CHUNKS;
    // one chunk more than the elements fill: a row may begin inside one
    const uint64_t parts = ((uint64_t)a.vocab + 2 * VEC - 2) / VEC / SPAN + 1, grid = parts * a.rows;
    if (grid > 0x7FFFFFFFu) return cudaErrorInvalidValue;
    if (a.g_entropy) k_logprobs_grad<T, G, true><<<(unsigned)grid, LP_THREADS, 0, s>>>(a, (uint32_t)parts);
    else k_logprobs_grad<T, G, false><<<(unsigned)grid, LP_THREADS, 0, s>>>(a, (uint32_t)parts);
    return cudaGetLastError();
}
template <typename T>
cudaError_t launch_grad_of(const LogprobsGradArgs& a, cudaStream_t s) {
    if (a.grad_dtype == LSSM_DT_F16) return launch_grad<T, __half>(a, s);
    if (a.grad_dtype == LSSM_DT_BF16) return launch_grad<T, __nv_bfloat16>(a, s);
    return launch_grad<T, float>(a, s);
}

}  // namespace

cudaError_t launch_logprobs(const LogprobsArgs& a, cudaStream_t s) {
    if (!a.rows) return cudaSuccess;
    // A few long rows: a cluster of CTAs a row. A cluster costs its join and the CTAs' own ends: slices below 32 K
    // entries and more than about three CTAs an SM lose by it (with 1 / 2 / 4 / 8 CTAs a row: 1 row of 256000 fp16,
    // top 5, 20.1 / 14.4 / 10.3 / 8.9 us; 64 rows 28.7 / 18.6 / 14.4 / 16.5; 333 rows of 32001 fp32, top 8,
    // 14.4 / 20.6 / 23.2 / 37.2; 128 rows of 50288 fp16, top 20, 10.1 / 10.3 / 12.5 / 18.7).
    uint32_t nc = 1;
    while (nc < LP_CLUSTER_MAX && (uint64_t)a.rows * nc * 2 <= 3ull * a.sm_count && a.vocab / (nc * 2) >= 32000) nc *= 2;
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
    if (a.dtype == LSSM_DT_F16) return launch_grad_of<__half>(a, s);
    if (a.dtype == LSSM_DT_BF16) return launch_grad_of<__nv_bfloat16>(a, s);
    return launch_grad_of<float>(a, s);
}

}  // namespace lssm
