// k_state_cache.cu — the quantised state cache: SSD states held as 8- or 16-bit codes with one
// scale per row of N, plus a window of the last tokens that the codes do not hold yet.
//
// For a sequence and head with decay rate a = -exp(A_log), window tokens j = 0..n and
//     w_j = dt_j exp(a sum_{i>j} dt_i)      alpha = exp(a sum_i dt_i)      S_q = code * scale
// the state after token n and the step's output are
//     S = alpha S_q + sum_j w_j x_j B_j^T           y = S C + D x_n
// so a decode step reads the codes once and writes only the new token's row of the window. When
// the window is full (n + 1 = W) the step also rounds S into new codes and empties it. The state
// is then rounded once in W tokens instead of at every token, and moved at 1 or 2 bytes an
// element instead of the 8 (read and write) of an fp32 state.
//
// A row of N elements has scale = max|S| / Q (Q = 127 or 32767, correctly rounded) and
// code = S / scale to the nearest whole number, ties to even. Rows whose scale would be below the
// smallest normal number are held as zeros; a row with a non-finite element gets scale NaN, so it
// reads back as NaN.
#include "device_util.cuh"
#include "lssm_internal.h"

namespace lssm {

namespace {

constexpr float kTiny = 1.17549435e-38f;

// dt of one token: clamp(softplus(raw + bias)). log1p keeps the digits of a small dt.
__device__ __forceinline__ float token_dt(float raw, float lo, float hi) {
    return fminf(fmaxf(raw > 20.0f ? raw : log1pf(expf(raw)), lo), hi);
}

// A row's scale and what its codes are computed with.
struct RowQuant {
    float scale, inv, half;   // half: what a remainder may be at most
    bool sound;               // no NaN, no infinity
    // amax: the row's largest magnitude, NaN or infinite where an element is
    __device__ __forceinline__ RowQuant(float amax, float Q) {
        scale = __fdiv_rn(amax, Q);
        sound = amax < INFINITY;
        if (!sound) scale = __int_as_float(0x7FC00000);
        else if (scale < kTiny) scale = 0.0f;
        inv = scale > 0.0f ? __frcp_rn(scale) : 0.0f;
        half = scale > 0.0f ? 0.5f * scale : INFINITY;
    }
    // of a scale that is worked out already
    struct Known { float scale, inv; };
    __device__ __forceinline__ RowQuant(Known k) : scale(k.scale), inv(k.inv) {
        half = scale > 0.0f ? 0.5f * scale : INFINITY;
        sound = scale == scale;
    }
    // what lane l of the warp has
    __device__ __forceinline__ RowQuant of_lane(int l) const {
        return RowQuant(Known{__shfl_sync(0xffffffffu, scale, l), __shfl_sync(0xffffffffu, inv, l)});
    }
};
// Codes of four elements as whole numbers in the low bits of the results. Added to 1.5 * 2^23, v / scale is rounded
// to a whole number, ties to even, but the reciprocal may have carried it over a half step. The remainder
// v - q * scale, exact in one fma, tells: only where it is half a step or more (about once in a million) is the
// code looked at again.
__device__ __forceinline__ void quantise4(const float (&v)[4], const RowQuant& z, uint32_t (&c)[4]) {
    constexpr float MAGIC = 12582912.0f;
    float worst = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float m = fmaf(v[i], z.inv, MAGIC);
        c[i] = __float_as_uint(m);
        worst = fmaxf(worst, fabsf(fmaf(MAGIC - m, z.scale, v[i])));
    }
    if (worst >= z.half) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float q = __uint_as_float(c[i]) - MAGIC, r = fmaf(-q, z.scale, v[i]);
            if (fabsf(r) > z.half || (fabsf(r) == z.half && (c[i] & 1))) c[i] += r > 0.0f ? 1 : -1;
        }
    }
}

template <typename Code>
__device__ __forceinline__ Code quantise1(float v, const RowQuant& z) {
    const float four[4] = {v, 0.0f, 0.0f, 0.0f};
    uint32_t c[4];
    quantise4(four, z, c);
    return z.sound ? (Code)c[0] : (Code)0;
}
// four codes, side by side
__device__ __forceinline__ uint32_t pack_codes8(const uint32_t (&c)[4]) {
    return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
}
__device__ __forceinline__ uint2 pack_codes16(const uint32_t (&c)[4]) {
    return make_uint2(__byte_perm(c[0], c[1], 0x5410), __byte_perm(c[2], c[3], 0x5410));
}
template <typename Code>
__device__ __forceinline__ void store_codes4(Code* to, const float (&v)[4], const RowQuant& z) {
    uint32_t c[4];
    quantise4(v, z, c);
    if constexpr (sizeof(Code) == 1) *reinterpret_cast<uint32_t*>(to) = z.sound ? pack_codes8(c) : 0u;
    else *reinterpret_cast<uint2*>(to) = z.sound ? pack_codes16(c) : make_uint2(0u, 0u);
}
// Window weights of one head, lane j of a warp for token j (W <= 32): the sum over later tokens
// is taken from the end, so one very large dt costs the tokens after it no digits.
__device__ __forceinline__ void window_weights(float a, float dt, uint32_t lane, uint32_t count, float* w, float* alpha) {
    if (lane >= count) dt = 0.0f;
    float s = lane < count ? a * dt : 0.0f;   // a may be -inf
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const float t = __shfl_down_sync(0xffffffffu, s, o);
        if (lane + o < 32) s += t;
    }
    float later = __shfl_down_sync(0xffffffffu, s, 1);
    if (lane == 31) later = 0.0f;
    *w = dt * expf(later);
    *alpha = expf(__shfl_sync(0xffffffffu, s, 0));
}

constexpr int SC_THREADS = 256;

// Any shape: one CTA per (sequence, head), ANY_ROWS rows at a time; lane l of a warp takes elements l, l + 32, ... of a
// row, so neighbours are read and written together whatever N and the arrays' alignment are.
// A step: S_q C of the rows by warps, C . B_j of the window's tokens by warps, then y by a thread a row.
// A fold or a load: a warp keeps 32 elements of every B_j in registers (KB * 16 of them) and walks down the rows.
// Only for P or N above 256, which no known model has: it is right for every shape, and issue bounds it (the products
// are on the CUDA cores). With the shapes above that k_state_tc takes it took twice that kernel's time.
constexpr uint32_t ANY_ROWS = 128, ANY_ILP = 8;   // rows at a time; of them, rows a warp has on their way
template <typename Code, int MODE, int KB>
__global__ void __launch_bounds__(SC_THREADS, KB == 1 ? 3 : 2) k_state_any(StateCacheArgs a) {
    constexpr float Q = sizeof(Code) == 1 ? 127.0f : 32767.0f;
    constexpr int WARPS = SC_THREADS / 32, J = 16 * KB;
    __shared__ __align__(16) float s_xw[ANY_ROWS][J + 4];   // w_j x_j[p], 0 behind the window's tokens
    __shared__ float s_w[32], s_cb[32], s_row[ANY_ROWS], s_scale[ANY_ROWS], s_inv[ANY_ROWS], s_alpha;
    __shared__ uint32_t s_top[ANY_ROWS];
    const uint32_t h = blockIdx.x % a.H, b = blockIdx.x / a.H, g = h / (a.H / a.G);
    const uint32_t tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const uint64_t bh = blockIdx.x, xrow = (uint64_t)a.H * a.P, brow = (uint64_t)a.G * a.N;
    // a step's token is number n of the window; `count` tokens with it
    const uint32_t filled = a.fill[bh], n = MODE == 0 ? min(filled, a.W - 1) : a.W;
    const uint32_t count = MODE == 0 ? n + 1 : min(filled, a.W);
    const bool fold = MODE == 0 && count == a.W;
    const __half* wx = a.win_x + (uint64_t)b * a.W * xrow + (uint64_t)h * a.P;
    __half* wB = a.win_B + (uint64_t)b * a.W * brow + (uint64_t)g * a.N;
    const __half* xn = MODE == 0 ? a.x + b * a.x_bs + (uint64_t)h * a.P : nullptr;
    const __half* Bn = MODE == 0 ? a.B + b * a.bc_bs + (uint64_t)g * a.N : nullptr;
    const __half* Cn = MODE == 0 ? a.C + b * a.bc_bs + (uint64_t)g * a.N : nullptr;
    auto token_x = [&](uint32_t j) { return MODE == 0 && j == n ? xn : wx + j * xrow; };
    auto token_B = [&](uint32_t j) { return MODE == 0 && j == n ? Bn : wB + j * brow; };
    if (wid == 0) {
        float dt = 0.0f;
        if (lane < count && lane != n) dt = a.win_dt[bh * a.W + lane];
        if (MODE == 0 && lane == n)
            dt = token_dt(__half2float(a.dt_raw[b * a.dt_bs + h]) + __half2float(a.dt_bias[h]), a.dt_min, a.dt_max);
        float wj, al;
        window_weights(-expf(__half2float(a.A_log[h])), dt, lane, count, &wj, &al);
        s_w[lane] = wj;
        if (lane == 0) s_alpha = al;
        if (MODE == 0 && lane == n) a.win_dt[bh * a.W + n] = dt;
    }
    if (MODE == 0)
        for (uint32_t j = wid; j < count; j += WARPS) {
            const __half* B = token_B(j);
            float d = 0.0f;
#pragma unroll 4
            for (uint32_t i = lane; i < a.N; i += 32) d = fmaf(__half2float(B[i]), __half2float(Cn[i]), d);
            d = warp_sum(d);
            if (lane == 0) s_cb[j] = d;
        }
    __syncthreads();
    const float alpha = s_alpha;
    const uint32_t chunks = (a.N + 31) / 32, splits = chunks >= WARPS ? 1 : WARPS / chunks;
    for (uint32_t p0 = 0; p0 < a.P; p0 += ANY_ROWS) {
        const uint32_t rows = min(ANY_ROWS, a.P - p0);
        Code* codes = static_cast<Code*>(a.codes) + (bh * a.P + p0) * a.N;
        float* scales = a.scales + bh * a.P + p0;
        if (MODE == 0) {
            for (uint32_t p = wid * 4; p < rows; p += WARPS * 4) {
                float d[4] = {};
#pragma unroll 4
                for (uint32_t i = lane; i < a.N; i += 32) {
                    const float c = __half2float(Cn[i]);
#pragma unroll
                    for (uint32_t r = 0; r < 4; ++r)
                        if (p + r < rows) d[r] = fmaf((float)codes[(uint64_t)(p + r) * a.N + i], c, d[r]);
                }
#pragma unroll
                for (uint32_t r = 0; r < 4; ++r) {
                    d[r] = warp_sum(d[r]);
                    if (lane == r && p + r < rows) s_row[p + r] = d[r];
                }
            }
            __syncthreads();
            if (tid < rows) {
                const uint64_t o = (uint64_t)h * a.P + p0 + tid;
                __half x[J];   // all on their way before the first is used
#pragma unroll
                for (uint32_t j = 0; j < J; ++j) x[j] = j < count ? token_x(j)[p0 + tid] : __ushort_as_half(0);
                float yw = 0.0f;
#pragma unroll
                for (uint32_t j = 0; j < J; ++j)
                    if (j < count) yw = fmaf(s_w[j] * s_cb[j], __half2float(x[j]), yw);
                const __half xh = xn[p0 + tid];
                const float Dh = a.has_D ? __half2float(a.D[h]) : 0.0f;
                const __half yh = __float2half_rn(fmaf(alpha * scales[tid], s_row[tid], yw) + Dh * __half2float(xh));
                a.y[b * a.y_bs + o] = a.z ? __float2half_rn(silu(__half2float(a.z[b * a.z_bs + o])) * __half2float(yh)) : yh;
                a.win_x[((uint64_t)b * a.W + n) * xrow + o] = xh;
            }
            __syncthreads();
            if (!fold) continue;
        }
        for (uint32_t p = lane; p < rows; p += 32)
#pragma unroll
            for (uint32_t j = wid; j < J; j += WARPS) s_xw[p][j] = j < count ? s_w[j] * __half2float(token_x(j)[p0 + p]) : 0.0f;
        if (tid < rows) {
            s_row[tid] = alpha * scales[tid];
            s_top[tid] = 0;
        }
        __syncthreads();
        // PASS 0: the rows' largest magnitudes (fold) or the state itself (load); 1: the codes. A walk down the rows
        // for every 32 elements.
        auto walk = [&](auto pass) {
            for (uint32_t task = wid; task < chunks * splits; task += WARPS) {
                const uint32_t i = task % chunks * 32 + lane;
                const bool in = i < a.N;
                float B[J];
#pragma unroll
                for (uint32_t j = 0; j < J; ++j) B[j] = in && j < count ? __half2float(token_B(j)[i]) : 0.0f;
                for (uint32_t p = task / chunks * ANY_ILP; p < rows; p += splits * ANY_ILP) {
                    float v[ANY_ILP];
                    const uint32_t here = min(ANY_ILP, rows - p);
#pragma unroll
                    for (uint32_t r = 0; r < ANY_ILP; ++r) v[r] = in && r < here ? (float)codes[(uint64_t)(p + r) * a.N + i] : 0.0f;
#pragma unroll
                    for (uint32_t r = 0; r < ANY_ILP; ++r) {
                        if (r >= here) break;
                        v[r] *= s_row[p + r];
#pragma unroll
                        for (uint32_t j = 0; j < J; j += 4) {
                            if (j >= count) break;
                            const float4 x = *reinterpret_cast<const float4*>(&s_xw[p + r][j]);
                            v[r] = fmaf(x.x, B[j], v[r]);
                            v[r] = fmaf(x.y, B[j + 1], v[r]);
                            v[r] = fmaf(x.z, B[j + 2], v[r]);
                            v[r] = fmaf(x.w, B[j + 3], v[r]);
                        }
                        const uint64_t at = (uint64_t)(p + r) * a.N + i;
                        if constexpr (MODE == 1) {
                            if (in) store_any(a.state, (bh * a.P + p0) * a.N + at, a.state_dtype, v[r]);
                        } else if constexpr (decltype(pass)::value == 0) {
                            // the bits of |v| order as the values do, NaN above infinity
                            const uint32_t top = __reduce_max_sync(0xffffffffu, in ? __float_as_uint(v[r]) & 0x7FFFFFFFu : 0u);
                            if (lane == 0) atomicMax(&s_top[p + r], top);
                        } else if (in) {
                            codes[at] = quantise1<Code>(v[r], RowQuant(RowQuant::Known{s_scale[p + r], s_inv[p + r]}));
                        }
                    }
                }
            }
        };
        walk(std::integral_constant<int, 0>());
        __syncthreads();
        if (MODE == 0) {
            if (tid < rows) {
                const RowQuant z(__uint_as_float(s_top[tid]), Q);
                scales[tid] = s_scale[tid] = z.scale;
                s_inv[tid] = z.inv;
            }
            __syncthreads();
            walk(std::integral_constant<int, 1>());
            __syncthreads();
        }
    }
    if (MODE == 0) {
        // the first head of a group keeps the group's B row; every head takes row n from its argument
        if (h % (a.H / a.G) == 0)
            for (uint32_t i = tid; i < a.N; i += SC_THREADS) wB[n * brow + i] = Bn[i];
        if (tid == 0) a.fill[bh] = fold ? 0 : count;
    }
}

// ---------------------------------------------------------------------------
//  N = 64, 128 or 256, P a multiple of 16: tensor-core kernel
// ---------------------------------------------------------------------------
// A CTA takes `heads` heads of one group and sequence; a warp 16 rows of a head's state at a time. With m16n8k16
// (f16 in, f32 out), lane (g, t) = (lane / 4, lane % 4), and an order of k that lets a lane load its codes as they lie:
//   S_q C       A = codes (exact in f16: 8 bits as they are, 16 bits as 256 * high + low), B = C in every column
//   C . B_j     A = the window's B rows, B = C in every column (one warp; 16 tokens an instruction)
//   sum_j w_j x_j B_j^T (fold, load)   m16n8k8 in tf32: A = w_j x_j[p] as two terms of 11 bits, which have fp32's range, B =
//               the window's B (exact: f16 has 11 bits too); a lane gets the elements whose codes it holds.
// A code is converted, multiplied and added in about one instruction for 30 elements.
constexpr int TC_THREADS = 256, TC_WARPS = TC_THREADS / 32, TC_HEADS = 4;
constexpr uint32_t STAGE_PITCH = 48;        // words a row of a load's staged stores: two rows' lanes share no bank
constexpr uint32_t TC_BYTES = 32 * 1024;   // of codes a CTA holds (one head may have more)
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma1688(float (&d)[4], const uint32_t (&a)[4], float b0, float b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(__float_as_uint(b0)), "r"(__float_as_uint(b1)));
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { uint32_t u; memcpy(&u, &h, 4); return u; }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { __half2 h; memcpy(&h, &u, 4); return h; }
// Two unsigned bytes of w (chosen by sel, the 0x64 bytes from the constant) as f16 minus `off`: exact, 1024 + byte is.
__device__ __forceinline__ uint32_t bytes_h2(uint32_t w, uint32_t sel, float off) {
    return h2_bits(__hsub2(bits_h2(__byte_perm(w, 0x64646464u, sel)), __float2half2_rn(off)));
}

// Four codes as fp32.
__device__ __forceinline__ void code_values_of(uint32_t c, float (&v)[4]) {
    const uint32_t w = c ^ 0x80808080u;
    const float2 a = __half22float2(bits_h2(bytes_h2(w, 0x4140, 1152.0f)));
    const float2 b = __half22float2(bits_h2(bytes_h2(w, 0x4342, 1152.0f)));
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}
__device__ __forceinline__ void code_values_of(uint2 c, float (&v)[4]) {
    // added to 1.5 * 2^23 a 16-bit number is a float's low bits
    const uint32_t w[2] = {c.x ^ 0x80008000u, c.y ^ 0x80008000u};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = __uint_as_float(__byte_perm(w[i / 2], 0x4B400000u, i & 1 ? 0x7632 : 0x7610)) - (12582912.0f + 32768.0f);
}

template <typename Code>
__device__ __forceinline__ void code_values(const uint8_t* at, float (&v)[4]) {
    if constexpr (sizeof(Code) == 1) code_values_of(*reinterpret_cast<const uint32_t*>(at), v);
    else code_values_of(*reinterpret_cast<const uint2*>(at), v);
}

__device__ __forceinline__ float max_keep_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ void copy_async16(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void ldmatrix_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
// Two tf32 terms of v: 22 bits together, whatever its size (the second is lost below 2^-115).
__device__ __forceinline__ uint32_t tf32_bits(float v) { uint32_t u; asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(u) : "f"(v)); return u; }
__device__ __forceinline__ void split2(float v, uint32_t* hi, uint32_t* lo) {
    *hi = tf32_bits(v);
    *lo = tf32_bits(v - __uint_as_float(*hi));
}

// Shared memory of a CTA: the heads' codes (rows of N, their 16-byte pieces exchanged by row so that neither
// 16-byte nor 4-byte reads of 8 rows meet in a bank), the window's x (a row a token) and B, C,
// S_q C of every row, and the pair layout of B.
template <typename Code, int KB, int N>
struct TcShared {
    static constexpr uint32_t ROW = N * sizeof(Code), PIECES = ROW / 16;
    static constexpr uint32_t B_PITCH = N * 2 + 16, PAIR_PITCH = N + 8;   // bytes; words
    uint32_t x_pitch, x, B, C, dot, pairs, total;   // bytes from the start; codes are first
    __host__ __device__ TcShared(uint32_t rows) {   // rows: heads * P
        x_pitch = rows * 2 + 16;
        x = rows * ROW;
        B = x + KB * 16 * x_pitch;
        C = B + KB * 16 * B_PITCH;
        dot = C + N * 2;
        pairs = dot + rows * 4;
        total = pairs + KB * 8 * PAIR_PITCH * 4;
    }
    // rows of 64 bytes lie two to a line of banks; others have a line or more of their own
    static __device__ __forceinline__ uint32_t swap(uint32_t row) { return PIECES == 4 ? row >> 1 & 3 : (row & 1) << 2 | (row >> 1 & 3); }
    static __device__ __forceinline__ uint32_t piece(uint32_t row, uint32_t i) { return row * ROW + ((i ^ swap(row)) << 4); }
};

__device__ __forceinline__ uint4 lds16(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }

// A padded load: four neighbours of the state in one store; if not, its 16-bit states through shared memory.
__host__ __device__ __forceinline__ bool wide_rows(const StateCacheArgs& a) { return a.N % 4 == 0 && (reinterpret_cast<uintptr_t>(a.state) & 15) == 0; }
__host__ __device__ __forceinline__ bool staged_load(const StateCacheArgs& a) { return !wide_rows(a) && a.state_dtype != LSSM_DT_F32; }

// A step or a load on the tensor cores. A CTA takes the codes of one to TC_HEADS heads of a group: they share the
// window's B, C and C . B_j. MODE 0: a step, which folds where it fills the window; MODE 1: a load.
// KB: blocks of 16 window tokens (W <= 16 * KB). Grid: blocks of heads, groups, sequences.
// PAD: any N up to the template's and any P, alignment and stride: one head a CTA, read and written element by element,
// with zeros behind its rows and columns.
//
// y = alpha scale (code . C) + sum_j w_j (C . B_j) x_j + D x: the codes are the A operand as they are, since whole
// numbers up to 2048 are exact in f16 (16 bits: two bytes, 256 hi + lo), and C is an f16 input: the product has no
// rounding but its fp32 sums'. Bytes become f16 by one byte permutation into 0x64.. and one subtraction, so that no
// conversion runs. A fold or load adds sum_j (w_j x_j) B_j^T, the product of two 16 x W operands: w_j x_j, an fp32
// product, goes in as two tf32 terms (22 bits). f16 terms would want a scale, and under any that rows or tokens share,
// the small ones lose digits to the large ones: decays alone put 2^37 between a window's first token and its last. They take
// half as many instructions and were faster at the 64 sequences below: a step with folds 26.2 us against 27.6, a load to fp16
// 29.7 against 31.1 (with W 32 29.3 against 32.3 and 37.5 against 48.9).
// Codes wait in shared memory in an order that lets a lane take 16 bytes of a row without two lanes on one bank.
//
// What bounds it, at 64 sequences x 80 heads of 64 x 128, 8 bits, W 16: 17.0 us without a fold (42 MB of codes, 47 MB
// in all; 2.8 TB/s, 42 % of a copy's rate). 1280 CTAs of about 6 us are 2.2 waves of 4 CTAs an SM, each a chain of
// reads, three barriers and products: latency and issue, not HBM. With one sequence in 16 folding at each step, as
// sequences that began at different times do, 27.6 us; with all of them folding 60 us, once in 16 steps. The fp32 step
// (ssd_step_batched) takes 51 us each time. 16 bits: 25.0 us. One sequence of 24 heads: 4.1 us, a launch's latency.
// A load of the same 64 sequences takes 31.1 us to fp16 (126 MB, 4.1 TB/s; shared memory's and the products' latency)
// and 38.8 us to fp32 (210 MB, 5.4 TB/s; HBM).
// 16 sequences x 64 heads of 75 x 203, 8 bits, padded: 29 us a step (55 on the CUDA cores).
// Measured and not kept: a persistent CTA with the next heads' codes on their way (24.8-30 us against 23.8 at the time:
// registers for two of everything leave 2 CTAs an SM), codes in two parts that are waited for one after the other
// (18.6 against 17.2), all W rows of the window read without waiting for `fill` (19.3; one sequence 5.0 against 4.1),
// 3 or 5 CTAs an SM, CTAs of half the size (19.0), odd N's codes through an aligned copy in shared memory; fp32 pairs
// in one instruction (f32x2) for the fold and the load: 2 % less a step, 1 % more a load.
template <typename Code, int MODE, int KB, int N, bool PAD>
__global__ void __launch_bounds__(TC_THREADS, KB == 1 ? 4 : 3) k_state_tc(StateCacheArgs a, uint32_t heads, uint32_t per_group) {
    constexpr float Q = sizeof(Code) == 1 ? 127.0f : 32767.0f;
    using Sh = TcShared<Code, KB, N>;
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ __align__(16) float s_w[TC_HEADS][32];
    __shared__ __align__(16) float s_cb[MODE == 0 ? 16 * KB : 1];
    __shared__ float s_alpha[TC_HEADS], s_D[TC_HEADS];
    const uint32_t first = blockIdx.x * heads, nh = min(heads, per_group - first), b = blockIdx.z;
    const uint32_t h0 = blockIdx.y * per_group + first;   // heads h0 .. h0 + nh - 1
    const uint32_t tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t real = nh * a.P, rows = PAD ? (a.P + 15) / 16 * 16 : real, bh0 = b * a.H + h0;   // with padding: rows
    const uint32_t n_real = PAD ? a.N : N, xrow = a.H * a.P, brow = a.G * n_real;
    const Sh sh(PAD ? rows : heads * a.P);
    const uint32_t sm0 = smem_u32(sm);
    Code* const g_codes = static_cast<Code*>(a.codes) + (uint64_t)bh0 * a.P * n_real;
    uint8_t* codes = reinterpret_cast<uint8_t*>(g_codes);
    float* scales = a.scales + (uint64_t)bh0 * a.P;
    const uint32_t filled = a.fill[bh0];
    // what warp w < nh needs for head w's weights, and this thread's row
    float p_dt = 0.0f;
    __half p_raw = __ushort_as_half(0), p_bias = p_raw, p_A = p_raw, p_D = p_raw;
    if (wid < nh) {
        const uint32_t h = h0 + wid;
        if (lane < a.W) p_dt = a.win_dt[(uint64_t)(bh0 + wid) * a.W + lane];
        p_A = a.A_log[h];
        if (MODE == 0) {
            p_raw = a.dt_raw[b * a.dt_bs + h];
            p_bias = a.dt_bias[h];
            if (a.has_D) p_D = a.D[h];
        }
    }
    const float my_scale = tid < real ? scales[tid] : 0.0f;
    auto code_at = [&](uint32_t row, uint32_t e) { return Sh::piece(row, e * sizeof(Code) >> 4) + (e * sizeof(Code) & 15); };
    if constexpr (PAD) {
        for (uint32_t r = wid; r < rows; r += TC_WARPS)
#pragma unroll
            for (uint32_t e = lane; e < N; e += 32)
                *reinterpret_cast<Code*>(sm + code_at(r, e)) = r < real && e < n_real ? g_codes[r * n_real + e] : (Code)0;
    } else {
        const uint8_t* from = codes + tid * 16;
        constexpr uint32_t STEP = TC_THREADS / Sh::PIECES;   // rows a round, a multiple of 8: the exchange repeats
        uint32_t to = sm0 + Sh::piece(tid / Sh::PIECES, tid % Sh::PIECES);
        for (uint32_t r = tid / Sh::PIECES; r < rows; r += STEP, from += TC_THREADS * 16, to += TC_THREADS * 16) copy_async16(to, from);
    }
    // A step's token is number n of the window; `count` tokens with it. All heads of a sequence have the same.
    const uint32_t n = MODE == 0 ? min(filled, a.W - 1) : a.W, count = MODE == 0 ? n + 1 : min(filled, a.W);
    const bool fold = MODE == 0 && count == a.W;
    const __half* wx = a.win_x + ((uint64_t)b * a.W * xrow + (uint64_t)h0 * a.P);
    __half* wB = a.win_B + ((uint64_t)b * a.W * brow + blockIdx.y * n_real);
    const __half* xn = MODE == 0 ? a.x + b * a.x_bs + (uint64_t)h0 * a.P : nullptr;
    const __half* Bn = MODE == 0 ? a.B + b * a.bc_bs + blockIdx.y * n_real : nullptr;
    const __half* Cn = MODE == 0 ? a.C + b * a.bc_bs + blockIdx.y * n_real : nullptr;
    // the window's rows, a warp each of x; those behind its tokens are zeros, so that their
    // products are
    if constexpr (PAD) {
        const __half zero = __ushort_as_half(0);
        if (MODE == 0 || count)
            for (uint32_t j = wid; j < KB * 16; j += TC_WARPS) {
                const __half* xj = MODE == 0 && j == n ? xn : wx + (uint64_t)j * xrow;
                const __half* Bj = MODE == 0 && j == n ? Bn : wB + (uint64_t)j * brow;
#pragma unroll 4
                for (uint32_t e = lane; e < rows; e += 32)
                    *reinterpret_cast<__half*>(sm + sh.x + j * sh.x_pitch + e * 2) = j < count && e < real ? xj[e] : zero;
#pragma unroll
                for (uint32_t e = lane; e < N; e += 32)
                    *reinterpret_cast<__half*>(sm + sh.B + j * Sh::B_PITCH + e * 2) = j < count && e < n_real ? Bj[e] : zero;
            }
        if (MODE == 0 && tid < N) *reinterpret_cast<__half*>(sm + sh.C + tid * 2) = tid < n_real ? Cn[tid] : zero;
    } else if (MODE == 0 || count) {
        for (uint32_t j = wid; j < KB * 16; j += TC_WARPS) {
            const __half* from = MODE == 0 && j == n ? xn : wx + (uint64_t)j * xrow;
            const uint32_t to = sh.x + j * sh.x_pitch;
            for (uint32_t e = lane; e < rows / 8; e += 32) {
                if (j < count) copy_async16(sm0 + to + e * 16, from + e * 8);
                else *reinterpret_cast<uint4*>(sm + to + e * 16) = make_uint4(0, 0, 0, 0);
            }
        }
#pragma unroll
        for (uint32_t i = tid; i < KB * 16 * (N / 8); i += TC_THREADS) {
            const uint32_t j = i / (N / 8), e = i % (N / 8), to = sh.B + j * Sh::B_PITCH + e * 16;
            if (j < count) copy_async16(sm0 + to, (MODE == 0 && j == n ? Bn : wB + (uint64_t)j * brow) + e * 8);
            else *reinterpret_cast<uint4*>(sm + to) = make_uint4(0, 0, 0, 0);
        }
    }
    if (!PAD && MODE == 0 && tid < N / 8) copy_async16(sm0 + sh.C + tid * 16, Cn + tid * 8);
    if (wid < nh) {
        float dt = lane < count ? p_dt : 0.0f;
        if (MODE == 0 && lane == n) dt = token_dt(__half2float(p_raw) + __half2float(p_bias), a.dt_min, a.dt_max);
        float wj, al;
        window_weights(-expf(__half2float(p_A)), dt, lane, count, &wj, &al);
        s_w[wid][lane] = wj;
        if (lane == 0) { s_alpha[wid] = al; s_D[wid] = __half2float(p_D); }
        if (MODE == 0 && lane == n) a.win_dt[(uint64_t)(bh0 + wid) * a.W + n] = dt;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    uint32_t(*pairs)[Sh::PAIR_PITCH] = reinterpret_cast<uint32_t(*)[Sh::PAIR_PITCH]>(sm + sh.pairs);
    if (MODE == 1 ? count > 0 : fold) {
        // tokens 2 jp and 2 jp + 1 of the window's B side by side, as the product wants them
#pragma unroll
        for (uint32_t i = tid; i < KB * 8 * (N / 2); i += TC_THREADS) {
            const uint32_t jp = i / (N / 2), e = i % (N / 2) * 2;
            const uint8_t* from = sm + sh.B + 2 * jp * Sh::B_PITCH + e * 2;
            const uint32_t p0 = *reinterpret_cast<const uint32_t*>(from), p1 = *reinterpret_cast<const uint32_t*>(from + Sh::B_PITCH);
            // of every four elements in the order 0, 2, 1, 3: a lane uses 0 and 2, or 1 and 3, of them
            const uint32_t at = (e & ~3u) + (e >> 1 & 1);
            pairs[jp][at] = __byte_perm(p0, p1, 0x5410);
            pairs[jp][at + 2] = __byte_perm(p0, p1, 0x7632);
        }
        if (MODE == 1) __syncthreads();
    }
    auto head_of = [&](uint32_t row) { return (uint32_t)(row >= a.P) + (row >= 2 * a.P) + (row >= 3 * a.P); };
    if constexpr (MODE == 0) {
        float* s_dot = reinterpret_cast<float*>(sm + sh.dot);
        // S_q C of every row
        for (uint32_t tile = wid; tile < rows / 16; tile += TC_WARPS) {
            const uint32_t row = tile * 16 + g, sw = Sh::swap(row);   // of row + 8, too
            const uint8_t* r0 = sm + row * Sh::ROW;
            // 16 bytes a row and lane at a time, piece 4 i + t
            float lo[2][4] = {}, hi[2][4] = {};
#pragma unroll
            for (int i = 0; i < (int)Sh::PIECES / 4; ++i) {
                const uint32_t at = ((4 * i + t) ^ sw) << 4;
                const uint4 u4 = lds16(r0 + at), v4 = lds16(r0 + 8 * Sh::ROW + at);
                const uint32_t u[4] = {u4.x, u4.y, u4.z, u4.w}, v[4] = {v4.x, v4.y, v4.z, v4.w};
                constexpr int PER = 16 / sizeof(Code);   // codes a piece
                uint32_t c[PER / 2];
#pragma unroll
                for (int k = 0; k < PER / 8; ++k) {
                    const uint4 w = lds16(sm + sh.C + ((4 * i + t) * PER + 8 * k) * 2);
                    c[4 * k] = w.x; c[4 * k + 1] = w.y; c[4 * k + 2] = w.z; c[4 * k + 3] = w.w;
                }
                if constexpr (sizeof(Code) == 1) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const uint32_t x = u[q] ^ 0x80808080u, y = v[q] ^ 0x80808080u;
                        mma16816(lo[q & 1], bytes_h2(x, 0x4140, 1152.0f), bytes_h2(y, 0x4140, 1152.0f), bytes_h2(x, 0x4342, 1152.0f),
                                 bytes_h2(y, 0x4342, 1152.0f), c[2 * q], c[2 * q + 1]);
                    }
                } else {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const uint32_t x0 = u[2 * q], x1 = u[2 * q + 1], y0 = v[2 * q], y1 = v[2 * q + 1];
                        mma16816(lo[q], bytes_h2(x0, 0x4240, 1024.0f), bytes_h2(y0, 0x4240, 1024.0f), bytes_h2(x1, 0x4240, 1024.0f),
                                 bytes_h2(y1, 0x4240, 1024.0f), c[2 * q], c[2 * q + 1]);
                        mma16816(hi[q], bytes_h2(x0 ^ 0x80008000u, 0x4341, 1152.0f), bytes_h2(y0 ^ 0x80008000u, 0x4341, 1152.0f),
                                 bytes_h2(x1 ^ 0x80008000u, 0x4341, 1152.0f), bytes_h2(y1 ^ 0x80008000u, 0x4341, 1152.0f), c[2 * q],
                                 c[2 * q + 1]);
                    }
                }
            }
            if (t < 2) {   // every column has the dot; lane t = 0 stores row g, t = 1 row g + 8
                const float l = t ? lo[0][2] + lo[1][2] : lo[0][0] + lo[1][0], h = t ? hi[0][2] + hi[1][2] : hi[0][0] + hi[1][0];
                s_dot[row + 8 * t] = sizeof(Code) == 1 ? l : fmaf(256.0f, h, l);
            }
        }
        // C . B_j of the window's tokens: 16 a warp, from the last warp on
        if (wid >= TC_WARPS - KB) {
            float d[4] = {};
            const uint32_t j0 = 16 * (TC_WARPS - 1 - wid) + g;
            const uint8_t* r0 = sm + sh.B + j0 * Sh::B_PITCH + 16 * t;
#pragma unroll
            for (int i = 0; i < N / 32; ++i) {
                const uint4 p0 = lds16(r0 + 64 * i), p1 = lds16(r0 + 8 * Sh::B_PITCH + 64 * i), c = lds16(sm + sh.C + 64 * i + 16 * t);
                mma16816(d, p0.x, p1.x, p0.y, p1.y, c.x, c.y);
                mma16816(d, p0.z, p1.z, p0.w, p1.w, c.z, c.w);
            }
            if (t == 0) { s_cb[j0] = d[0]; s_cb[j0 + 8] = d[2]; }
        }
        __syncthreads();
        // y: a thread a row
        if (tid < real) {
            const uint32_t hh = PAD ? 0 : head_of(tid);
            const __half* x = reinterpret_cast<const __half*>(sm + sh.x) + tid;
            const float* w = s_w[hh];
            float yw = 0.0f;
#pragma unroll
            for (uint32_t j0 = 0; j0 < 16 * KB; j0 += 4) {
                if (j0 >= count) break;   // a token behind the window's has weight 0 and x 0
                const float4 c4 = *reinterpret_cast<const float4*>(&s_cb[j0]), w4 = *reinterpret_cast<const float4*>(&w[j0]);
                const float cw[4] = {c4.x * w4.x, c4.y * w4.y, c4.z * w4.z, c4.w * w4.w};
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j)
                    yw = fmaf(cw[j], __half2float(*reinterpret_cast<const __half*>(reinterpret_cast<const uint8_t*>(x) + (j0 + j) * sh.x_pitch)), yw);
            }
            const __half xh = *reinterpret_cast<const __half*>(reinterpret_cast<const uint8_t*>(x) + n * sh.x_pitch);
            const __half yh = __float2half_rn(fmaf(s_alpha[hh] * my_scale, s_dot[tid], yw) + s_D[hh] * __half2float(xh));
            const uint32_t o = h0 * a.P + tid;
            a.y[b * a.y_bs + o] = a.z ? __float2half_rn(silu(__half2float(a.z[b * a.z_bs + o])) * __half2float(yh)) : yh;
            a.win_x[((uint64_t)b * a.W + n) * xrow + o] = xh;
        }
        // the first head of a group keeps the group's B row; every head takes row n from its argument
        if (PAD) {
            if (first == 0 && tid < n_real) wB[(uint64_t)n * brow + tid] = *reinterpret_cast<const __half*>(sm + sh.B + n * Sh::B_PITCH + tid * 2);
        } else if (first == 0 && tid < N / 8) {
            *reinterpret_cast<uint4*>(wB + (uint64_t)n * brow + 8 * tid) = lds16(sm + sh.B + n * Sh::B_PITCH + 16 * tid);
        }
        if (tid < nh) a.fill[bh0 + tid] = fold ? 0 : count;
        if (!fold) return;
    }
    float* s_as = reinterpret_cast<float*>(sm + sh.dot);   // alpha * scale of every row
    if (MODE == 0) __syncthreads();
    if (tid < rows) s_as[tid] = tid < real ? s_alpha[PAD ? 0 : head_of(tid)] * my_scale : 0.0f;
    __syncthreads();
    const uint32_t ldm = sm0 + sh.x + ((lane & 7) + (lane >> 4 & 1) * 8) * sh.x_pitch + (lane >> 3 & 1) * 16;
    for (uint32_t tile = wid; tile < rows / 16; tile += TC_WARPS) {
        const uint32_t row = tile * 16 + g, hh = PAD ? 0 : head_of(tile * 16), sw = Sh::swap(row);   // of row + 8, too
        const float as[2] = {s_as[row], s_as[row + 8]};
        // w_j x_j[p] of the lane's tokens: [0], [1] row g, tokens 2t, 2t + 1; [2], [3] row g + 8; [4] .. [7] tokens + 8
        float xw[KB * 8];
#pragma unroll
        for (int k = 0; k < KB; ++k) {
            uint32_t X[4] = {};
            if (MODE == 0 || count) ldmatrix_t(X, ldm + 16 * k * sh.x_pitch + tile * 32);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = __half22float2(bits_h2(X[i])), w = *reinterpret_cast<const float2*>(&s_w[hh][16 * k + 2 * t + 8 * (i >> 1)]);
                xw[8 * k + 2 * i] = w.x * f.x;
                xw[8 * k + 2 * i + 1] = w.y * f.y;
            }
        }
        // products of eight tokens: the first of a block of 16 has the lane's tokens 2t, 2t + 1, the second the other two
        uint32_t ah[2 * KB][4], al[2 * KB][4];
#pragma unroll
        for (int k = 0; k < 2 * KB; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) split2(xw[4 * k + 2 * (i & 1) + (i >> 1)], &ah[k][i], &al[k][i]);
        // elements 16 q + 4 t .. + 3 of the state, rows g and g + 8. Their codes: piece q (8 bits; 16 bits: 2 q + t / 2),
        // exchanged, so the address for q differs from the one for 0 in the bits of q alone
        const uint32_t in_piece = 4 * t * sizeof(Code), at0 = row * Sh::ROW + (((in_piece >> 4) ^ sw) << 4) + (in_piece & 15);
        auto word_at = [&](int q) { return at0 ^ (uint32_t)(q * 16 * sizeof(Code)); };
        const uint32_t* pair0 = &pairs[t][4 * (g >> 1) + 2 * (g & 1)];
        auto word = [&](int q, float (&s)[2][4]) {
            float cu[4], cv[4];
            const uint8_t* at = sm + word_at(q);
            code_values<Code>(at, cu);
            code_values<Code>(at + 8 * Sh::ROW, cv);
#pragma unroll
            for (int i = 0; i < 4; ++i) { s[0][i] = as[0] * cu[i]; s[1][i] = as[1] * cv[i]; }
            if (MODE == 1 && !count) return;
            // column c of a product is element 16 q + 4 (c / 2) + c % 2 + 2 half: a lane gets what its codes are. W <= 16
            // sums onto the codes' part (a load to fp16: 33.0 -> 31.1 us); beyond that it would spill.
            float d[2][4] = {};
            if constexpr (KB == 1) {
#pragma unroll
                for (int i = 0; i < 4; ++i) { d[i >> 1][i & 1] = s[0][i]; d[i >> 1][2 + (i & 1)] = s[1][i]; }
            }
#pragma unroll
            for (int k = 0; k < 2 * KB; k += 2) {
                const uint2 p0 = *reinterpret_cast<const uint2*>(pair0 + 4 * k * Sh::PAIR_PITCH + 16 * q);
                const uint2 p1 = *reinterpret_cast<const uint2*>(pair0 + 4 * (k + 1) * Sh::PAIR_PITCH + 16 * q);
                const uint32_t b[2][2] = {{p0.x, p0.y}, {p1.x, p1.y}};
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const float2 f = __half22float2(bits_h2(b[half][n]));
                        mma1688(d[n], ah[k + half], f.x, f.y);
                        mma1688(d[n], al[k + half], f.x, f.y);
                    }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[0][i] = KB == 1 ? d[i >> 1][i & 1] : s[0][i] + d[i >> 1][i & 1];
                s[1][i] = KB == 1 ? d[i >> 1][2 + (i & 1)] : s[1][i] + d[i >> 1][2 + (i & 1)];
            }
        };
        if constexpr (MODE == 1) {
            const uint64_t o0 = ((uint64_t)bh0 * a.P + row) * n_real + 4 * t;
            // padded rows and columns are left out; without them, stores of four where the state's rows allow it
            const bool wide = !PAD || wide_rows(a);
            auto pack16 = [&](const float (&v)[4]) {
                if (a.state_dtype == LSSM_DT_F16)
                    return make_uint2(h2_bits(__floats2half2_rn(v[0], v[1])), h2_bits(__floats2half2_rn(v[2], v[3])));
                const __nv_bfloat162 m0 = __floats2bfloat162_rn(v[0], v[1]), m1 = __floats2bfloat162_rn(v[2], v[3]);
                uint2 w;
                memcpy(&w.x, &m0, 4);
                memcpy(&w.y, &m1, 4);
                return w;
            };
            if (!PAD && a.state_dtype != LSSM_DT_F32) {
                // two words at a time: lanes t and t ^ 1 exchange, so that each stores 8 neighbours, the even one of q
                const bool odd = t & 1;
                uint16_t* out = static_cast<uint16_t*>(a.state) + o0 + (odd ? 12 : 0);
#pragma unroll
                for (int q = 0; q < N / 16; q += 2) {
                    float s0[2][4], s1[2][4];
                    word(q, s0);
                    word(q + 1, s1);
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const uint2 w0 = pack16(s0[r]), w1 = pack16(s1[r]);
                        const uint32_t x = __shfl_xor_sync(0xffffffffu, odd ? w0.x : w1.x, 1), y = __shfl_xor_sync(0xffffffffu, odd ? w0.y : w1.y, 1);
                        __stcs(reinterpret_cast<uint4*>(out + 8 * n_real * r + 16 * q),
                               odd ? make_uint4(x, y, w1.x, w1.y) : make_uint4(w0.x, w0.y, x, y));
                    }
                }
            } else if (PAD && staged_load(a)) {
                // 16 rows x 32 columns at a time through shared memory, so that a store instruction writes 32 neighbours
                // (16 x 64 heads of 75 x 203, 8 bits, to fp16: 59 -> 43 us when it came, 45 now; to fp32, whose stores of one element fill
                // more of a line, it costs 5 %)
                float(*stage)[STAGE_PITCH] = reinterpret_cast<float(*)[STAGE_PITCH]>(sm + sh.total) + 16 * wid;
                const uint64_t t0 = ((uint64_t)bh0 * a.P + tile * 16) * n_real;
                for (int q = 0; q < N / 16 && 16u * q < n_real; q += 2) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float s[2][4];
                        word(q + k, s);
#pragma unroll
                        for (int r = 0; r < 2; ++r)
                            *reinterpret_cast<float4*>(&stage[g + 8 * r][16 * k + 4 * t]) = make_float4(s[r][0], s[r][1], s[r][2], s[r][3]);
                    }
                    __syncwarp();
                    const uint32_t e = 16 * q + lane;
#pragma unroll
                    for (uint32_t r = 0; r < 16; ++r)
                        if (tile * 16 + r < real && e < n_real) store_any(a.state, t0 + r * n_real + e, a.state_dtype, stage[r][lane]);
                    __syncwarp();
                }
            } else
#pragma unroll
            for (int q = 0; q < N / 16; ++q) {
                float s[2][4];
                word(q, s);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint64_t o = o0 + 8 * n_real * r + 16 * q;
                    if (PAD && (row + 8 * r >= real || 16 * q + 4 * t >= n_real)) continue;
                    if (PAD && !wide) {
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i)
                            if (16 * q + 4 * t + i < n_real) store_any(a.state, o + i, a.state_dtype, s[r][i]);
                    } else if (a.state_dtype == LSSM_DT_F32)
                        __stcs(reinterpret_cast<float4*>(static_cast<float*>(a.state) + o), make_float4(s[r][0], s[r][1], s[r][2], s[r][3]));
                    else
                        __stcs(reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.state) + o), pack16(s[r]));
                }
            }
        } else {
            // The rows' largest elements first, then the codes: computed twice, once in W steps, so that no step
            // holds the registers for it.
            float amax[2] = {};
#pragma unroll
            for (int q = 0; q < N / 16; ++q) {
                float s[2][4];
                word(q, s);
#pragma unroll
                for (int i = 0; i < 8; ++i) amax[i / 4] = max_keep_nan(amax[i / 4], fabsf(s[i / 4][i % 4]));
            }
#pragma unroll
            for (int o = 1; o <= 2; o <<= 1)
#pragma unroll
                for (int r = 0; r < 2; ++r) amax[r] = max_keep_nan(amax[r], __shfl_xor_sync(0xffffffffu, amax[r], o));
            const RowQuant z0(amax[0], Q), z1(amax[1], Q);
#pragma unroll
            for (int q = 0; q < N / 16; ++q) {
                float s[2][4];
                word(q, s);
                uint8_t* at = sm + word_at(q);
                store_codes4(reinterpret_cast<Code*>(at), s[0], z0);
                store_codes4(reinterpret_cast<Code*>(at + 8 * Sh::ROW), s[1], z1);
            }
            if (t == 0) {
                if (!PAD || row < real) scales[row] = z0.scale;
                if (!PAD || row + 8 < real) scales[row + 8] = z1.scale;
            }
            __syncwarp();
            if constexpr (PAD) {
                for (uint32_t r = tile * 16; r < min(tile * 16 + 16, real); ++r)
                    for (uint32_t e = lane; e < n_real; e += 32) g_codes[r * n_real + e] = *reinterpret_cast<const Code*>(sm + code_at(r, e));
            } else for (uint32_t i = lane; i < 16 * Sh::PIECES; i += 32) {
                const uint32_t rr = tile * 16 + i / Sh::PIECES, q = i % Sh::PIECES;
                *reinterpret_cast<uint4*>(codes + rr * Sh::ROW + q * 16) = lds16(sm + Sh::piece(rr, q));
            }
        }
    }
}

template <typename Code, int MODE, int KB, int N, bool PAD>
cudaError_t launch_tc(const StateCacheArgs& a, cudaStream_t s) {
    // Heads of a group share the window's B and what is computed from it: as many as TC_BYTES of codes allow, fewer
    // where less than two CTAs an SM would be left. Steps without folds, with 1 / 2 / 4 heads a CTA of 64 x 128, W 16: 8 bits,
    // 80 heads, 64 sequences 28.9 / 20.1 / 17.1 us, 16 10.6 / 9.8 / 8.2, 2 4.5 / 4.9 / 6.1; all folding, 8 sequences 17.9 /
    // 14.4 / 17.3, 2 8.4 / 9.8 / 12.4. 16 bits (64 KB of codes for four), 64 sequences 32.9 / 25.5 / 27.7, all folding
    // 91.9 / 76.9 / 82.3. (One sequence in 16 folding, 64 sequences of 8 bits: 33.5 / 25.9 / 27.7, but the host does not
    // know which do, and a session's sequences fold together.)
    const uint32_t per_group = a.H / a.G;
    uint32_t heads = PAD ? 1 : TC_HEADS;
    while (heads > 1 && (heads * a.P > TC_THREADS || heads * a.P * N * sizeof(Code) > TC_BYTES ||
                         (uint64_t)a.batch * a.G * ((per_group + heads - 1) / heads) < 2ull * (uint32_t)a.sm_count)) heads /= 2;
    constexpr uint32_t STAGE = PAD && MODE == 1 ? TC_WARPS * 16 * STAGE_PITCH * 4 : 0;
    const uint32_t bytes = TcShared<Code, KB, N>(PAD ? (a.P + 15) / 16 * 16 : heads * a.P).total + (STAGE && staged_load(a) ? STAGE : 0);
    const auto kernel = k_state_tc<Code, MODE, KB, N, PAD>;
    if (bytes > 36 * 1024) {   // with the static part, more than 48 KB
        // The limit is the kernel's, for every thread of the process: set to what the largest call takes, so that no
        // thread's smaller call lowers it between another's set and launch.
        const int most = (int)(TcShared<Code, KB, N>(TC_THREADS).total + STAGE);
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != cudaSuccess) return e;
    }
    kernel<<<dim3((per_group + heads - 1) / heads, a.G, a.batch), TC_THREADS, bytes, s>>>(a, heads, per_group);
    return cudaGetLastError();
}
template <typename Code, int MODE, int N, bool PAD>
cudaError_t launch_tc_of(const StateCacheArgs& a, cudaStream_t s) {
    return a.W <= 16 ? launch_tc<Code, MODE, 1, N, PAD>(a, s) : launch_tc<Code, MODE, 2, N, PAD>(a, s);
}

template <typename Code, int MODE>
cudaError_t launch_cached(const StateCacheArgs& a, cudaStream_t s) {
    // a thread has a row
    if (a.P <= TC_THREADS && a.N <= 256 && a.G <= 65535 && a.batch <= 65535) {
        // such rows, and heads of 16 rows, keep the arrays' 16-byte alignment
        bool whole = a.P % 16 == 0 && aligned(a.codes, 16) && aligned(a.win_x, 16) && aligned(a.win_B, 16);
        if (MODE == 0) whole = whole && aligned(a.x, 16) && aligned(a.B, 16) && aligned(a.C, 16) && a.bc_bs % 8 == 0 && a.x_bs % 8 == 0;
        else whole = whole && aligned(a.state, 16);
        if (whole && a.N == 128) return launch_tc_of<Code, MODE, 128, false>(a, s);
        if (whole && a.N == 64) return launch_tc_of<Code, MODE, 64, false>(a, s);
        if (whole && a.N == 256) return launch_tc_of<Code, MODE, 256, false>(a, s);
        if (a.N <= 64) return launch_tc_of<Code, MODE, 64, true>(a, s);
        if (a.N <= 128) return launch_tc_of<Code, MODE, 128, true>(a, s);
        return launch_tc_of<Code, MODE, 256, true>(a, s);
    }
    if (a.W <= 16) k_state_any<Code, MODE, 1><<<a.batch * a.H, SC_THREADS, 0, s>>>(a);
    else k_state_any<Code, MODE, 2><<<a.batch * a.H, SC_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}

// N above 256: a warp a row, read twice (the second time from L2).
template <typename Code>
__global__ void __launch_bounds__(SC_THREADS) k_state_store(StateCacheArgs a) {
    constexpr float Q = sizeof(Code) == 1 ? 127.0f : 32767.0f;
    const uint32_t lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const uint64_t row = (uint64_t)blockIdx.x * (SC_THREADS / 32) + wid, rows = (uint64_t)a.batch * a.H * a.P;
    if (row >= rows) return;
    const float* S = static_cast<const float*>(a.state) + row * a.N;
    Code* out = static_cast<Code*>(a.codes) + row * a.N;
    // the bits of |v| order as the values do, NaN above infinity
    uint32_t top = 0;
#pragma unroll 8
    for (uint32_t i = lane; i < a.N; i += 32) top = max(top, __float_as_uint(S[i]) & 0x7FFFFFFFu);
    const RowQuant z(__uint_as_float(__reduce_max_sync(0xffffffffu, top)), Q);
#pragma unroll 4
    for (uint32_t i = lane; i < a.N; i += 32) out[i] = quantise1<Code>(S[i], z);
    if (lane == 0) {
        a.scales[row] = z.scale;
        if (row % a.P == 0) a.fill[row / a.P] = 0;
    }
}

// Rounding a state into codes: one read, one write, bound by HBM: 64 sequences x 80 heads of 64 x 128, 8 bits, 36 us for
// 210 MB = 5.8 TB/s, 88 % of a copy's rate.
// N up to 256: a warp takes ROWS rows, a lane PER elements of each in registers: VEC neighbours at a time (VEC 4: N a
// multiple of 4 and the arrays aligned for it), runs of 32 * VEC. Lane r works out row r's scale. The largest magnitude
// is found on the bits of |v|, which order as the values do, with NaN above infinity.
template <typename Code, int ROWS, int PER, int VEC>
__global__ void __launch_bounds__(SC_THREADS) k_state_store_rows(StateCacheArgs a) {
    constexpr float Q = sizeof(Code) == 1 ? 127.0f : 32767.0f;
    const uint32_t lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const uint64_t row0 = ((uint64_t)blockIdx.x * (SC_THREADS / 32) + wid) * ROWS, rows = (uint64_t)a.batch * a.H * a.P;
    if (row0 >= rows) return;
    const uint32_t here = (uint32_t)(rows - row0 < ROWS ? rows - row0 : ROWS);
    const float* S = static_cast<const float*>(a.state) + row0 * a.N;
    Code* out = static_cast<Code*>(a.codes) + row0 * a.N;
    float v[ROWS][PER];
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int k = 0; k < PER; k += VEC) {
            const uint32_t e = k * 32 + lane * VEC;
            const bool in = r < (int)here && e < a.N;
            if constexpr (VEC == 4) {
                const float4 f = in ? __ldcs(reinterpret_cast<const float4*>(S + r * a.N + e)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                v[r][k] = f.x; v[r][k + 1] = f.y; v[r][k + 2] = f.z; v[r][k + 3] = f.w;
            } else v[r][k] = in ? __ldcs(S + r * a.N + e) : 0.0f;
        }
    uint32_t mine = 0;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k) top = max(top, __float_as_uint(v[r][k]) & 0x7FFFFFFFu);
        top = __reduce_max_sync(0xffffffffu, top);
        if ((int)lane == r) mine = top;
    }
    const RowQuant own(__uint_as_float(mine), Q);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const RowQuant z = own.of_lane(r);
#pragma unroll
        for (int k = 0; k < PER; k += 4) {
            const float four[4] = {v[r][k], v[r][k + 1], v[r][k + 2], v[r][k + 3]};
            if constexpr (VEC == 4) {
                const uint32_t e = k * 32 + lane * 4;
                if (r < (int)here && e < a.N) store_codes4(out + r * a.N + e, four, z);
            } else {
                uint32_t c[4];
                quantise4(four, z, c);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t e = (k + i) * 32 + lane;
                    if (r < (int)here && e < a.N) out[r * a.N + e] = z.sound ? (Code)c[i] : (Code)0;
                }
            }
        }
    }
    if (lane < here) {
        a.scales[row0 + lane] = own.scale;
        if ((row0 + lane) % a.P == 0) a.fill[(row0 + lane) / a.P] = 0;
    }
}
template <typename Code, int ROWS, int PER>
void launch_store_rows(const StateCacheArgs& a, uint64_t rows, cudaStream_t s) {
    constexpr uint64_t EACH = SC_THREADS / 32 * ROWS;
    const unsigned grid = (unsigned)((rows + EACH - 1) / EACH);
    if (a.N % 4 == 0 && aligned(a.state, 16) && aligned(a.codes, 4 * sizeof(Code))) k_state_store_rows<Code, ROWS, PER, 4><<<grid, SC_THREADS, 0, s>>>(a);
    else k_state_store_rows<Code, ROWS, PER, 1><<<grid, SC_THREADS, 0, s>>>(a);
}
template <typename Code>
cudaError_t launch_store_of(const StateCacheArgs& a, uint64_t rows, cudaStream_t s) {
    // 32 elements a lane in flight
    if (a.N <= 128) launch_store_rows<Code, 8, 4>(a, rows, s);
    else if (a.N <= 256) launch_store_rows<Code, 4, 8>(a, rows, s);
    else k_state_store<Code><<<(unsigned)((rows + SC_THREADS / 32 - 1) / (SC_THREADS / 32)), SC_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_state_store(const StateCacheArgs& a, cudaStream_t s) {
    const uint64_t rows = (uint64_t)a.batch * a.H * a.P;
    if (!rows || !a.N) return cudaSuccess;
    return a.bits == 8 ? launch_store_of<int8_t>(a, rows, s) : launch_store_of<int16_t>(a, rows, s);
}

cudaError_t launch_state_load(const StateCacheArgs& a, cudaStream_t s) {
    if (!a.batch || !a.H || !a.P || !a.N) return cudaSuccess;
    return a.bits == 8 ? launch_cached<int8_t, 1>(a, s) : launch_cached<int16_t, 1>(a, s);
}

cudaError_t launch_ssd_step_cached(const StateCacheArgs& a, cudaStream_t s) {
    if (!a.batch || !a.H || !a.P || !a.N) return cudaSuccess;
    return a.bits == 8 ? launch_cached<int8_t, 0>(a, s) : launch_cached<int16_t, 0>(a, s);
}

}  // namespace lssm
