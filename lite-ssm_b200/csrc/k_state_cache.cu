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

// The nearest code to v / scale. The product with the reciprocal may land on the wrong side of a
// half step; the remainder v - q * scale, exact in one fma, decides.
__device__ __forceinline__ int nearest_code(float v, float scale, float inv, float Q) {
    if (!(scale > 0.0f)) return 0;   // zero row, or NaN scale
    float q = fminf(fmaxf(rintf(v * inv), -Q), Q);
    const float r = fmaf(-q, scale, v), half = 0.5f * scale;
    if (fabsf(r) > half) q += r > 0.0f ? 1.0f : -1.0f;
    else if (fabsf(r) == half && ((int)q & 1)) q += r > 0.0f ? 1.0f : -1.0f;
    return (int)fminf(fmaxf(q, -Q), Q);
}
__device__ __forceinline__ float row_scale(float amax, float Q) {
    const float s = __fdiv_rn(amax, Q);
    if (!(amax < INFINITY)) return __int_as_float(0x7FC00000);
    return s < kTiny ? 0.0f : s;
}
// max|.| that keeps NaN
__device__ __forceinline__ float max_nan(float a, float b) { return a != a || b != b ? __int_as_float(0x7FC00000) : fmaxf(a, b); }
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Window weights of one head, lane j of a warp for token j (W <= 32): the sum over later tokens
// is taken from the end, so one very large dt costs the tokens after it no digits.
__device__ __forceinline__ void window_weights(float a, float dt, uint32_t lane, uint32_t count, float* w, float* alpha) {
    if (lane >= count) dt = 0.0f;
    float s = a * dt;
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

// General shapes: one CTA per (sequence, head), a warp per row of N.
// MODE 0: step (y, window append, requantise when full); MODE 1: load (the state as it stands).
template <typename Code, int MODE>
__global__ void __launch_bounds__(SC_THREADS) k_state_cached(StateCacheArgs a) {
    __shared__ float w[LSSM_STATE_WINDOW_MAX];
    __shared__ float s_alpha;
    const uint32_t h = blockIdx.x % a.H, b = blockIdx.x / a.H, g = h / (a.H / a.G);
    const uint32_t lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const uint64_t bh = (uint64_t)b * a.H + h;
    constexpr float Q = sizeof(Code) == 1 ? 127.0f : 32767.0f;
    uint32_t n = a.fill[bh];
    if (MODE == 0) n = n < a.W ? n : a.W - 1;
    const uint32_t count = MODE == 0 ? n + 1 : (n < a.W ? n : a.W);
    if (wid == 0) {
        const float rate = -expf(__half2float(a.A_log[h]));
        float dt = 0.0f;
        if (lane < count) dt = a.win_dt[bh * a.W + lane];
        if (MODE == 0 && lane == n)
            dt = token_dt(__half2float(a.dt_raw[b * a.dt_bs + h]) + __half2float(a.dt_bias[h]), a.dt_min, a.dt_max);
        float wj, al;
        window_weights(rate, dt, lane, count, &wj, &al);
        w[lane] = wj;
        if (lane == 0) s_alpha = al;
        if (MODE == 0 && lane == n) a.win_dt[bh * a.W + n] = dt;
    }
    __syncthreads();
    const float alpha = s_alpha;
    const uint64_t xrow = (uint64_t)a.H * a.P, brow = (uint64_t)a.G * a.N;
    const __half* wx = a.win_x + (uint64_t)b * a.W * xrow + (uint64_t)h * a.P;
    const __half* wB = a.win_B + (uint64_t)b * a.W * brow + (uint64_t)g * a.N;
    const __half* xn = MODE == 0 ? a.x + b * a.x_bs + (uint64_t)h * a.P : nullptr;
    const __half* Bn = MODE == 0 ? a.B + b * a.bc_bs + (uint64_t)g * a.N : nullptr;
    const __half* Cn = MODE == 0 ? a.C + b * a.bc_bs + (uint64_t)g * a.N : nullptr;
    const bool fold = MODE == 0 && n + 1 == a.W;
    for (uint32_t p = wid; p < a.P; p += SC_THREADS / 32) {
        Code* row = static_cast<Code*>(a.codes) + (bh * a.P + p) * a.N;
        const float as = alpha * a.scales[bh * a.P + p];
        // x of every window token of this row, scaled: lane j holds token j
        float xw = 0.0f;
        if (lane < count) xw = w[lane] * __half2float(MODE == 0 && lane == n ? xn[p] : wx[lane * xrow + p]);
        auto state = [&](uint32_t i, bool in) {
            float v = in ? as * (float)row[i] : 0.0f;
            for (uint32_t j = 0; j < count; ++j) {
                const float xj = __shfl_sync(0xffffffffu, xw, j);
                if (in) v = fmaf(xj, __half2float(MODE == 0 && j == n ? Bn[i] : wB[j * brow + i]), v);
            }
            return v;
        };
        float acc = 0.0f, amax = 0.0f;
        for (uint32_t i0 = 0; i0 < a.N; i0 += 32) {
            const uint32_t i = i0 + lane;
            const bool in = i < a.N;
            const float v = state(i, in);
            if (MODE == 1) {
                if (in) store_any(a.state, (bh * a.P + p) * a.N + i, a.state_dtype, v);
            } else if (in) {
                acc = fmaf(v, __half2float(Cn[i]), acc);
                amax = max_nan(amax, fabsf(v));
            }
        }
        if (MODE == 0) {
            acc = warp_sum(acc);
            if (lane == 0) {
                const float xv = __half2float(xn[p]);
                const float Dh = a.has_D ? __half2float(a.D[h]) : 0.0f;
                const __half yh = __float2half_rn(acc + Dh * xv);
                const uint64_t o = (uint64_t)h * a.P + p;
                a.y[b * a.y_bs + o] =
                    a.z ? __float2half_rn(silu(__half2float(a.z[b * a.z_bs + o])) * __half2float(yh)) : yh;
                a.win_x[((uint64_t)b * a.W + n) * xrow + o] = xn[p];
            }
            if (fold) {
                const float scale = row_scale(warp_max_nan(amax), Q), inv = scale > 0.0f ? 1.0f / scale : 0.0f;
                for (uint32_t i0 = 0; i0 < a.N; i0 += 32) {
                    const uint32_t i = i0 + lane;
                    const float v = state(i, i < a.N);
                    if (i < a.N) row[i] = (Code)nearest_code(v, scale, inv, Q);
                }
                if (lane == 0) a.scales[bh * a.P + p] = scale;
            }
        }
    }
    if (MODE == 0) {
        // the first head of a group keeps the group's B row; every head takes row n from its argument
        if (h % (a.H / a.G) == 0)
            for (uint32_t i = threadIdx.x; i < a.N; i += SC_THREADS)
                a.win_B[((uint64_t)b * a.W + n) * brow + (uint64_t)g * a.N + i] = Bn[i];
        if (threadIdx.x == 0) a.fill[bh] = fold ? 0 : n + 1;
    }
}

// ---------------------------------------------------------------------------
//  N = 128, P a multiple of 16: tensor-core kernel
// ---------------------------------------------------------------------------
// A CTA per (sequence, head); a warp takes 16 rows of the state at a time. With m16n8k16 (f16 in, f32 out), lane
// (g, t) = (lane / 4, lane % 4), and an order of k that lets a lane load its codes as they lie:
//   S_q C       A = codes (exact in f16: 8 bits as they are, 16 bits as 256 * high + low), B = C in every column
//   C . B_j     A = the window's B rows, B = C in every column (one warp; 16 tokens an instruction)
//   sum_j w_j x_j B_j^T (fold, load)   A = w_j x_j[p] as two f16 terms (22 bits), scaled by a power of two that puts
//               the largest at 2^14, B = the window's B; a lane gets the elements whose codes it holds.
// A code is converted, multiplied and added in about one instruction for 30 elements, so the step is bound by the
// codes' bytes and the latency of a short CTA.
constexpr int TC_THREADS = 128, TC_N = 128;
// Element order: lane t's word q (4 codes) is elements k0 .. k0 + 3. Steps load 16 bytes a lane; loads write 16 bytes
// of fp32 a lane, with 4 neighbours in 4 lanes.
template <typename Code, int MODE>
__device__ __forceinline__ constexpr int tc_k0(int q, int t) {
    return MODE == 1 ? 16 * q + 4 * t : sizeof(Code) == 1 ? 64 * (q / 4) + 16 * t + 4 * (q % 4) : 32 * (q / 2) + 8 * t + 4 * (q % 2);
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { uint32_t u; memcpy(&u, &h, 4); return u; }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { __half2 h; memcpy(&h, &u, 4); return h; }
// Two unsigned bytes of w (chosen by sel, the 0x64 bytes from the constant) as f16 minus `off`: exact, 1024 + byte is.
__device__ __forceinline__ uint32_t bytes_h2(uint32_t w, uint32_t sel, float off) {
    return h2_bits(__hsub2(bits_h2(__byte_perm(w, 0x64646464u, sel)), __float2half2_rn(off)));
}

// The codes of one row that a lane holds: 8 words of 4.
template <typename Code>
struct RowCodes {
    static constexpr int REGS = 8 * sizeof(Code);
    uint32_t r[REGS];
    template <int MODE>
    __device__ __forceinline__ void load(const Code* row, int t) {
        if constexpr (MODE == 1) {
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                if constexpr (sizeof(Code) == 1) r[q] = *reinterpret_cast<const uint32_t*>(row + tc_k0<Code, 1>(q, t));
                else {
                    const uint2 v = *reinterpret_cast<const uint2*>(row + tc_k0<Code, 1>(q, t));
                    r[2 * q] = v.x; r[2 * q + 1] = v.y;
                }
            }
        } else {
            constexpr int PER = 16 / sizeof(Code);   // codes a load
#pragma unroll
            for (int i = 0; i < REGS / 4; ++i) {
                const uint4 v = *reinterpret_cast<const uint4*>(row + tc_k0<Code, 0>(i * PER / 4, t));
                r[4 * i] = v.x; r[4 * i + 1] = v.y; r[4 * i + 2] = v.z; r[4 * i + 3] = v.w;
            }
        }
    }
    __device__ __forceinline__ void store(Code* row, int t) const {
        constexpr int PER = 16 / sizeof(Code);
#pragma unroll
        for (int i = 0; i < REGS / 4; ++i)
            *reinterpret_cast<uint4*>(row + tc_k0<Code, 0>(i * PER / 4, t)) = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
    }
    // word q as fp32
    __device__ __forceinline__ void values(int q, float (&v)[4]) const {
        if constexpr (sizeof(Code) == 1) {
            const uint32_t w = r[q] ^ 0x80808080u;
            const float2 a = __half22float2(bits_h2(bytes_h2(w, 0x4140, 1152.0f)));
            const float2 b = __half22float2(bits_h2(bytes_h2(w, 0x4342, 1152.0f)));
            v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
        } else {
            v[0] = (float)(int16_t)(r[2 * q] & 0xFFFF); v[1] = (float)((int32_t)r[2 * q] >> 16);
            v[2] = (float)(int16_t)(r[2 * q + 1] & 0xFFFF); v[3] = (float)((int32_t)r[2 * q + 1] >> 16);
        }
    }
    __device__ __forceinline__ void set(int q, const int (&c)[4]) {
        if constexpr (sizeof(Code) == 1)
            r[q] = (c[0] & 0xFF) | (c[1] & 0xFF) << 8 | (c[2] & 0xFF) << 16 | (uint32_t)c[3] << 24;
        else {
            r[2 * q] = (c[0] & 0xFFFF) | (uint32_t)c[1] << 16;
            r[2 * q + 1] = (c[2] & 0xFFFF) | (uint32_t)c[3] << 16;
        }
    }
};

// acc[0], acc[2] += codes . C of rows g and g + 8
template <typename Code>
__device__ __forceinline__ void codes_dot_c(const RowCodes<Code>& u, const RowCodes<Code>& v, const uint32_t (&c)[16], float (&y)[2]) {
    float lo[4] = {}, hi[4] = {};
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        if constexpr (sizeof(Code) == 1) {
            const uint32_t a = u.r[q] ^ 0x80808080u, b = v.r[q] ^ 0x80808080u;
            mma16816(lo, bytes_h2(a, 0x4140, 1152.0f), bytes_h2(b, 0x4140, 1152.0f), bytes_h2(a, 0x4342, 1152.0f),
                     bytes_h2(b, 0x4342, 1152.0f), c[2 * q], c[2 * q + 1]);
        } else {
            const uint32_t a0 = u.r[2 * q], a1 = u.r[2 * q + 1], b0 = v.r[2 * q], b1 = v.r[2 * q + 1];
            mma16816(lo, bytes_h2(a0, 0x4240, 1024.0f), bytes_h2(b0, 0x4240, 1024.0f), bytes_h2(a1, 0x4240, 1024.0f),
                     bytes_h2(b1, 0x4240, 1024.0f), c[2 * q], c[2 * q + 1]);
            mma16816(hi, bytes_h2(a0 ^ 0x80008000u, 0x4341, 1152.0f), bytes_h2(b0 ^ 0x80008000u, 0x4341, 1152.0f),
                     bytes_h2(a1 ^ 0x80008000u, 0x4341, 1152.0f), bytes_h2(b1 ^ 0x80008000u, 0x4341, 1152.0f), c[2 * q], c[2 * q + 1]);
        }
    }
    y[0] = sizeof(Code) == 1 ? lo[0] : fmaf(256.0f, hi[0], lo[0]);
    y[1] = sizeof(Code) == 1 ? lo[2] : fmaf(256.0f, hi[2], lo[2]);
}

__device__ __forceinline__ float max_keep_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// KB: blocks of 16 window tokens (W <= 16 * KB).
template <typename Code, int MODE, int KB>
__global__ void __launch_bounds__(TC_THREADS) k_state_tc(StateCacheArgs a) {
    constexpr float Q = sizeof(Code) == 1 ? 127.0f : 32767.0f;
    constexpr int PITCH = MODE == 1 ? TC_N + 16 : TC_N + 4;   // spreads the lanes' rows over the banks
    __shared__ float s_w[32], s_cb[32], s_alpha;
    __shared__ uint32_t s_B[KB * 8][PITCH];   // tokens 2 jp and 2 jp + 1 of the window, side by side
    const uint32_t h = blockIdx.x % a.H, b = blockIdx.x / a.H, g0 = h / (a.H / a.G);
    const uint32_t tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, g = lane >> 2, t = lane & 3;
    const uint64_t bh = (uint64_t)b * a.H + h;
    const uint64_t xrow = (uint64_t)a.H * a.P, brow = (uint64_t)a.G * TC_N;
    Code* codes = static_cast<Code*>(a.codes) + bh * a.P * TC_N;
    const uint32_t tiles = a.P / 16;
    const uint32_t filled = a.fill[bh];
    RowCodes<Code> u, v;
    float sc[2];
    uint32_t tile = wid;
    auto fetch = [&] {
        u.template load<MODE>(codes + (uint64_t)(tile * 16 + g) * TC_N, t);
        v.template load<MODE>(codes + (uint64_t)(tile * 16 + g + 8) * TC_N, t);
        sc[0] = a.scales[bh * a.P + tile * 16 + g];
        sc[1] = a.scales[bh * a.P + tile * 16 + g + 8];
    };
    if (tile < tiles) fetch();
    const __half* wx = a.win_x + (uint64_t)b * a.W * xrow + (uint64_t)h * a.P;
    __half* wB = a.win_B + (uint64_t)b * a.W * brow + (uint64_t)g0 * TC_N;
    const __half* xn = MODE == 0 ? a.x + b * a.x_bs + (uint64_t)h * a.P : nullptr;
    const __half* Bn = MODE == 0 ? a.B + b * a.bc_bs + (uint64_t)g0 * TC_N : nullptr;
    const __half* Cn = MODE == 0 ? a.C + b * a.bc_bs + (uint64_t)g0 * TC_N : nullptr;
    // the step's token is number n of the window; `count` tokens with it
    const uint32_t n = MODE == 0 ? min(filled, a.W - 1) : a.W, count = MODE == 0 ? n + 1 : min(filled, a.W);
    const bool fold = MODE == 0 && count == a.W;
    if (wid == 3) {
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
    if (MODE == 0 && wid < KB) {
        // C . B_j for tokens 16 wid + g and + g + 8; a row beyond the window's tokens is not read
        float cb[4] = {};
        const uint32_t j0 = 16 * wid + g, j1 = j0 + 8;
        const __half* r0 = j0 == n ? Bn : wB + j0 * brow;
        const __half* r1 = j1 == n ? Bn : wB + j1 * brow;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 z = make_uint4(0, 0, 0, 0);
            const uint4 p0 = j0 < count ? *reinterpret_cast<const uint4*>(r0 + 32 * i + 8 * t) : z;
            const uint4 p1 = j1 < count ? *reinterpret_cast<const uint4*>(r1 + 32 * i + 8 * t) : z;
            const uint4 c = *reinterpret_cast<const uint4*>(Cn + 32 * i + 8 * t);
            mma16816(cb, p0.x, p1.x, p0.y, p1.y, c.x, c.y);
            mma16816(cb, p0.z, p1.z, p0.w, p1.w, c.z, c.w);
        }
        if (t == 0) { s_cb[j0] = cb[0]; s_cb[j1] = cb[2]; }
    }
    if (MODE == 1 || fold) {
        // the window's B, two tokens a word: 8 KB rows of TC_N words
        for (uint32_t i = tid; i < KB * 8 * (TC_N / 2); i += TC_THREADS) {
            const uint32_t jp = i / (TC_N / 2), e = i % (TC_N / 2) * 2, j0 = 2 * jp, j1 = j0 + 1;
            uint32_t p0 = 0, p1 = 0;
            if (j0 < count) p0 = *reinterpret_cast<const uint32_t*>((MODE == 0 && j0 == n ? Bn : wB + j0 * brow) + e);
            if (j1 < count) p1 = *reinterpret_cast<const uint32_t*>((MODE == 0 && j1 == n ? Bn : wB + j1 * brow) + e);
            s_B[jp][e] = __byte_perm(p0, p1, 0x5410);
            s_B[jp][e + 1] = __byte_perm(p0, p1, 0x7632);
        }
    }
    uint32_t c[16];
    if (MODE == 0) {
        constexpr int PER = 16 / sizeof(Code);
#pragma unroll
        for (int i = 0; i < (int)(8 * sizeof(Code) / 4); ++i)
#pragma unroll
            for (int k = 0; k < PER / 8; ++k) {
                const uint4 w = *reinterpret_cast<const uint4*>(Cn + tc_k0<Code, 0>(i * PER / 4, t) + 8 * k);
                const int o = i * PER / 2 + 4 * k;
                c[o] = w.x; c[o + 1] = w.y; c[o + 2] = w.z; c[o + 3] = w.w;
            }
    }
    __syncthreads();
    const float alpha = s_alpha;
    for (; tile < tiles; tile += TC_THREADS / 32) {
        if (tile != wid) fetch();
        const uint32_t p0 = tile * 16 + g;
        // w_j x_j[p] of this lane's tokens 16 k + {2t, 2t + 1, 2t + 8, 2t + 9}, rows g and g + 8
        float xw[KB][4][2], ywin[2] = {};
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t j = 16 * k + 2 * t + (i & 1) + 8 * (i >> 1);
                const __half* xj = MODE == 0 && j == n ? xn : wx + j * xrow;
                const float wj = s_w[j];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float x = j < count ? __half2float(xj[p0 + 8 * r]) : 0.0f;
                    xw[k][i][r] = wj * x;
                    if (MODE == 0 && j < count) ywin[r] = fmaf(s_cb[j], xw[k][i][r], ywin[r]);
                }
            }
        if (MODE == 0) {
            float y[2];
            codes_dot_c(u, v, c, y);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                ywin[r] += __shfl_xor_sync(0xffffffffu, ywin[r], 1);
                ywin[r] += __shfl_xor_sync(0xffffffffu, ywin[r], 2);
                if (t == r) {
                    const uint64_t o = (uint64_t)h * a.P + p0 + 8 * r;
                    const __half xh = xn[p0 + 8 * r];
                    const float Dh = a.has_D ? __half2float(a.D[h]) : 0.0f;
                    const __half yh = __float2half_rn(fmaf(alpha * sc[r], y[r], ywin[r]) + Dh * __half2float(xh));
                    a.y[b * a.y_bs + o] =
                        a.z ? __float2half_rn(silu(__half2float(a.z[b * a.z_bs + o])) * __half2float(yh)) : yh;
                    a.win_x[((uint64_t)b * a.W + n) * xrow + o] = xh;
                }
            }
            if (!fold) continue;
        }
        // the window's part of the state. Terms that are not finite set no scale, and come out as they are.
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t bits = __float_as_uint(xw[k][i / 2][i % 2]) & 0x7FFFFFFFu;
                if (bits < 0x7F800000u) top = max(top, bits);
            }
        const uint32_t eb = max(__reduce_max_sync(0xffffffffu, top) >> 23, 15u);
        const float up = __uint_as_float(min(268u - eb, 254u) << 23), down = __uint_as_float((eb - 14u) << 23);
        uint32_t ah[KB][4], al[KB][4];
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // a0 (g; 2t, 2t + 1), a1 (g + 8; same), a2 (g; 2t + 8, + 9), a3 (g + 8; same)
                const int r = i & 1, at = i & 2;
                const float x0 = xw[k][at][r] * up, x1 = xw[k][at + 1][r] * up;
                const __half2 hh = __floats2half2_rn(x0, x1);
                const float2 f = __half22float2(hh);
                ah[k][i] = h2_bits(hh);
                al[k][i] = h2_bits(__floats2half2_rn(x0 - f.x, x1 - f.y));
            }
        const float as0 = alpha * sc[0], as1 = alpha * sc[1];
        // word q of the state, rows g and g + 8
        auto word = [&](int q, float (&s)[2][4]) {
            float cu[4], cv[4];
            u.values(q, cu);
            v.values(q, cv);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float d[4] = {};
                const int e = tc_k0<Code, MODE>(q, g >> 1) + (g & 1) + 2 * half;
#pragma unroll
                for (int k = 0; k < KB; ++k) {
                    const uint32_t b0 = s_B[8 * k + t][e], b1 = s_B[8 * k + t + 4][e];
                    mma16816(d, ah[k][0], ah[k][1], ah[k][2], ah[k][3], b0, b1);
                    mma16816(d, al[k][0], al[k][1], al[k][2], al[k][3], b0, b1);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    s[0][2 * half + i] = fmaf(d[i], down, as0 * cu[2 * half + i]);
                    s[1][2 * half + i] = fmaf(d[2 + i], down, as1 * cv[2 * half + i]);
                }
            }
        };
        if constexpr (MODE == 1) {
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                float s[2][4];
                word(q, s);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint64_t o = (bh * a.P + p0 + 8 * r) * TC_N + tc_k0<Code, 1>(q, t);
                    if (a.state_dtype == LSSM_DT_F32)
                        __stcs(reinterpret_cast<float4*>(static_cast<float*>(a.state) + o), make_float4(s[r][0], s[r][1], s[r][2], s[r][3]));
                    else {
                        uint2 w;
                        if (a.state_dtype == LSSM_DT_F16)
                            w = make_uint2(h2_bits(__floats2half2_rn(s[r][0], s[r][1])), h2_bits(__floats2half2_rn(s[r][2], s[r][3])));
                        else {
                            const __nv_bfloat162 m0 = __floats2bfloat162_rn(s[r][0], s[r][1]), m1 = __floats2bfloat162_rn(s[r][2], s[r][3]);
                            memcpy(&w.x, &m0, 4);
                            memcpy(&w.y, &m1, 4);
                        }
                        __stcs(reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.state) + o), w);
                    }
                }
            }
        } else {
            // the rows' largest elements first, then the codes: computed twice, once in W steps, instead of
            // held in 64 registers at every step
            float amax0 = 0.0f, amax1 = 0.0f;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                float s[2][4];
                word(q, s);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    amax0 = max_keep_nan(amax0, fabsf(s[0][i]));
                    amax1 = max_keep_nan(amax1, fabsf(s[1][i]));
                }
            }
#pragma unroll
            for (int o = 1; o <= 2; o <<= 1) {
                amax0 = max_keep_nan(amax0, __shfl_xor_sync(0xffffffffu, amax0, o));
                amax1 = max_keep_nan(amax1, __shfl_xor_sync(0xffffffffu, amax1, o));
            }
            const float n0 = row_scale(amax0, Q), n1 = row_scale(amax1, Q);
            const float i0 = n0 > 0.0f ? 1.0f / n0 : 0.0f, i1 = n1 > 0.0f ? 1.0f / n1 : 0.0f;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                float s[2][4];
                int c0[4], c1[4];
                word(q, s);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    c0[i] = nearest_code(s[0][i], n0, i0, Q);
                    c1[i] = nearest_code(s[1][i], n1, i1, Q);
                }
                u.set(q, c0);
                v.set(q, c1);
            }
            u.store(codes + (uint64_t)p0 * TC_N, t);
            v.store(codes + (uint64_t)(p0 + 8) * TC_N, t);
            if (t == 0) {
                a.scales[bh * a.P + p0] = n0;
                a.scales[bh * a.P + p0 + 8] = n1;
            }
        }
    }
    if (MODE == 0) {
        // the first head of a group keeps the group's B row; every head takes row n from its argument
        if (h % (a.H / a.G) == 0 && tid < TC_N / 8)
            *reinterpret_cast<uint4*>(wB + n * brow + 8 * tid) = *reinterpret_cast<const uint4*>(Bn + 8 * tid);
        if (tid == 0) a.fill[bh] = fold ? 0 : n + 1;
    }
}

template <typename Code, int MODE>
cudaError_t launch_cached(const StateCacheArgs& a, cudaStream_t s) {
    const unsigned grid = a.batch * a.H;
    // 16-byte loads of codes, B and C, 8- or 16-byte stores of the state: rows of 128 keep the base's alignment
    bool tc = a.N == TC_N && a.P % 16 == 0 && aligned(a.codes, 16) && aligned(a.win_B, 16);
    if (MODE == 0) tc = tc && aligned(a.B, 16) && aligned(a.C, 16) && a.bc_bs % 8 == 0;
    else tc = tc && aligned(a.state, 16);
    if (tc && a.W <= 16) k_state_tc<Code, MODE, 1><<<grid, TC_THREADS, 0, s>>>(a);
    else if (tc) k_state_tc<Code, MODE, 2><<<grid, TC_THREADS, 0, s>>>(a);
    else k_state_cached<Code, MODE><<<grid, SC_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}

template <typename Code>
__global__ void __launch_bounds__(SC_THREADS) k_state_store(StateCacheArgs a) {
    constexpr float Q = sizeof(Code) == 1 ? 127.0f : 32767.0f;
    const uint32_t lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const uint64_t row = (uint64_t)blockIdx.x * (SC_THREADS / 32) + wid, rows = (uint64_t)a.batch * a.H * a.P;
    if (row >= rows) return;
    const float* S = static_cast<const float*>(a.state) + row * a.N;
    Code* out = static_cast<Code*>(a.codes) + row * a.N;
    float amax = 0.0f;
    for (uint32_t i = lane; i < a.N; i += 32) amax = max_nan(amax, fabsf(S[i]));
    const float scale = row_scale(warp_max_nan(amax), Q), inv = scale > 0.0f ? 1.0f / scale : 0.0f;
    for (uint32_t i = lane; i < a.N; i += 32) out[i] = (Code)nearest_code(S[i], scale, inv, Q);
    if (lane == 0) {
        a.scales[row] = scale;
        if (row % a.P == 0) a.fill[row / a.P] = 0;
    }
}

// N = 128: a warp takes STORE_ROWS rows, a lane four neighbours of each. The largest magnitude is found on the
// bits of |v|, which order as the values do, with NaN above infinity.
constexpr int STORE_ROWS = 8;
template <typename Code>
__global__ void __launch_bounds__(SC_THREADS) k_state_store128(StateCacheArgs a) {
    constexpr float Q = sizeof(Code) == 1 ? 127.0f : 32767.0f;
    const uint32_t lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const uint64_t row0 = ((uint64_t)blockIdx.x * (SC_THREADS / 32) + wid) * STORE_ROWS, rows = (uint64_t)a.batch * a.H * a.P;
    const float* S = static_cast<const float*>(a.state) + row0 * 128 + 4 * lane;
    Code* out = static_cast<Code*>(a.codes) + row0 * 128 + 4 * lane;
    float4 v[STORE_ROWS];
#pragma unroll
    for (int r = 0; r < STORE_ROWS; ++r)
        if (row0 + r < rows) v[r] = __ldcs(reinterpret_cast<const float4*>(S + r * 128));
#pragma unroll
    for (int r = 0; r < STORE_ROWS; ++r) {
        if (row0 + r >= rows) break;
        const float e[4] = {v[r].x, v[r].y, v[r].z, v[r].w};
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(e[i]) & 0x7FFFFFFFu);
        const float scale = row_scale(__uint_as_float(__reduce_max_sync(0xffffffffu, top)), Q);
        const float inv = scale > 0.0f ? 1.0f / scale : 0.0f;
        int c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = nearest_code(e[i], scale, inv, Q);
        if constexpr (sizeof(Code) == 1)
            *reinterpret_cast<uint32_t*>(out + r * 128) = (c[0] & 0xFF) | (c[1] & 0xFF) << 8 | (c[2] & 0xFF) << 16 | (uint32_t)c[3] << 24;
        else
            *reinterpret_cast<uint2*>(out + r * 128) = make_uint2((c[0] & 0xFFFF) | (uint32_t)c[1] << 16, (c[2] & 0xFFFF) | (uint32_t)c[3] << 16);
        if (lane == 0) {
            a.scales[row0 + r] = scale;
            if ((row0 + r) % a.P == 0) a.fill[(row0 + r) / a.P] = 0;
        }
    }
}

}  // namespace

cudaError_t launch_state_store(const StateCacheArgs& a, cudaStream_t s) {
    const uint64_t rows = (uint64_t)a.batch * a.H * a.P;
    if (!rows || !a.N) return cudaSuccess;
    if (a.N == 128 && aligned(a.state, 16) && aligned(a.codes, 8)) {
        constexpr unsigned PER = SC_THREADS / 32 * STORE_ROWS;
        const unsigned grid = (unsigned)((rows + PER - 1) / PER);
        if (a.bits == 8) k_state_store128<int8_t><<<grid, SC_THREADS, 0, s>>>(a);
        else k_state_store128<int16_t><<<grid, SC_THREADS, 0, s>>>(a);
        return cudaGetLastError();
    }
    const unsigned grid = (unsigned)((rows + SC_THREADS / 32 - 1) / (SC_THREADS / 32));
    if (a.bits == 8) k_state_store<int8_t><<<grid, SC_THREADS, 0, s>>>(a);
    else k_state_store<int16_t><<<grid, SC_THREADS, 0, s>>>(a);
    return cudaGetLastError();
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
