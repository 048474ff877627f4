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

}  // namespace

cudaError_t launch_state_store(const StateCacheArgs& a, cudaStream_t s) {
    const uint64_t rows = (uint64_t)a.batch * a.H * a.P;
    if (!rows || !a.N) return cudaSuccess;
    const unsigned grid = (unsigned)((rows + SC_THREADS / 32 - 1) / (SC_THREADS / 32));
    if (a.bits == 8) k_state_store<int8_t><<<grid, SC_THREADS, 0, s>>>(a);
    else k_state_store<int16_t><<<grid, SC_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_state_load(const StateCacheArgs& a, cudaStream_t s) {
    if (!a.batch || !a.H || !a.P || !a.N) return cudaSuccess;
    if (a.bits == 8) k_state_cached<int8_t, 1><<<a.batch * a.H, SC_THREADS, 0, s>>>(a);
    else k_state_cached<int16_t, 1><<<a.batch * a.H, SC_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_ssd_step_cached(const StateCacheArgs& a, cudaStream_t s) {
    if (!a.batch || !a.H || !a.P || !a.N) return cudaSuccess;
    if (a.bits == 8) k_state_cached<int8_t, 0><<<a.batch * a.H, SC_THREADS, 0, s>>>(a);
    else k_state_cached<int16_t, 0><<<a.batch * a.H, SC_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace lssm
