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
#include "device_util.cuh"
#include "lssm_internal.h"

namespace lssm {

namespace {

constexpr int LP_THREADS = 256;

// Orders values as whole numbers: NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t order_key(float v) {
    v = v != v ? -INFINITY : v + 0.0f;
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
// Larger key first, of equal ones the lower index: one number to compare, never equal for two indices.
__device__ __forceinline__ uint64_t rank_key(float v, uint32_t i) { return (uint64_t)order_key(v) << 32 | (~i); }

__device__ __forceinline__ uint64_t warp_max64(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t w = __shfl_xor_sync(0xffffffffu, v, o);
        v = w > v ? w : v;
    }
    return v;
}

__global__ void __launch_bounds__(LP_THREADS) k_logprobs(LogprobsArgs a) {
    __shared__ float red[32];
    __shared__ uint64_t best[LP_THREADS / 32];
    const uint32_t r = blockIdx.x, tid = threadIdx.x, V = a.vocab;
    const uint64_t base = (uint64_t)r * a.row_stride;
    const int lane = tid & 31, wid = tid >> 5;

    auto block_best = [&](uint64_t k) {
        k = warp_max64(k);
        __syncthreads();
        if (lane == 0) best[wid] = k;
        __syncthreads();
        uint64_t b = best[0];
        for (int i = 1; i < LP_THREADS / 32; ++i) b = best[i] > b ? best[i] : b;
        return b;
    };
    uint64_t top = 0;
    float bad = 0.0f;
    for (uint32_t i = tid; i < V; i += LP_THREADS) {
        const float x = load_any(a.logits, base + i, a.dtype);
        const uint64_t k = rank_key(x, i);
        top = k > top ? k : top;
        if (x != x || x == INFINITY) bad = 1.0f;
    }
    top = block_best(top);
    bad = block_sum(bad, red);
    const float m = key_value((uint32_t)(top >> 32));
    const bool none = m == -INFINITY && bad == 0.0f;
    float s = 0.0f, u = 0.0f;
    for (uint32_t i = tid; i < V; i += LP_THREADS) {
        const float d = load_any(a.logits, base + i, a.dtype) - m, e = expf(d);
        s += e;
        if (e > 0.0f) u += e * d;
    }
    s = block_sum(s, red);
    u = block_sum(u, red);
    const float nan = __int_as_float(0x7FC00000);
    const float ls = bad > 0.0f ? nan : logf(s);
    if (tid == 0) {
        if (a.lse) a.lse[r] = none ? -INFINITY : m + ls;
        if (a.entropy) a.entropy[r] = none ? 0.0f : ls - u / s;
        if (a.logp) {
            const uint32_t t = a.targets[r];
            float v = 0.0f;
            if (t != LSSM_NO_TOKEN)
                v = t >= V ? nan : none ? -INFINITY : (load_any(a.logits, base + t, a.dtype) - m) - ls;
            a.logp[r] = v;
        }
    }
    uint64_t last = top;
    for (uint32_t k = 0; k < a.top_k; ++k) {
        if (k) {
            uint64_t next = 0;
            for (uint32_t i = tid; i < V; i += LP_THREADS) {
                const uint64_t c = rank_key(load_any(a.logits, base + i, a.dtype), i);
                if (c < last && c > next) next = c;
            }
            last = block_best(next);
        }
        if (tid == 0) {
            a.top_ids[(uint64_t)r * a.top_k + k] = ~(uint32_t)last;
            a.top_logp[(uint64_t)r * a.top_k + k] = none ? -INFINITY : (key_value((uint32_t)(last >> 32)) - m) - ls;
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
    k_logprobs<<<a.rows, LP_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_logprobs_grad(const LogprobsGradArgs& a, cudaStream_t s) {
    if (!a.rows) return cudaSuccess;
    k_logprobs_grad<<<a.rows, LP_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace lssm
