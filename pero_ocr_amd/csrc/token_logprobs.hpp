// token_logprobs.hpp — scores of given tokens under rows of logits: per row r with x = logits[r], Z = sum_c exp(x_c - max x)
//   logprob(c) = x_c - max x - log Z
//   entropy    = -sum_c p_c log p_c = log Z - (1/Z) sum_c (x_c - max x) exp(x_c - max x)
//   top        = the `top` largest logits, equal ones in the order of their index (NaN ranks above everything, as in torch.argmax:
//                the rule of ctc.hpp), with their log probabilities
// A logit of -inf has probability 0 and adds nothing to the entropy; a row of nothing else has log probability -inf everywhere and
// entropy 0; a row with a NaN or +inf has NaN for both.  Sums are in 32 bits.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "kv_cache.hpp"

namespace pocr {

struct LogprobArgs {
    const void *x;
    int64_t stride;                   // elements between rows
    const void *tokens;               // [rows][given]
    float *logprob;                   // [rows][given]
    float *entropy;                   // [rows]
    float *top_logprob;               // [rows][top]
    int32_t *top_index;               // [rows][top]
    int64_t rows;
    int32_t C, given, top, tokens64;
};

constexpr int LP_MAX_TOP = 64;

// order of the alternatives as an unsigned number: larger = better; -0 and +0 are equal, NaN is the largest
__device__ __forceinline__ uint32_t lp_key(float v) {
    if (v != v) return 0xffffffffu;
    const uint32_t u = __float_as_uint(v + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t key) {
    if (key == 0xffffffffu) return __builtin_nanf("");
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// One workgroup per row; the alternatives one after the other.
template <int DT>
__global__ __launch_bounds__(256) void token_logprobs_kernel(LogprobArgs a) {
    using T = typename ElemOf<DT>::type;
    __shared__ float red[8];
    __shared__ unsigned long long best[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r = blockIdx.x;
    const T *x = static_cast<const T *>(a.x) + r * a.stride;
    float m = -INFINITY;
    int bad = 0;
    for (int c = tid; c < a.C; c += 256) { const float v = (float)x[c]; m = fmaxf(m, v); bad |= v != v; }
    for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    if (lane == 0) red[wave] = m;
    bad = __syncthreads_or(bad);
    m = bad ? __builtin_nanf("") : fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float base = m == -INFINITY ? 0.f : m;
    float z = 0.f, e = 0.f;
    for (int c = tid; c < a.C; c += 256) {
        const float d = (float)x[c] - base, p = expf(d);
        z += p;
        e += p == 0.f ? 0.f : p * d;
    }
    for (int off = 32; off >= 1; off >>= 1) { z += __shfl_xor(z, off, 64); e += __shfl_xor(e, off, 64); }
    __syncthreads();
    if (lane == 0) { red[wave] = z; red[4 + wave] = e; }
    __syncthreads();
    z = red[0] + red[1] + red[2] + red[3];
    e = red[4] + red[5] + red[6] + red[7];
    const float logz = logf(z);
    auto logp = [&](float v) { return z == 0.f ? -INFINITY : (v - base) - logz; };
    if (tid == 0) a.entropy[r] = z == 0.f ? 0.f : logz - e / z;
    for (int g = tid; g < a.given; g += 256) {
        const int64_t at = r * a.given + g;
        const int64_t t = a.tokens64 ? static_cast<const int64_t *>(a.tokens)[at] : static_cast<const int32_t *>(a.tokens)[at];
        a.logprob[at] = t < 0 ? 0.f : t >= a.C ? __builtin_nanf("") : logp((float)x[t]);
    }
    unsigned long long last = ~0ull;                            // (key, ~index) of the previous alternative
    for (int i = 0; i < a.top; ++i) {
        unsigned long long b = 0;
        for (int c = tid; c < a.C; c += 256) {
            const unsigned long long k = (unsigned long long)lp_key((float)x[c]) << 32 | (uint32_t)~c;
            if ((i == 0 || k < last) && k > b) b = k;
        }
        for (int off = 32; off >= 1; off >>= 1) { const unsigned long long o = __shfl_xor(b, off, 64); b = o > b ? o : b; }
        __syncthreads();
        if (lane == 0) best[wave] = b;
        __syncthreads();
        for (int w = 0; w < 4; ++w) b = best[w] > b ? best[w] : b;
        last = b;
        if (tid == 0) {
            a.top_logprob[r * a.top + i] = logp(lp_value((uint32_t)(b >> 32)));
            a.top_index[r * a.top + i] = (int32_t)~(uint32_t)b;
        }
    }
}

}  // namespace pocr
