// token_logprobs.hpp — scores of given tokens under rows of logits: per row r with x = logits[r], Z = sum_c exp(x_c - max x)
//   logprob(c) = x_c - max x - log Z
//   entropy    = -sum_c p_c log p_c = log Z - (1/Z) sum_c (x_c - max x) exp(x_c - max x)
//   top        = the `top` largest logits, equal ones in the order of their index (NaN ranks above everything, as in torch.argmax:
//                the rule of ctc.hpp), with their log probabilities
// A logit of -inf has probability 0 and adds nothing to the entropy; a row of nothing else has log probability -inf everywhere and
// entropy 0; a row with a NaN or +inf has NaN for both.  Sums are in 32 bits.  exp(d) is 2^(d / ln 2) with the product rounded once: off by
// about |d| 2^-24 of itself, most where it is smallest; logarithms are log2 times ln 2 (error against 64 bits: 5e-8 of the results, the plain form's 8e-8).
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
    int32_t C, given, top, tokens64, dtype;
    int32_t slices, slice;            // workgroups of a row, classes of each but the last
    float *part;                      // slices > 1: [rows * slices][4] maximum, sum, weighted sum; then the alternatives [rows * slices][top] as 64-bit keys
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


// ---- few classes: G lanes per row (16: four rows per wave, so that a reduction of four steps serves four rows; or 64), NV logits in a lane's registers
// (class lane + G i).  The alternatives are picked one after the other: the largest key, then the lowest class that has it.  Bound by the vector
// unit: 36864 rows of 232 in fp32 with 4 alternatives 12.3 us = 2.9 TB/s, without any 7.5 us = 4.7 TB/s (1.2 us an alternative).
template <int CTRL> __device__ __forceinline__ uint32_t lp_turn(uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, false); }

// the same value in all G lanes: by rotations within 16 lanes, then by exchanging the halves and quarters of the wave
template <int G, class Op> __device__ __forceinline__ uint32_t lp_all(uint32_t x, Op op) {
    x = op(x, lp_turn<0x128>(x));                               // row_ror:8, 4, 2, 1
    x = op(x, lp_turn<0x124>(x));
    x = op(x, lp_turn<0x122>(x));
    x = op(x, lp_turn<0x121>(x));
    if constexpr (G == 64) {
        const auto h = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        x = op((uint32_t)h[0], (uint32_t)h[1]);
        const auto q = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        x = op((uint32_t)q[0], (uint32_t)q[1]);
    }
    return x;
}
template <int G> __device__ __forceinline__ uint32_t lp_max(uint32_t x) { return lp_all<G>(x, [](uint32_t a, uint32_t b) { return max(a, b); }); }
template <int G> __device__ __forceinline__ float lp_max(float x) {
    return __uint_as_float(lp_all<G>(__float_as_uint(x), [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
}
template <int G> __device__ __forceinline__ float lp_sum(float x) {
    return __uint_as_float(lp_all<G>(__float_as_uint(x), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}

__device__ __forceinline__ void lp_given(const LogprobArgs &a, int64_t r, int first, int step, float base, float logz, bool none) {
    for (int g = first; g < a.given; g += step) {
        const int64_t at = r * a.given + g;
        const int64_t t = a.tokens64 ? static_cast<const int64_t *>(a.tokens)[at] : static_cast<const int32_t *>(a.tokens)[at];
        float lp = 0.f;
        if (t >= a.C) lp = __builtin_nanf("");
        else if (t >= 0) {
            const int64_t e = r * a.stride + t;
            const float v = a.dtype == DT_F32 ? static_cast<const float *>(a.x)[e] : a.dtype == DT_BF16 ? (float)static_cast<const __bf16 *>(a.x)[e] : (float)static_cast<const _Float16 *>(a.x)[e];
            lp = none ? -INFINITY : (v - base) - logz;
        }
        a.logprob[at] = lp;
    }
}

template <int DT, int G, int NV>
__global__ __launch_bounds__(256) void token_logprobs_few_kernel(LogprobArgs a) {
    using T = typename ElemOf<DT>::type;
    const int lane = threadIdx.x & (G - 1);
    const int64_t r = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    if (r >= a.rows) return;                                    // (whole groups of G lanes)
    const T *x = static_cast<const T *>(a.x) + r * a.stride;
    float v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        v[i] = -INFINITY;
        if (G * i + G <= a.C || lane + G * i < a.C) v[i] = (float)x[lane + G * i];
    }
    float m = v[0];
#pragma unroll
    for (int i = 1; i < NV; ++i) m = fmaxf(m, v[i]);
    m = lp_max<G>(m);
    const float base = m == -INFINITY ? 0.f : m;
    float z = 0.f, e = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const float d = v[i] - base, p = __builtin_amdgcn_exp2f(d * 1.44269504088896f);
        z += p;
        e = fmaf(p, fmaxf(d, -200.f), e);                       // (p is 0 from -104 on)
    }
    z = lp_sum<G>(z);
    e = lp_sum<G>(e);
    const bool none = z == 0.f;
    const float logz = __builtin_amdgcn_logf(z) * 0.693147180559945f;
    if (lane == 0) a.entropy[r] = none ? 0.f : logz - e / z;
    lp_given(a, r, lane, G, base, logz, none);
    float *top_lp = a.top_logprob + r * a.top;
    int32_t *top_at = a.top_index + r * a.top;
    // ---- the alternatives: rows of ordinary numbers by the numbers themselves, a taken one becomes -inf
    bool plain = __ballot(!(z > 0.f && z <= 3.402823466e38f)) == 0;
    float best = m;
    for (int t = 0; plain && t < a.top; ++t) {
        if (t) {
            best = v[0];
#pragma unroll
            for (int i = 1; i < NV; ++i) best = fmaxf(best, v[i]);
            best = lp_max<G>(best);
            if (__ballot(best == -INFINITY)) { plain = false; break; }          // fewer numbers than alternatives
        }
        int slot = NV;
#pragma unroll
        for (int i = NV - 1; i >= 0; --i) slot = v[i] == best ? i : slot;
        const uint32_t mine = slot == NV ? 0u : ~(uint32_t)(lane + G * slot), low = lp_max<G>(mine);          // ~class: the largest is the lowest class
        slot = mine == low ? slot : NV;
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = slot == i ? -INFINITY : v[i];
        if (lane == 0) {
            top_lp[t] = (best - base) - logz;
            top_at[t] = (int32_t)~low;
        }
    }
    if (plain) return;
    // rows with NaN or infinities, or with fewer numbers than alternatives: by integer keys
    uint32_t key[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) key[i] = lane + G * i < a.C ? lp_key((float)x[lane + G * i]) : 0u;          // (below the key of -inf)
    for (int t = 0; t < a.top; ++t) {
        uint32_t most = 0, low = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) most = max(most, key[i]);
        most = lp_max<G>(most);
#pragma unroll
        for (int i = NV - 1; i >= 0; --i) low = key[i] == most ? ~(uint32_t)(lane + G * i) : low;
        low = lp_max<G>(low);
#pragma unroll
        for (int i = 0; i < NV; ++i) key[i] = ~low == (uint32_t)(lane + G * i) ? 0u : key[i];
        if (lane == 0) {
            top_lp[t] = none ? -INFINITY : (lp_value(most) - base) - logz;
            top_at[t] = (int32_t)~low;
        }
    }
}

// ---- many classes: a workgroup of B threads per row, one pass over it in pieces of 16 bytes; thread t takes pieces t, t + B, ... and keeps the
// running maximum, sum and weighted sum of its own.  The alternatives cost no second pass: a row's k best lie with the threads whose
// own maximum is among the k largest, so only these threads' pieces (k of B shares) are read again, and of them only what reaches the k-th
// largest maximum T is kept and ranked.  Where many threads share T (equal logits, rows that are masked but for a few classes) the
// numbers above T are kept and the lowest classes equal to T are found by reading the row from its start.  What does not fit
// the list of candidates, and rows with NaN or +inf, take one pass per alternative.
// Few long rows are cut into slices, a workgroup each (SPLIT), whose sums and alternatives the kernel below joins.
//
// Bound by HBM where rows are long (1024 rows of 131072 in bf16, top 20: 52.7 us = 5.1 TB/s; 9 rows of 151003 in fp32 in 18 slices each 11.6 us,
// read by 9 CUs 16.0, 36 GB/s a CU); where they are short by the choice of the alternatives, which a wave makes alone (36864 rows of 1000 in fp32: none 30.5 us, top 4 47.5,
// top 20 64).  So reductions stay in registers, and the list of a single wave is short: 2.6 KB of LDS let 32 of them share a CU (with 9 KB 17,
// 52 -> 33 us for rows of 500, top 4).
constexpr int LP_CAND = 1024, LP_SLACK = 32, LP_GRID = 1 << 21;       // (rows in the first axis of the grid)
constexpr int LP_WAVE_TOP = 26;                                       // alternatives that a single wave picks
constexpr int lp_cand(int threads) { return threads == 64 ? 256 : LP_CAND; }

template <int DT, int V> __device__ __forceinline__ void lp_load(const void *p, float (&x)[V]) {
    using T = typename ElemOf<DT>::type;
    alignas(16) T t[V];
    __builtin_memcpy(t, static_cast<const T *>(p), 16);         // one load, aligned to an element or better
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = (float)t[i];
}

template <int DT, int B, bool SPLIT = false>
__global__ __launch_bounds__(B) void token_logprobs_kernel(LogprobArgs a) {
    using T = typename ElemOf<DT>::type;
    constexpr int V = 16 / sizeof(T), W = B / 64, U = 4, CAND = lp_cand(B);
    static_assert(B <= CAND && LP_MAX_TOP <= B, "the list of candidates; a maximum per thread for every alternative");
    __shared__ float red[3][W];
    __shared__ uint32_t maxima[B];
    __shared__ uint32_t picked[B];                              // threads whose pieces are read again
    __shared__ unsigned long long cand[CAND + LP_MAX_TOP];
    __shared__ uint32_t limit[2];
    __shared__ int count[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r = SPLIT ? blockIdx.x / (uint32_t)a.slices : blockIdx.x + (int64_t)blockIdx.y * LP_GRID;
    if (r >= a.rows) return;
    const int class0 = SPLIT ? (int)(blockIdx.x - (uint32_t)r * (uint32_t)a.slices) * a.slice : 0, C = SPLIT ? min(a.slice, a.C - class0) : a.C;
    const T *x = static_cast<const T *>(a.x) + r * a.stride + class0;
    // pieces from the row's start, wherever that lies: which thread sums what, and so the last bit, is not a matter of the address
    const int pieces = C / V, tail = C - pieces * V;

    float m = -INFINITY, ref = 0.f, z = 0.f, e = 0.f;
    auto add = [&](float v) {
        const float d = v - ref, p = __builtin_amdgcn_exp2f(d * 1.44269504088896f);
        z += p;
        e = fmaf(p, fmaxf(d, -200.f), e);                       // (p is 0 from -104 on)
    };
    auto raise = [&](float mx) {                                // a new maximum: the sums so far in its units
        if (mx > m) {
            const float s = m == -INFINITY ? 0.f : m - mx, f = __builtin_amdgcn_exp2f(s * 1.44269504088896f);
            e = f == 0.f ? 0.f : f * fmaf(s, z, e);
            z *= f;
            m = ref = mx;
        }
    };
    int i = tid;
    for (; i + (U - 1) * B < pieces; i += U * B) {
        float v[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) lp_load<DT, V>(x + (int64_t)(i + u * B) * V, v[u]);
        float mx = v[0][0];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < V; ++j) mx = fmaxf(mx, v[u][j]);
        raise(mx);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < V; ++j) add(v[u][j]);
    }
    for (; i < pieces; i += B) {
        float v[V];
        lp_load<DT, V>(x + (int64_t)i * V, v);
        float mx = v[0];
#pragma unroll
        for (int j = 1; j < V; ++j) mx = fmaxf(mx, v[j]);
        raise(mx);
#pragma unroll
        for (int j = 0; j < V; ++j) add(v[j]);
    }
    if (tid < tail) { const float v = (float)x[pieces * V + tid]; raise(v); add(v); }
    const float mine = m;
    // ---- the row's maximum and sums
    m = lp_max<64>(m);
    if (lane == 0) red[0][wave] = m;
    __syncthreads();
    for (int w = 0; w < W; ++w) m = fmaxf(m, red[0][w]);
    {
        const float s = mine == -INFINITY ? 0.f : mine - m, f = __builtin_amdgcn_exp2f(s * 1.44269504088896f);
        e = f == 0.f && z == z ? 0.f : f * fmaf(s, z, e);       // (a NaN sum stays one)
        z *= f;
    }
    z = lp_sum<64>(z);
    e = lp_sum<64>(e);
    if (lane == 0) { red[1][wave] = z; red[2][wave] = e; }
    if (a.top > 0) maxima[tid] = lp_key(mine);                  // (-inf where a thread has nothing: never among the k best of a larger set)
    if (tid < 2) count[tid] = 0;
    __syncthreads();
    z = red[1][0];
    e = red[2][0];
    for (int w = 1; w < W; ++w) { z += red[1][w]; e += red[2][w]; }
    const float base = m == -INFINITY ? 0.f : m;
    const bool none = z == 0.f, odd = !(z <= 3.402823466e38f);
    const float logz = __builtin_amdgcn_logf(z) * 0.693147180559945f;
    if constexpr (SPLIT) {
        if (tid == 0) *reinterpret_cast<float4 *>(a.part + (int64_t)blockIdx.x * 4) = make_float4(m, z, e, 0.f);
    } else {
        if (tid == 0) a.entropy[r] = none ? 0.f : logz - e / z;
        lp_given(a, r, tid, B, base, logz, none);
    }
    const int k = a.top;
    if (k == 0) return;
    auto put = [&](int at, unsigned long long c) {
        if constexpr (SPLIT) {
            reinterpret_cast<unsigned long long *>(a.part + (int64_t)a.rows * a.slices * 4)[(int64_t)blockIdx.x * k + at] = c - (uint32_t)class0;      // (low word: ~class)
            return;
        }
        a.top_logprob[r * k + at] = none ? -INFINITY : (lp_value((uint32_t)(c >> 32)) - base) - logz;
        a.top_index[r * k + at] = (int32_t)~(uint32_t)c;
    };
    bool done = false;
    if (!odd) {
        // ---- T: the largest number (or near it) that at least k threads' maxima reach
        if (wave == 0) {
            uint32_t mk[W], lo = ~0u;
#pragma unroll
            for (int w = 0; w < W; ++w) { mk[w] = maxima[w * 64 + lane]; lo = min(lo, mk[w]); }
            lo = ~lp_max<64>(~lo);
            uint32_t hi = lp_key(m) + 1;                        // reached by nobody; lo by all B >= k
            lo = __builtin_amdgcn_readfirstlane(lo);
            hi = __builtin_amdgcn_readfirstlane(hi);
            int n_lo = B;
            while (hi - lo > 1 && n_lo > k + LP_SLACK) {
                const uint32_t mid = lo + (hi - lo) / 2;
                int n = 0;
#pragma unroll
                for (int w = 0; w < W; ++w) n += __popcll(__ballot(mk[w] >= mid));
                if (n >= k) { lo = mid; n_lo = n; } else hi = mid;
            }
            if (lane == 0) { limit[0] = lo; limit[1] = n_lo > k + LP_SLACK; }
        }
        __syncthreads();
        const uint32_t T0 = limit[0];
        const bool ties = limit[1] != 0;                        // then T0 is exactly the k-th largest maximum, and many threads have it
        const uint32_t from = ties ? T0 + 1 : T0;
        if (maxima[tid] >= from) picked[atomicAdd(&count[0], 1)] = tid;
        __syncthreads();
        const int n_picked = count[0], per = (pieces + B - 1) / B;
        auto keep = [&](float v, int c) {
            const uint32_t key = lp_key(v);
            if (key >= from) {
                const int at = atomicAdd(&count[1], 1);
                if (at < CAND) cand[at] = (unsigned long long)key << 32 | (uint32_t)~c;
            }
        };
        for (int64_t j = tid; j < (int64_t)n_picked * per; j += B) {
            const int piece = (int)(j % per) * B + (int)picked[j / per];
            if (piece < pieces) {
                float v[V];
                lp_load<DT, V>(x + (int64_t)piece * V, v);
#pragma unroll
                for (int q = 0; q < V; ++q) keep(v[q], piece * V + q);
            }
        }
        for (int j = tid; j < n_picked; j += B) {
            const int t = (int)picked[j];
            if (t < tail) keep((float)x[pieces * V + t], pieces * V + t);
        }
        __syncthreads();
        int n = count[1];
        bool fits = n <= CAND;
        if (ties && n < k) {                                    // the lowest classes equal to T0 make up the rest
            __syncthreads();
            for (int c0 = 0; c0 < C && n < k; c0 += B) {
                const int c = c0 + tid;
                if (c < C && lp_key((float)x[c]) == T0) cand[atomicAdd(&count[1], 1)] = (unsigned long long)T0 << 32 | (uint32_t)~c;
                __syncthreads();
                n = count[1];                                   // (at most k - 1 + B)
                __syncthreads();
            }
        }
        if (fits) {
            for (int j = tid; j < n; j += B) {
                const unsigned long long c = cand[j];
                int rank = 0;
                for (int q = 0; q < n; ++q) rank += cand[q] > c;
                if (rank < k) put(rank, c);
            }
            done = true;
        }
    }
    if (done) return;
    unsigned long long last = ~0ull;                            // (key, ~class) of the previous alternative
    for (int t = 0; t < k; ++t) {
        unsigned long long b = 0;
        for (int c = tid; c < C; c += B) {
            const unsigned long long q = (unsigned long long)lp_key((float)x[c]) << 32 | (uint32_t)~c;
            if ((t == 0 || q < last) && q > b) b = q;
        }
        for (int o = 32; o >= 1; o >>= 1) { const unsigned long long q = __shfl_xor(b, o, 64); b = q > b ? q : b; }
        __syncthreads();
        if (lane == 0) cand[wave] = b;
        __syncthreads();
        for (int w = 0; w < W; ++w) b = cand[w] > b ? cand[w] : b;
        last = b;
        if (tid == 0) put(t, b);
    }
}

// The slices of a row meet: a workgroup per row; a lane per slice for the sums.  Every slice's alternatives come in order, so a row's k best reach
// the least of the slices' ceil(k / slices)-th ones (these and the better ones are k or more), and the best of the slices' k-th ones; only what
// does is ranked (16 slices, k = 64: all 1024 against each other took 60 us).
template <int DT>
__global__ __launch_bounds__(256) void token_logprobs_join_kernel(LogprobArgs a) {
    __shared__ unsigned long long cand[LP_CAND], limit;
    __shared__ float whole[2];
    __shared__ int kept;
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    const int n = a.slices * a.top;                             // <= LP_CAND
    const unsigned long long *found = reinterpret_cast<const unsigned long long *>(a.part + a.rows * a.slices * 4) + r * n;
    if (tid < 64 && a.top > 0) {                                // (slices <= 64)
        const int at = min(tid, a.slices - 1) * a.top;
        unsigned long long least = found[at + (a.top + a.slices - 1) / a.slices - 1], last = found[at + a.top - 1];
        for (int o = 32; o >= 1; o >>= 1) {
            const unsigned long long p = __shfl_xor(least, o, 64), q = __shfl_xor(last, o, 64);
            least = p < least ? p : least;
            last = q > last ? q : last;
        }
        if (tid == 0) limit = least > last ? least : last;
    }
    if (tid == 64) kept = 0;
    if (tid < 64) {
        float4 s = make_float4(-INFINITY, 0.f, 0.f, 0.f);
        if (tid < a.slices) s = *reinterpret_cast<const float4 *>(a.part + (r * a.slices + tid) * 4);
        float m = s.x, z = s.y, e = s.z;
        for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        const float d = s.x == -INFINITY ? 0.f : s.x - m, f = __builtin_amdgcn_exp2f(d * 1.44269504088896f);
        e = f == 0.f && z == z ? 0.f : f * fmaf(d, z, e);
        z *= f;
        for (int o = 32; o >= 1; o >>= 1) { z += __shfl_xor(z, o, 64); e += __shfl_xor(e, o, 64); }
        if (tid == 0) {
            const bool none = z == 0.f;
            const float logz = __builtin_amdgcn_logf(z) * 0.693147180559945f;
            a.entropy[r] = none ? 0.f : logz - e / z;
            whole[0] = m;
            whole[1] = none ? -INFINITY : logz;                 // (an ordinary row's is not below 0)
        }
    }
    __syncthreads();
    const float m = whole[0], base = m == -INFINITY ? 0.f : m, logz = whole[1];
    const bool none = logz == -INFINITY;
    lp_given(a, r, tid, 256, base, logz, none);
    if (a.top == 0) return;
    for (int i = tid; i < n; i += 256) {
        const unsigned long long c = found[i];
        if (c >= limit) cand[atomicAdd(&kept, 1)] = c;
    }
    __syncthreads();
    const int left = kept;
    for (int i = tid; i < left; i += 256) {
        const unsigned long long c = cand[i];
        int rank = 0;
        for (int q = 0; q < left; ++q) rank += cand[q] > c;
        if (rank < a.top) {
            a.top_logprob[r * a.top + rank] = none ? -INFINITY : (lp_value((uint32_t)(c >> 32)) - base) - logz;
            a.top_index[r * a.top + rank] = (int32_t)~(uint32_t)c;
        }
    }
}

}  // namespace pocr
