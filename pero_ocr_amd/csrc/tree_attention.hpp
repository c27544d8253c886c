// tree_attention.hpp — attention of the newest tokens of many sequences over their paged caches (kv_cache.hpp).
//
// Token i of a sequence with n new tokens and L cached positions (the new ones are the last n of them) sees the L - n older positions
// and, among the new ones, those its mask names (the ancestors in a tree of drafted tokens, itself among them); without a mask
// positions up to its own.  With s_j = scale * q . k_j over the seen j:  out = sum_j softmax(s)_j v_j,  lse = log sum_j exp(s_j);
// a token that sees nothing gets out = 0, lse = -inf.  Query head h reads key head h / (heads / kv_heads).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "kv_cache.hpp"

namespace pocr {

struct TreeAttnArgs {
    const void *q;
    const void *k, *v;
    const uint8_t *k_exp, *v_exp;
    const int32_t *table, *lengths, *starts;
    const uint64_t *mask;
    void *out;
    float *lse;
    int64_t q_ts, q_hs, table_stride, mask_stride, tokens;
    int32_t seqs, heads, kv_heads, num_pages, page_shift, max_pages, mask_words, zero_rest;
    float scale;
};

struct TreeSeq { int64_t first; int64_t n, len; };

__device__ __forceinline__ TreeSeq tree_seq(const TreeAttnArgs &a, int s) {
    const int64_t b = a.starts[s], e = a.starts[s + 1];
    TreeSeq r;
    r.first = b < 0 ? 0 : (b > a.tokens ? a.tokens : b);
    const int64_t end = e > a.tokens ? a.tokens : e;
    r.n = end > r.first ? end - r.first : 0;
    const int64_t cap = (int64_t)a.max_pages << a.page_shift, l = a.lengths[s];
    r.len = l < 0 ? 0 : (l > cap ? cap : l);
    return r;
}

// does new token i of a sequence with n new tokens see position j of L?  (row = its mask row)
__device__ __forceinline__ bool tree_sees(const uint64_t *row, int32_t words, int64_t i, int64_t n, int64_t len, int64_t j) {
    const int64_t d = j - (len - n);
    if (d < 0) return true;
    if (!row) return d <= i;
    return (d >> 6) < words && (row[d >> 6] >> (d & 63) & 1);
}

// One wave per (token, query head): a lane per key for the scores, a lane per element for the values.
template <int DT, int FMT, int D>
__global__ __launch_bounds__(64) void tree_attention_kernel(TreeAttnArgs a) {
    using T = typename ElemOf<DT>::type;
    const int lane = threadIdx.x, s = blockIdx.x, h = blockIdx.y, hk = h / (a.heads / a.kv_heads);
    __shared__ float qs[D];
    __shared__ float ps[64];
    __shared__ int64_t rows[64];
    const TreeSeq sq = tree_seq(a, s);
    if (a.zero_rest && s == a.seqs - 1)
        for (int64_t t = sq.first + sq.n + blockIdx.z; t < a.tokens; t += gridDim.z) {
            for (int d = lane; d < D; d += 64) static_cast<T *>(a.out)[(t * a.heads + h) * D + d] = (T)0.f;
            if (a.lse && lane == 0) a.lse[t * a.heads + h] = -INFINITY;
        }
    const int32_t *table = a.table + s * a.table_stride;
    for (int64_t i = blockIdx.z; i < sq.n; i += gridDim.z) {
        const int64_t t = sq.first + i;
        __syncthreads();
        for (int d = lane; d < D; d += 64) qs[d] = (float)static_cast<const T *>(a.q)[t * a.q_ts + h * a.q_hs + d];
        __syncthreads();
        const uint64_t *mrow = a.mask ? a.mask + t * a.mask_stride : nullptr;
        float m = -INFINITY, l = 0.f, acc[(D + 63) / 64] = {};
        for (int64_t j0 = 0; j0 < sq.len; j0 += 64) {
            const int64_t j = j0 + lane;
            int64_t row = -1;
            if (j < sq.len && tree_sees(mrow, a.mask_words, i, sq.n, sq.len, j))
                row = kv_row_base(table, a.max_pages, a.num_pages, a.kv_heads, hk, a.page_shift, j);
            float sc = -INFINITY;
            if (row >= 0) {
                float dot = 0.f;
                for (int d = 0; d < D; ++d) {
                    float kd;
                    if constexpr (FMT == KV_BF16) kd = (float)static_cast<const __bf16 *>(a.k)[row * D + d];
                    else kd = __builtin_amdgcn_cvt_f32_fp8((int)static_cast<const uint8_t *>(a.k)[row * D + d], 0);
                    dot += qs[d] * kd;
                }
                if constexpr (FMT == KV_FP8) dot *= kv_scale(a.k_exp[row]);
                sc = dot * a.scale;
            }
            float mt = sc;
            for (int off = 32; off >= 1; off >>= 1) mt = fmaxf(mt, __shfl_xor(mt, off, 64));
            const bool bad = __ballot(sc != sc) != 0;                 // a NaN score makes the row NaN, whatever the maximum says
            const float mn = bad ? __builtin_nanf("") : fmaxf(m, mt);
            const float base = mn == -INFINITY ? 0.f : mn;
            const float alpha = m == -INFINITY ? 0.f : expf(m - base);
            const float p = row >= 0 ? expf(sc - base) : 0.f;
            float sum = p;
            for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
            l = l * alpha + sum;
            m = mn;
            __syncthreads();
            ps[lane] = p;
            rows[lane] = row;
            __syncthreads();
#pragma unroll
            for (int c = 0; c < (D + 63) / 64; ++c) {
                const int d = lane + 64 * c;
                if (d >= D) continue;
                float o = acc[c] * alpha;
                for (int u = 0; u < 64; ++u) {
                    const int64_t rw = rows[u];
                    if (rw < 0) continue;
                    float vd;
                    if constexpr (FMT == KV_BF16) vd = (float)static_cast<const __bf16 *>(a.v)[rw * D + d];
                    else vd = __builtin_amdgcn_cvt_f32_fp8((int)static_cast<const uint8_t *>(a.v)[rw * D + d], 0) * kv_scale(a.v_exp[rw]);
                    o += ps[u] * vd;
                }
                acc[c] = o;
            }
        }
#pragma unroll
        for (int c = 0; c < (D + 63) / 64; ++c) {
            const int d = lane + 64 * c;
            if (d < D) static_cast<T *>(a.out)[(t * a.heads + h) * D + d] = (T)(l == 0.f ? 0.f : acc[c] / l);
        }
        if (a.lse && lane == 0) a.lse[t * a.heads + h] = l == 0.f ? -INFINITY : m + logf(l);
    }
}

}  // namespace pocr
