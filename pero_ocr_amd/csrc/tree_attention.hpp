// tree_attention.hpp — attention of the newest tokens of many sequences over their paged caches (kv_cache.hpp).
//
// Token i of a sequence with n new tokens and L cached positions (the new ones are the last n of them) sees the L - n older positions
// and, among the new ones, those its mask names (the ancestors in a tree of drafted tokens, itself among them); without a mask
// positions up to its own.  With s_j = scale * q . k_j over the seen j:  out = sum_j softmax(s)_j v_j,  lse = log sum_j exp(s_j);
// a token that sees nothing gets out = 0, lse = -inf.  Query head h reads key head h / (heads / kv_heads).
//
// One pass over the keys with a running maximum and sum.  A wave owns RT * 16 rows (a row = one new token and one of the query heads that
// share the key head) and takes blocks of 32 keys; both products run on v_mfma_f32_16x16x32_bf16, transposed, so that a row is always
// lane & 15 and nothing is exchanged between lanes but the row maximum:
//   S^T = K Q^T     lane (row, g = lane / 16) gets the scores of keys 4 g + r and 16 + 4 g + r of the block, r = 0..3
//   O^T = V^T P^T   takes exactly these eight probabilities as its operand when V^T is fed in the same key order
// Keys and values go from HBM straight into registers, no LDS and no barrier in the loop.  K: a lane holds a quarter of one key's
// row (which quarter of each 64 elements is free to choose, Q is laid out to match), so whole lines are read.  V: a lane loads D / 16 neighbouring elements
// of eight keys and transposes them with byte permutes; tile c of the product then is elements c, D/16 + c, 2 D/16 + c, ... and a lane ends up with
// D / 4 neighbouring outputs of its row.
// 8-bit codes become bfloat16 exactly, K's by v_cvt_scalef32 with the key's own power of two; V's power of two goes to the probability.
// What is rounded: the probability enters the second product as bf16 planes (cut, cut, rounded), two for 16-bit queries (2^-17 of it: one plane's 2^-9
// would add as much error as rounding the result does) and three for float32 (2^-25); a float16 or float32 query is two or three bf16 planes (exact / 2^-25).
// Scores, statistics and sums are float32.
//
// A NaN or infinity in V spreads in a matrix product to the masked rows, whose probability is 0; testing every element for it costs more than the
// transposition, so the loop does not.  A wave whose sums come out not finite goes through its keys again one by one, every row with the
// keys that it sees: slow, and met only where such numbers are.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "kv_cache.hpp"

namespace pocr {

typedef __bf16 ta_bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 ta_bf16x8 __attribute__((ext_vector_type(8)));
typedef float ta_f32x4 __attribute__((ext_vector_type(4)));

struct TreeAttnArgs {
    const void *q;
    const void *k, *v;
    const uint8_t *k_exp, *v_exp;
    const int32_t *table, *lengths, *starts;
    const uint64_t *mask;
    void *out;
    float *lse;
    float *part;                  // nsplit > 1: sums [nsplit][tokens * heads][D], then (maximum, sum) [nsplit][tokens * heads][2]
    int64_t q_ts, q_hs, table_stride, mask_stride, tokens;
    int32_t seqs, heads, kv_heads, num_pages, page_shift, max_pages, mask_words, zero_rest, nsplit, tiles, q_vec;
    float scale;
};

// arrays that no kernel of the call writes, read by a whole wave at one place: through the scalar cache
typedef const __attribute__((address_space(4))) int32_t *ScalarInts;

struct TreeSeq { int32_t first, n, len; };          // (positions and rows are 32-bit numbers: lengths and q_start are)

__device__ __forceinline__ TreeSeq tree_seq(const TreeAttnArgs &a, int s) {
    const ScalarInts starts = (ScalarInts)a.starts, lengths = (ScalarInts)a.lengths;
    const int32_t b = starts[s], e = starts[s + 1], total = (int32_t)a.tokens, l = lengths[s];
    TreeSeq r;
    r.first = min(max(b, 0), total);
    r.n = max(min(e, total) - r.first, 0);
    const int64_t cap = (int64_t)a.max_pages << a.page_shift;
    r.len = (int32_t)min((int64_t)max(l, 0), cap);
    return r;
}

// low `n` bits of a word, n of any size
__device__ __forceinline__ uint32_t low_bits(int32_t n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

// which of the 32 drafted tokens d0 .. d0 + 31 new token i sees; d < 0: an older position, seen by all
__device__ __forceinline__ uint32_t tree_window(const uint64_t *row, int32_t words, int32_t i, int32_t d0) {
    if (d0 < -31) return ~0u;
    if (!row) return low_bits(i - d0 + 1);
    const int32_t f = max(d0, 0), w = f >> 6, sh = f & 63;
    uint64_t lo = w < words ? row[w] : 0;
    lo >>= sh;
    if (sh && w + 1 < words) lo |= row[w + 1] << (64 - sh);
    const uint32_t bits = (uint32_t)lo;
    return d0 < 0 ? (bits << -d0) | low_bits(-d0) : bits;
}

__device__ __forceinline__ float row_max(float x) {          // over the four lanes of a row
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float row_sum(float x) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

union Frag { uint32_t u[4]; ta_bf16x8 b; };

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    union { ta_bf16x2 b; uint32_t u; } r;
    r.b = (ta_bf16x2){(__bf16)lo, (__bf16)hi};
    return r.u;
}

// eight floats as NP bf16 planes: all but the last cut, the last rounded
template <int NP> __device__ __forceinline__ void split_planes(const float (&x)[8], Frag (&f)[NP]) {
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = x[j];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        if (p == NP - 1) {
#pragma unroll
            for (int j = 0; j < 4; ++j) f[p].u[j] = pack_bf16(y[2 * j], y[2 * j + 1]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f[p].u[j] = __builtin_amdgcn_perm(__float_as_uint(y[2 * j + 1]), __float_as_uint(y[2 * j]), 0x07060302u);
                y[2 * j] -= __uint_as_float(__float_as_uint(y[2 * j]) & 0xffff0000u);
                y[2 * j + 1] -= __uint_as_float(__float_as_uint(y[2 * j + 1]) & 0xffff0000u);
            }
        }
    }
}

__device__ __forceinline__ uint32_t fp8_pair(uint32_t w, float scale, bool high) {
    union { ta_bf16x2 b; uint32_t u; } r;
    r.b = high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false);
    return r.u;
}

// A block of 32 keys as a lane holds it: for K its quarter of key (lane & 15) of both 16-key halves, for V D / 16 elements (from lane & 15 on) of
// the eight keys 4 g + a and 16 + 4 g + a.
template <int FMT, int D> struct KvBlock {
    static constexpr int ES = FMT == KV_FP8 ? 1 : 2;
    static constexpr int KW = D * ES / 16;                   // dwords of a quarter row
    static constexpr int VB = D * ES / 16;                   // bytes of V a lane holds per key
    static constexpr int VW = VB < 4 ? 1 : VB / 4;
    uint32_t k[2][KW];
    uint32_t v[8][VW];
    uint32_t ke[2], ve[2];

    // base[h]: row number of key 0 of half h (of row 0 where the page is absent: in bounds, and masked by the caller)
    __device__ __forceinline__ void load_keys(const TreeAttnArgs &a, const int64_t (&base)[2], int lane) {
        const int i = lane & 15, g = lane >> 4;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint8_t *kr = static_cast<const uint8_t *>(a.k) + (base[h] + i) * (D * ES);
            if constexpr (KW == 2) {
                *reinterpret_cast<kv_u32x2 *>(k[h]) = *reinterpret_cast<const kv_u32x2 *>(kr + g * 8);
            } else {
#pragma unroll
                for (int c = 0; c < KW / 4; ++c) *reinterpret_cast<kv_u32x4 *>(k[h] + 4 * c) = *reinterpret_cast<const kv_u32x4 *>(kr + c * 64 + g * 16);
            }
            if constexpr (FMT == KV_FP8) ke[h] = a.k_exp[base[h] + i];
        }
    }
    __device__ __forceinline__ void load_values(const TreeAttnArgs &a, const int64_t (&base)[2], int lane) {
        const int i = lane & 15, g = lane >> 4;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint8_t *vr = static_cast<const uint8_t *>(a.v) + (base[h] + 4 * g) * (D * ES) + i * VB;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                uint32_t *w = v[4 * h + t];
                const uint8_t *p = vr + t * (D * ES);
                if constexpr (VB == 2) w[0] = *reinterpret_cast<const uint16_t *>(p);
                else if constexpr (VB == 4) w[0] = *reinterpret_cast<const uint32_t *>(p);
                else if constexpr (VB == 8) *reinterpret_cast<kv_u32x2 *>(w) = *reinterpret_cast<const kv_u32x2 *>(p);
                else {
#pragma unroll
                    for (int c = 0; c < VB / 16; ++c) *reinterpret_cast<kv_u32x4 *>(w + 4 * c) = reinterpret_cast<const kv_u32x4 *>(p)[c];
                }
            }
            if constexpr (FMT == KV_FP8) ve[h] = *reinterpret_cast<const uint32_t *>(a.v_exp + base[h] + 4 * g);
        }
    }
    // operand of the first product: elements of step st (32 of them) of the keys of half h
    __device__ __forceinline__ Frag key(int h, int st) const {
        Frag f;
        if constexpr (FMT == KV_FP8) {
            const float s = kv_scale((uint8_t)ke[h]);
#pragma unroll
            for (int j = 0; j < 2; ++j) { f.u[2 * j] = fp8_pair(k[h][2 * st + j], s, false); f.u[2 * j + 1] = fp8_pair(k[h][2 * st + j], s, true); }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) f.u[j] = k[h][4 * st + j];
        }
        return f;
    }
    // element of a row that operand element j of step st stands for
    __device__ static __forceinline__ int key_elem(int g, int st) {
        if constexpr (FMT == KV_BF16) return st * 32 + g * 8;
        else if constexpr (D == 32) return g * 8;
        else return (st >> 1) * 64 + g * 16 + (st & 1) * 8;
    }
    // operands of the second product: NT = min(4 or 2, D / 16) tiles made of dword w of every key
    static constexpr int TW = FMT == KV_FP8 ? (VB < 4 ? 2 : 4) : 2;
    __device__ __forceinline__ void values(int w, Frag (&f)[TW]) const {
        if constexpr (FMT == KV_FP8) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t w0 = v[4 * h][w], w1 = v[4 * h + 1][w], w2 = v[4 * h + 2][w], w3 = v[4 * h + 3][w];
                const uint32_t x0 = __builtin_amdgcn_perm(w1, w0, 0x05010400u), y0 = __builtin_amdgcn_perm(w3, w2, 0x05010400u);
                uint32_t t[4];
                t[0] = __builtin_amdgcn_perm(y0, x0, 0x05040100u);
                t[1] = __builtin_amdgcn_perm(y0, x0, 0x07060302u);
                if constexpr (TW == 4) {
                    const uint32_t x1 = __builtin_amdgcn_perm(w1, w0, 0x07030602u), y1 = __builtin_amdgcn_perm(w3, w2, 0x07030602u);
                    t[2] = __builtin_amdgcn_perm(y1, x1, 0x05040100u);
                    t[3] = __builtin_amdgcn_perm(y1, x1, 0x07060302u);
                }
#pragma unroll
                for (int c = 0; c < TW; ++c) { f[c].u[2 * h] = fp8_pair(t[c], 1.f, false); f[c].u[2 * h + 1] = fp8_pair(t[c], 1.f, true); }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f[0].u[j] = __builtin_amdgcn_perm(v[2 * j + 1][w], v[2 * j][w], 0x05040100u);
                f[1].u[j] = __builtin_amdgcn_perm(v[2 * j + 1][w], v[2 * j][w], 0x07060302u);
            }
        }
    }
    // keys of the block that nobody may see: their values must not meet a probability 0 (the memory may hold NaN)
    __device__ __forceinline__ void drop_values(uint32_t there, int g) {
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            const bool keep = there >> ((t >> 2) * 16 + 4 * g + (t & 3)) & 1;
#pragma unroll
            for (int w = 0; w < VW; ++w) v[t][w] = keep ? v[t][w] : 0u;
        }
    }
};

template <int FMT> __device__ __forceinline__ float kv_element(const void *data, const uint8_t *exp, int64_t row, int dim, int d) {
    if constexpr (FMT == KV_BF16) return (float)static_cast<const __bf16 *>(data)[row * dim + d];
    else return __builtin_amdgcn_cvt_f32_fp8((int)static_cast<const uint8_t *>(data)[row * dim + d], 0) * kv_scale(exp[row]);
}

constexpr int TA_WAVES = 4;            // waves of a workgroup: they take the key blocks in turn

template <int DT, int FMT, int D, int RT>
__global__ __launch_bounds__(64 * TA_WAVES, D <= 128 ? 2 : 1) void tree_attention_kernel(TreeAttnArgs a) {
    using T = typename ElemOf<DT>::type;
    using Block = KvBlock<FMT, D>;
    constexpr int QP = DT == DT_F32 ? 3 : DT == DT_F16 ? 2 : 1;      // planes of the query
    constexpr int PP = DT == DT_F32 ? 3 : 2;                         // planes of the probabilities
    constexpr int NB = D / 16, ST = D / 32, TW = Block::TW;
    const int tid = threadIdx.x, lane = tid & 63, row = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nw = blockDim.x >> 6;
    __shared__ ta_f32x4 osum[TA_WAVES / 2][RT * NB][64];
    __shared__ float stat[TA_WAVES][RT][16][2];

    // workgroups that read the same keys (the row tiles of one sequence, key head and split) are 8 apart: consecutive workgroups go to
    // different XCDs, so these share an L2
    const uint32_t lane8 = blockIdx.x & 7, rest8 = blockIdx.x >> 3, tile0 = rest8 % (uint32_t)a.tiles;
    const uint32_t stream = (rest8 / (uint32_t)a.tiles) * 8 + lane8, pairs = (uint32_t)a.seqs * a.kv_heads;
    if (stream >= pairs * (uint32_t)a.nsplit) return;
    const int split = (int)(stream / pairs), pair = (int)(stream - split * pairs), s = pair / a.kv_heads, hk = pair - s * a.kv_heads;
    const TreeSeq sq = tree_seq(a, s);
    const int group = a.heads / a.kv_heads;
    const uint32_t rows = (uint32_t)sq.n * (uint32_t)group;           // (tokens * heads < 2^31)
    const int32_t *table = a.table + s * a.table_stride;
    // scores in units of log2: the sign of the scale goes to the query, so that the largest product is the largest score; 0 makes the query 0
    const float c = a.scale * 1.44269504088896f;
    const float csign = c == 0.f ? 0.f : c < 0.f ? -1.f : 1.f, cabs = c == 0.f ? 1.f : fabsf(c);

    if (a.zero_rest && s == a.seqs - 1 && split == 0) {               // rows of no sequence
        const uint32_t rest = ((uint32_t)a.tokens - (uint32_t)(sq.first + sq.n)) * (uint32_t)group;
        for (uint32_t r = tile0 * blockDim.x + tid; r < rest; r += (uint32_t)a.tiles * blockDim.x) {
            const int64_t at = (int64_t)(sq.first + sq.n + (int32_t)(r / group)) * a.heads + hk * group + (int32_t)(r % group);
#pragma unroll 1
            for (int d = 0; d < D; ++d) static_cast<T *>(a.out)[at * D + d] = (T)0.f;
            if (a.lse) a.lse[at] = -INFINITY;
        }
    }

    const int32_t blocks = (int32_t)(((uint32_t)sq.len + 31u) >> 5), per = (int32_t)(((uint32_t)blocks + a.nsplit - 1u) / (uint32_t)a.nsplit);
    const int32_t first_block = min(split * per, blocks), end_block = min(first_block + per, blocks);
    const int32_t ctx = sq.len - sq.n;

    for (uint32_t r0 = tile0 * (16 * RT); r0 < rows; r0 += (uint32_t)a.tiles * (16 * RT)) {
        int32_t tok[RT];
        int64_t at[RT];                                               // row of out, -1: none
        Frag q[RT][ST][QP];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const uint32_t r = r0 + 16 * rt + row, rr = min(r, rows - 1);
            tok[rt] = (int32_t)(rr / (uint32_t)group);
            const int head = hk * group + (int)(rr - (uint32_t)tok[rt] * (uint32_t)group);
            at[rt] = r < rows ? (int64_t)(sq.first + tok[rt]) * a.heads + head : -1;
            const T *qr = static_cast<const T *>(a.q) + (int64_t)(sq.first + tok[rt]) * a.q_ts + head * a.q_hs;
#pragma unroll
            for (int st = 0; st < ST; ++st) {
                float x[8];
                if (a.q_vec) load8<DT, true>(qr + Block::key_elem(g, st), x);
                else load8<DT, false>(qr + Block::key_elem(g, st), x);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] *= csign;
                split_planes<QP>(x, q[rt][st]);
            }
        }

        ta_f32x4 o[RT][NB];
        float m[RT], l[RT];                                           // m: of the raw scores (x csign); l: this lane's keys only
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            m[rt] = -INFINITY;
            l[rt] = 0.f;
#pragma unroll
            for (int t = 0; t < NB; ++t) o[rt][t] = (ta_f32x4){0.f, 0.f, 0.f, 0.f};
        }
        // a block's keys are requested as soon as the registers of the last one's are free, behind its scores, and its values behind its sums
        const ScalarInts pages = (ScalarInts)table;
        auto place = [&](int32_t b, int64_t (&base)[2], uint32_t &there) {
            const int32_t key0 = b << 5;
            there = low_bits(sq.len - key0);                          // keys that exist at all
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int32_t key = key0 + 16 * h;
                base[h] = 0;
                const int32_t page = key < sq.len ? pages[key >> a.page_shift] : -1;          // (len <= max_pages * page_size)
                if (page >= 0 && page < a.num_pages) base[h] = (((int64_t)page * a.kv_heads + hk) << a.page_shift) + (key & ((1 << a.page_shift) - 1));
                else there &= h ? 0x0000ffffu : 0xffff0000u;
            }
        };
        Block kv;
        int64_t base[2];
        uint32_t there = 0;
        if (first_block + wave < end_block) {
            place(first_block + wave, base, there);
            kv.load_keys(a, base, lane);
            kv.load_values(a, base, lane);
        }
        for (int32_t b = first_block + wave; b < end_block; b += nw) {
                const int32_t key0 = b << 5;
                int64_t next[2];
                uint32_t next_there = 0;
                const bool more = b + nw < end_block;
                if (more) place(b + nw, next, next_there);
                const bool edge = there != ~0u || key0 + 31 >= ctx;   // some key is not seen by every row
                ta_f32x4 sc[RT][2];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) sc[rt][0] = sc[rt][1] = (ta_f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int st = 0; st < ST; ++st) {
                        const Frag kf = kv.key(h, st);
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                            for (int pl = QP - 1; pl >= 0; --pl) sc[rt][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf.b, q[rt][st][pl].b, sc[rt][h], 0, 0, 0);
                    }
                if (more) kv.load_keys(a, next, lane);
                float p[RT][8];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) p[rt][j] = sc[rt][j >> 2][j & 3];
                    if (edge) {
                        const uint32_t vis = there & tree_window(a.mask ? a.mask + (int64_t)(sq.first + tok[rt]) * a.mask_stride : nullptr, a.mask_words, tok[rt], key0 - ctx);
#pragma unroll
                        for (int j = 0; j < 8; ++j) p[rt][j] = vis >> ((j >> 2) * 16 + 4 * g + (j & 3)) & 1 ? p[rt][j] : -INFINITY;
                    }
                    float mx = p[rt][0];
#pragma unroll
                    for (int j = 1; j < 8; ++j) mx = fmaxf(mx, p[rt][j]);
                    mx = fmaxf(m[rt], row_max(mx));
                    if (__ballot(mx > m[rt])) {
                        const float alpha = m[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m[rt] - mx) * cabs);
                        l[rt] *= alpha;
#pragma unroll
                        for (int t = 0; t < NB; ++t) o[rt][t] *= alpha;
                        m[rt] = mx;
                    }
                    // (2^-inf is 0; without a maximum yet the reference is 0)
                    const float mc = m[rt] == -INFINITY ? 0.f : m[rt] * cabs;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        p[rt][j] = __builtin_amdgcn_exp2f(fmaf(p[rt][j], cabs, -mc));
                        l[rt] += p[rt][j];
                    }
                    if constexpr (FMT == KV_FP8) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) p[rt][j] *= kv_scale((uint8_t)(kv.ve[j >> 2] >> (8 * (j & 3))));
                    }
                }
                if (there != ~0u) kv.drop_values(there, g);
                Frag pf[RT][PP];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) split_planes<PP>(p[rt], pf[rt]);
#pragma unroll
                for (int w = 0; w < NB / TW; ++w) {
                    Frag vf[TW];
                    kv.values(w, vf);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int t = 0; t < TW; ++t)
#pragma unroll
                            for (int pl = PP - 1; pl >= 0; --pl)
                                o[rt][w * TW + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[t].b, pf[rt][pl].b, o[rt][w * TW + t], 0, 0, 0);
                }
                if (more) kv.load_values(a, next, lane);
                base[0] = next[0];
                base[1] = next[1];
                there = next_there;
        }
        bool odd = false;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int t = 0; t < NB; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) odd |= !(fabsf(o[rt][t][r]) <= 3.402823466e38f);
        if (__ballot(odd)) {                                          // key by key, each row only with what it sees
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                m[rt] = -INFINITY;
                l[rt] = 0.f;
#pragma unroll
                for (int t = 0; t < NB; ++t) o[rt][t] = (ta_f32x4){0.f, 0.f, 0.f, 0.f};
                const uint32_t rr = min(r0 + 16 * rt + row, rows - 1);
                const T *qr = static_cast<const T *>(a.q) + (int64_t)(sq.first + tok[rt]) * a.q_ts + (hk * group + (int)(rr - (uint32_t)tok[rt] * (uint32_t)group)) * a.q_hs;
                for (int32_t b = first_block + wave; b < end_block; b += nw)
                    for (int32_t key = b << 5, n = min(32, sq.len - key); n > 0; --n, ++key) {
                        const int64_t kr = kv_row_base(table, a.max_pages, a.num_pages, a.kv_heads, hk, a.page_shift, key);
                        if (kr < 0) continue;                         // (the same for all lanes)
                        float dot = 0.f;
#pragma unroll 1
                        for (int d = g * (D / 4); d < (g + 1) * (D / 4); ++d) dot += (float)qr[d] * csign * kv_element<FMT>(a.k, a.k_exp, kr, D, d);
                        dot = row_sum(dot);
                        const bool sees = tree_window(a.mask ? a.mask + (int64_t)(sq.first + tok[rt]) * a.mask_stride : nullptr, a.mask_words, tok[rt], key - ctx) & 1;
                        if (!sees) continue;
                        const float mx = fmaxf(m[rt], dot);
                        const float alpha = m[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m[rt] - mx) * cabs);
                        const float mc = mx == -INFINITY ? 0.f : mx * cabs, p = __builtin_amdgcn_exp2f(fmaf(dot, cabs, -mc));
                        m[rt] = mx;
                        l[rt] = l[rt] * alpha + (g == 0 ? p : 0.f);
#pragma unroll
                        for (int t = 0; t < NB; ++t)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                o[rt][t][e] = (alpha == 1.f ? o[rt][t][e] : o[rt][t][e] * alpha) + p * kv_element<FMT>(a.v, a.v_exp, kr, D, g * (D / 4) + e * NB + t);
                    }
            }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) l[rt] = row_sum(l[rt]);
        // ---- the waves' sums meet: one maximum, then halves add in a fixed order
        if (nw > 1) {
            __syncthreads();
            if (g == 0) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) { stat[wave][rt][row][0] = m[rt]; stat[wave][rt][row][1] = l[rt]; }
            }
            __syncthreads();
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float mm = stat[0][rt][row][0];
                for (int w = 1; w < nw; ++w) mm = fmaxf(mm, stat[w][rt][row][0]);
                float ll = 0.f;
                for (int w = 0; w < nw; ++w) {
                    const float mw = stat[w][rt][row][0];
                    ll += stat[w][rt][row][1] * (mw == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((mw - mm) * cabs));      // (no maximum: 0 or NaN)
                }
                const float f = m[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m[rt] - mm) * cabs);
                if (m[rt] != -INFINITY && f != 1.f) {
#pragma unroll
                    for (int t = 0; t < NB; ++t) o[rt][t] *= f;
                }
                m[rt] = mm;
                l[rt] = ll;
            }
            for (int half = nw >> 1; half >= 1; half >>= 1) {
                if (wave >= half && wave < 2 * half) {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int t = 0; t < NB; ++t) osum[wave - half][rt * NB + t][lane] = o[rt][t];
                }
                __syncthreads();
                if (wave < half) {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int t = 0; t < NB; ++t) o[rt][t] += osum[wave][rt * NB + t][lane];
                }
                __syncthreads();
            }
        }
        if (wave == 0) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                if (at[rt] < 0) continue;
                const float mc = m[rt] == -INFINITY ? 0.f : m[rt] * cabs;
                if (a.nsplit > 1) {
                    float *po = a.part + ((int64_t)split * a.tokens * a.heads + at[rt]) * D + g * (D / 4);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int t = 0; t < NB; t += 2) *reinterpret_cast<kv_f32x2 *>(po + r * NB + t) = (kv_f32x2){o[rt][t][r], o[rt][t + 1][r]};
                    if (g == 0) {
                        float *ml = a.part + (int64_t)a.nsplit * a.tokens * a.heads * D + ((int64_t)split * a.tokens * a.heads + at[rt]) * 2;
                        ml[0] = l[rt] == 0.f ? -INFINITY : mc;        // (in units of log2)
                        ml[1] = l[rt];
                    }
                } else {
                    const float inv = l[rt] == 0.f ? 0.f : 1.f / l[rt];
                    T *po = static_cast<T *>(a.out) + at[rt] * D + g * (D / 4);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int t = 0; t < NB; ++t) po[r * NB + t] = (T)(l[rt] == 0.f ? 0.f : o[rt][t][r] * inv);
                    if (a.lse && g == 0) a.lse[at[rt]] = l[rt] == 0.f ? -INFINITY : (mc + __builtin_amdgcn_logf(l[rt])) * 0.693147180559945f;
                }
            }
        }
    }
}

// The splits' sums of one row meet: a wave per (token, head) of a sequence.  Rows of no sequence are left to the kernel above.
constexpr int TA_MAX_SPLITS = 128;

template <int DT, int D>
__global__ __launch_bounds__(256) void tree_attention_join_kernel(TreeAttnArgs a) {
    using T = typename ElemOf<DT>::type;
    constexpr int E = D < 64 ? 1 : D / 64;                            // neighbouring elements of a lane
    const int lane = threadIdx.x & 63;
    const uint32_t total = (uint32_t)a.tokens * (uint32_t)a.heads, at = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= total) return;
    const int32_t token = (int32_t)(at / (uint32_t)a.heads);
    const ScalarInts starts = (ScalarInts)a.starts;
    if (token < starts[0] || token >= starts[a.seqs]) return;
    const float *ml = a.part + (int64_t)a.nsplit * total * D + (int64_t)at * 2;
    float ms[2], ls[2];                                               // splits lane and lane + 64
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int s = lane + 64 * i;
        ms[i] = s < a.nsplit ? ml[(int64_t)s * total * 2] : -INFINITY;
        ls[i] = s < a.nsplit ? ml[(int64_t)s * total * 2 + 1] : 0.f;
    }
    float m = fmaxf(ms[0], ms[1]);
    for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    float f[2], l = 0.f, acc[E] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        f[i] = ms[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms[i] - m);
        l += f[i] * ls[i];
    }
    for (int o = 32; o >= 1; o >>= 1) l += __shfl_xor(l, o, 64);
    const float *po = a.part + (int64_t)at * D + (D < 64 ? lane & (D - 1) : lane * E);
#pragma unroll 8
    for (int s = 0; s < a.nsplit; ++s) {
        const float fs = __shfl(s < 64 ? f[0] : f[1], s & 63, 64);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += fs * po[(int64_t)s * total * D + e];
    }
    T *out = static_cast<T *>(a.out) + (int64_t)at * D + lane * E;
    if (lane * E < D) {
#pragma unroll
        for (int e = 0; e < E; ++e) out[e] = (T)(l == 0.f ? 0.f : acc[e] / l);
    }
    if (a.lse && lane == 0) a.lse[at] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.693147180559945f;
}

}  // namespace pocr
