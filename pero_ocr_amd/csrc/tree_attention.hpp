// tree_attention.hpp — attention of the newest tokens of many sequences over their paged caches (kv_cache.hpp).
//
// Token i of a sequence with n new tokens and L cached positions (the new ones are the last n of them) sees the L - n older positions
// and, among the new ones, those its mask names (the ancestors in a tree of drafted tokens, itself among them); without a mask
// positions up to its own.  With s_j = scale * q . k_j over the seen j:  out = sum_j softmax(s)_j v_j,  lse = log sum_j exp(s_j);
// a token that sees nothing gets out = 0, lse = -inf.  Query head h reads key head h / (heads / kv_heads).
//
// One pass over the keys with a running reference (a maximum that lags by at most 2^8) and sum.  A wave owns RT * 16 rows (a row = one new token and one of the query heads that
// share the key head) and takes blocks of 32 keys; both products run on v_mfma_f32_16x16x32_bf16, transposed, so that a row is always
// lane & 15 and nothing is exchanged between lanes but, now and then, the row maximum:
//   S^T = K Q^T     lane (row, g = lane / 16) gets the scores of keys 4 g + r and 16 + 4 g + r of the block, r = 0..3
//   O^T = V^T P^T   takes exactly these eight probabilities as its operand when V^T is fed in the same key order
// No barrier in the loop: every wave fetches its own keys.  Which elements of K a step of 32 takes is free to choose, Q is laid out to match.  V goes
// straight into registers: a lane loads D / 16 neighbouring elements
// of eight keys and transposes them with byte permutes; tile c of the product then is elements c, D/16 + c, 2 D/16 + c, ... and a lane ends up with
// D / 4 neighbouring outputs of its row.
// 8-bit codes become bfloat16 exactly, by v_cvt_scalef32 with the key's own power of two.
// What is rounded: the probability enters the second product as bf16 planes, two for 16-bit queries: at most 2^-17 of it (rounding to the first leaves up
// to 2^-8, of which half a step is 2^-17 - 24 trees in bfloat16 204.7 us; cut instead 2^-16 and 203.8, and 0.35 % of the outputs round to a neighbour
// of what the exact ones round to, not 0.19 %; one plane's 2^-8 would add as much error as rounding the result does); three for float32
// are exact, as are the two or three planes of a float16 or float32 query.  Scores, statistics and sums are float32.
//
// What bounds it (8 key heads; calls one after the other): four sequences of 60 to 131 thousand keys of 128 in 8 bits, one token each, 169 us = 5.3 TB/s: the
// memory; 24 trees of 28 to 256 rows over 0.5 to 9 thousand keys of 128 in bfloat16 200 us, half of it matrix instructions (two planes of the
// probabilities) and conversions, which every wave repeats for its 32 rows, the rest waits for the address unit; one tree of 132 rows over 4129 keys of
// 128 in 8 bits 18.3 us (5 or 6 blocks a wave, one on its way at a time) and 512 single tokens over 40 to 272 keys of 64, fp32, 25 us (2 to 9 blocks
// a wave), where the start and the end of a workgroup (4 us) weigh most.  A chain takes all blocks of its sequence for every row tile and masks what lies
// behind the tile's own tokens: 2048 new tokens, nothing before them, 32 heads over 8 of 128, 141 us for 57 us of products, of which the mask leaves half.
//
// A NaN or infinity in V spreads in a matrix product to the masked rows, whose probability is 0; testing every element for it costs more than the
// transposition, so the loop does not.  Finite values near the end of the range may pass it in a sum of up to 2^8 times each, where the
// average does not.  A wave whose sums come out not finite goes through its keys again one by one, every row with the keys that it sees, and sums
// the average itself: slow, and met only where such numbers are.  Waves and splits meet as averages, weighted with their share of the row's sum.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>
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
    float *part;                  // nsplit > 1: averages [nsplit][part_rows][D], then (maximum, sum) [nsplit][part_rows][2]
    int64_t q_ts, q_hs, table_stride, mask_stride, tokens;
    int32_t seqs, heads, kv_heads, num_pages, page_shift, max_pages, mask_words, zero_rest, nsplit, tiles;
    uint32_t slots, run, part_rows, tile_rows;
    float scale;
};

// Row of `part` for row r of a sequence and key head: that of the output (tile_rows = 0), or, where that is fewer rows (padding behind the last sequence
// has none then), `tile_rows` for each sequence and key head.
__device__ __forceinline__ uint32_t part_row(const TreeAttnArgs &a, int s, int hk, uint32_t r, int64_t to) {
    return a.tile_rows ? ((uint32_t)s * (uint32_t)a.kv_heads + (uint32_t)hk) * a.tile_rows + r : (uint32_t)to;
}

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

// lanes of a wave write and read each other's LDS words in the order of the program (no instruction: LDS serves a wave in order)
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

union Frag { uint32_t u[4]; ta_bf16x8 b; };

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    union { ta_bf16x2 b; uint32_t u; } r;
    r.b = (ta_bf16x2){(__bf16)lo, (__bf16)hi};
    return r.u;
}

// eight floats as NP bf16 planes, the last rounded, the others cut or (NEAR) rounded too: the rest is half as large then, but a number next to the end
// of the range would become infinite
template <bool NEAR, int NP> __device__ __forceinline__ void split_planes(const float (&x)[8], Frag (&f)[NP]) {
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
                f[p].u[j] = NEAR ? pack_bf16(y[2 * j], y[2 * j + 1]) : __builtin_amdgcn_perm(__float_as_uint(y[2 * j + 1]), __float_as_uint(y[2 * j]), 0x07060302u);
                y[2 * j] -= __uint_as_float(NEAR ? f[p].u[j] << 16 : __float_as_uint(y[2 * j]) & 0xffff0000u);
                y[2 * j + 1] -= __uint_as_float((NEAR ? f[p].u[j] : __float_as_uint(y[2 * j + 1])) & 0xffff0000u);
            }
        }
    }
}

__device__ __forceinline__ uint32_t fp8_pair(uint32_t w, float scale, bool high) {
    union { ta_bf16x2 b; uint32_t u; } r;
    r.b = high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false);
    return r.u;
}

// A block of 32 keys as a lane holds it: for V D / 16 elements (from lane & 15 on) of the eight keys 4 g + a and 16 + 4 g + a.  For K a lane
// needs its quarter of key (lane & 15) of both 16-key halves.  Fetched like that, every lane of an instruction asks for 16 bytes of another
// row, and the address unit takes a cycle for each.  With rows of 8 bits that is still the faster way (24 sequences of 4736 keys, 128
// rows each: 119 us); with bfloat16, twice the pieces, the lanes fetch neighbouring pieces and the block turns in the wave's part of
// LDS (177 -> 141 us; in 8 bits it would cost 131).
template <int FMT, int D> struct KvBlock {
    static constexpr int ES = FMT == KV_FP8 ? 1 : 2;
    static constexpr bool STAGED = FMT == KV_BF16;
    static constexpr int RB = D * ES, PR = RB / 16, KI = PR / 2;      // bytes and pieces of a row, pieces of K a lane fetches
    static constexpr int PITCH = RB + 16, STAGE = STAGED ? 32 * PITCH : 0;         // of the wave's part of LDS (16 rows at one piece: all 64 banks)
    static constexpr int VB = D * ES / 16;                            // bytes of V a lane holds per key
    static constexpr int VW = VB < 4 ? 1 : VB / 4;
    kv_u32x4 k[KI];
    uint32_t v[8][VW];
    uint32_t ke[2], ve[2];                                            // four keys' exponents: the lane's among them, its own four

    // base[h]: row number of key 0 of half h (of row 0 where the page is absent: in bounds, and masked by the caller); the same for the whole
    // wave, so that a lane's part of the address is a constant 32-bit offset
    __device__ __forceinline__ void load_keys(const TreeAttnArgs &a, const int64_t (&base)[2], uint32_t lane) {
        constexpr int HALF = KI / 2;                                  // pieces of a half
        const uint32_t i = lane & 15, g = lane >> 4;
        const uint8_t *kb[2] = {static_cast<const uint8_t *>(a.k) + base[0] * RB, static_cast<const uint8_t *>(a.k) + base[1] * RB};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (STAGED) {
#pragma unroll
                for (int c = 0; c < HALF; ++c) k[h * HALF + c] = *reinterpret_cast<const kv_u32x4 *>(kb[h] + (c * 64 + lane) * 16);
            } else {
                if constexpr (D == 32) *(reinterpret_cast<kv_u32x2 *>(k) + h) = *reinterpret_cast<const kv_u32x2 *>(kb[h] + i * RB + g * 8);
                else {
#pragma unroll
                    for (int c = 0; c < HALF; ++c) k[h * HALF + c] = *reinterpret_cast<const kv_u32x4 *>(kb[h] + (i * RB + g * 16) + c * 64);
                }
                ke[h] = *reinterpret_cast<const uint32_t *>(a.k_exp + base[h] + (lane & 12));
            }
        }
    }
    __device__ __forceinline__ void stage_keys(uint8_t *stage, uint32_t lane) const {
#pragma unroll
        for (int c = 0; c < KI; ++c) {
            const uint32_t q = c * 64 + lane;
            *reinterpret_cast<kv_u32x4 *>(stage + q / PR * PITCH + q % PR * 16) = k[c];
        }
    }
    __device__ __forceinline__ void load_values(const TreeAttnArgs &a, const int64_t (&base)[2], uint32_t lane) {
        const uint32_t i = lane & 15, g = lane >> 4;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint8_t *vb = static_cast<const uint8_t *>(a.v) + base[h] * (D * ES);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                uint32_t *w = v[4 * h + t];
                const uint8_t *p = vb + (g * (4 * D * ES) + i * VB) + t * (D * ES);
                if constexpr (VB == 2) w[0] = *reinterpret_cast<const uint16_t *>(p);
                else if constexpr (VB == 4) w[0] = *reinterpret_cast<const uint32_t *>(p);
                else if constexpr (VB == 8) *reinterpret_cast<kv_u32x2 *>(w) = *reinterpret_cast<const kv_u32x2 *>(p);
                else {
#pragma unroll
                    for (int c = 0; c < VB / 16; ++c) *reinterpret_cast<kv_u32x4 *>(w + 4 * c) = *reinterpret_cast<const kv_u32x4 *>(p + 16 * c);
                }
            }
            if constexpr (FMT == KV_FP8) ve[h] = *reinterpret_cast<const uint32_t *>(a.v_exp + base[h] + 4 * g);
        }
    }
    // operands of the first product: steps STEPS * c .. of the keys of half h (a step: 32 elements), from one piece of every key
    static constexpr int STEPS = D == 32 ? 1 : 2 / ES, PIECES = D / 32 / STEPS;
    __device__ __forceinline__ void keys(const uint8_t *stage, int h, int c, uint32_t lane, Frag (&f)[STEPS]) const {
        if constexpr (STAGED) {
            *reinterpret_cast<kv_u32x4 *>(f[0].u) = *reinterpret_cast<const kv_u32x4 *>(stage + (16 * h + (lane & 15)) * PITCH + (4 * c + (lane >> 4)) * 16);
        } else {
            const float s = __uint_as_float(__builtin_amdgcn_ubfe(ke[h], (lane & 3) * 8, 8) << 23);
            const uint32_t *w = reinterpret_cast<const uint32_t *>(k) + 2 * STEPS * (h * PIECES + c);
#pragma unroll
            for (int j = 0; j < 2 * STEPS; ++j) {
                f[j / 2].u[2 * (j & 1)] = fp8_pair(w[j], s, false);
                f[j / 2].u[2 * (j & 1) + 1] = fp8_pair(w[j], s, true);
            }
        }
    }
    // element of a row that operand element j of step st stands for
    __device__ static __forceinline__ int key_elem(int g, int st) {
        if constexpr (FMT == KV_BF16) return st * 32 + g * 8;
        else if constexpr (D == 32) return g * 8;
        else return (st >> 1) * 64 + g * 16 + (st & 1) * 8;
    }
    // operands of the second product: the TW tiles made of dword w of every key
    static constexpr int TW = VB < 4 ? 2 : 4 / ES;
    __device__ __forceinline__ void values(int w, Frag (&f)[TW]) const {
        uint32_t x[8][TW / 2];                                        // neighbouring pairs of every key's elements, in bfloat16
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            if constexpr (FMT == KV_FP8) {
                const float s = kv_scale((uint8_t)(ve[t >> 2] >> (8 * (t & 3))));
                x[t][0] = fp8_pair(v[t][w], s, false);
                if constexpr (TW == 4) x[t][1] = fp8_pair(v[t][w], s, true);
            } else x[t][0] = v[t][w];
        }
#pragma unroll
        for (int c = 0; c < TW / 2; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f[2 * c].u[j] = __builtin_amdgcn_perm(x[2 * j + 1][c], x[2 * j][c], 0x05040100u);
                f[2 * c + 1].u[j] = __builtin_amdgcn_perm(x[2 * j + 1][c], x[2 * j][c], 0x07060302u);
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

// NW: waves of a workgroup, which take the key blocks in turn
template <int DT, int FMT, int D, int RT, int NW>
__global__ __launch_bounds__(64 * NW, D <= 128 ? 2 : 1) void tree_attention_kernel(TreeAttnArgs a) {
    using T = typename ElemOf<DT>::type;
    using Block = KvBlock<FMT, D>;
    constexpr int QP = DT == DT_F32 ? 3 : DT == DT_F16 ? 2 : 1;      // planes of the query
    constexpr int PP = DT == DT_F32 ? 3 : 2;                         // planes of the probabilities
    constexpr int NB = D / 16, ST = D / 32, TW = Block::TW;
    // The low plane of a float16 query lies in LDS, the same for all waves, where two tiles of 128 would not fit the registers of two waves a SIMD with it
    // (13 to 24 of them went to scratch memory).
    constexpr bool QLOW = DT == DT_F16 && RT == 2 && D == 128;
    constexpr int QR = QLOW ? 1 : QP;                                // planes in registers
    __shared__ kv_u32x4 qlow[QLOW ? RT * ST * 64 : 1];
    const int tid = threadIdx.x, lane = tid & 63, row = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    constexpr int PITCH = D + 4;                                      // (16 rows, four words each: all 64 banks)
    constexpr int OSUM = NW * RT * 16 * PITCH * 4, STAGES = NW * Block::STAGE;
    __shared__ __attribute__((aligned(16))) uint8_t memory[OSUM > STAGES ? OSUM : STAGES];     // the waves' keys; behind the loop their sums
    float (*osum)[RT * 16][PITCH] = reinterpret_cast<float (*)[RT * 16][PITCH]>(memory);
    uint8_t *stage = memory + wave * Block::STAGE;
    __shared__ float stat[NW][RT * 16][2], whole[RT * 16][2];
    __shared__ int64_t place_of[RT * 16];

    if (a.zero_rest) {                                                // rows of no sequence, a share for every workgroup; 1: out and lse, 2: lse alone
        const int32_t end = min(max(((ScalarInts)a.starts)[a.seqs], 0), (int32_t)a.tokens);
        const int64_t from = (int64_t)end * a.heads, rest = (a.tokens - end) * a.heads, all = (int64_t)gridDim.x * (64 * NW);
        constexpr int PIECES = D * sizeof(T) / 16;
        if (a.zero_rest != 2)
            for (int64_t p = (int64_t)blockIdx.x * (64 * NW) + tid; p < rest * PIECES; p += all) static_cast<kv_u32x4 *>(a.out)[from * PIECES + p] = (kv_u32x4){0, 0, 0, 0};
        if (a.lse)
            for (int64_t p = (int64_t)blockIdx.x * (64 * NW) + tid; p < rest; p += all) a.lse[from + p] = -INFINITY;
    }

    // A list of slots for each key head and split.  Row tiles of one sequence and key head read the same keys, so they should share an L2, and consecutive
    // workgroups go to different XCDs: every list stays on one XCD (run = 0; the XCD's lists side by side, so that unused slots come
    // last), or runs of `run` slots do.  With one tile a sequence, key heads are next to each other instead: no XCD has a long sequence to itself.
    const uint32_t kv_heads = (uint32_t)a.kv_heads, group = (uint32_t)a.heads / kv_heads, rest8 = blockIdx.x >> 3, xcd = blockIdx.x & 7;
    uint32_t list, slot;
    if (a.run == 0) {
        const uint32_t own = kv_heads * (uint32_t)a.nsplit / 8;       // lists of an XCD
        slot = rest8 / own;
        list = (rest8 - slot * own) * 8 + xcd;
    } else {
        const uint32_t turn = rest8 / a.run, number = (turn * 8 + xcd) * a.run + (rest8 - turn * a.run);
        if (a.tiles == 1) {
            const uint32_t at = number / kv_heads, split0 = at / a.slots;
            slot = at - split0 * a.slots;
            list = split0 * kv_heads + (number - at * kv_heads);
        } else {
            list = number / a.slots;
            slot = number - list * a.slots;
        }
    }
    const int split = (int)(list / kv_heads), hk = (int)(list - (uint32_t)split * kv_heads);
    if (split >= a.nsplit) return;
    // Slots: `tiles` for each sequence, or (tiles = 0) as many as its rows need, counted where a wave has a lane for each sequence; where not, sequence
    // s begins at slot_of(first row), which leaves it one more than its whole tiles.
    auto slot_of = [&](int32_t first, int i) { return (uint32_t)min(max(first, 0), (int32_t)a.tokens) * group / (16 * RT) + (uint32_t)i; };
    int s = 0;
    uint32_t first_slot = 0;
    if (a.tiles) s = (int)(slot / (uint32_t)a.tiles);
    else if (a.seqs <= 64) {
        const int32_t total = (int32_t)a.tokens, b = min(max(a.starts[min(lane, a.seqs - 1)], 0), total), e = min(a.starts[min(lane, a.seqs - 1) + 1], total);
        const int own = lane < a.seqs ? (int)(((uint32_t)max(e - b, 0) * group + 16 * RT - 1) / (16 * RT)) : 0;
        int until = own;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const int before = __shfl_up(until, o, 64);
            until += lane >= o ? before : 0;
        }
        s = (int)__popcll(__ballot(until <= (int)slot));
        if (s >= a.seqs) return;
        first_slot = (uint32_t)__builtin_amdgcn_readlane(until - own, s);
    } else {
        int left = a.seqs;
        while (left > 1) {                                            // the last sequence that begins at or before this slot: 64 looked at in a step
            const int step = (left + 63) / 64, at = s + min(lane * step, left - 1);
            const int n = (int)__popcll(__ballot(lane * step < left && slot_of(a.starts[at], at) <= slot)), skip = max(n - 1, 0) * step;
            s += skip;
            left = min(step, left - skip);
        }
        s = __builtin_amdgcn_readfirstlane(s);
    }
    const TreeSeq sq = tree_seq(a, s);
    const uint32_t rows = (uint32_t)sq.n * group, tile0 = slot - (a.tiles ? (uint32_t)(s * a.tiles) : a.seqs <= 64 ? first_slot : slot_of(sq.first, s));
    if (tile0 >= (rows + 16 * RT - 1) / (16 * RT)) return;            // an unused slot, or a sequence without new tokens
    const int32_t *table = a.table + s * a.table_stride;
    // scores in units of log2: the sign of the scale goes to the query, so that the largest product is the largest score; 0 makes the query 0
    const float c = a.scale * 1.44269504088896f;
    const float csign = c == 0.f ? 0.f : c < 0.f ? -1.f : 1.f, cabs = c == 0.f ? 1.f : fabsf(c);
    const uint32_t qkeep = c == 0.f ? 0u : ~0u, qflip = c < 0.f ? 0x80008000u : 0u;          // the same for bfloat16 queries, on the bits

    const int32_t blocks = (int32_t)(((uint32_t)sq.len + 31u) >> 5), per = (int32_t)(((uint32_t)blocks + a.nsplit - 1u) / (uint32_t)a.nsplit);
    const int32_t ctx = sq.len - sq.n;

    // (a second turn: the sequence has more new tokens than the caller said.  With tile_rows their splits have no room in `part`: the splits' workgroups
    // take whole tiles in turn)
    for (uint32_t r0 = tile0 * (16 * RT), turn = 0; r0 < rows; r0 += a.tiles ? (uint32_t)a.tiles * (16 * RT) : rows, ++turn) {
        const bool whole_tile = turn > 0 && a.tile_rows > 0;
        if (whole_tile && (turn - 1) % (uint32_t)a.nsplit != (uint32_t)split) continue;
        const int32_t first_block = whole_tile ? 0 : min(split * per, blocks), end_block = whole_tile ? blocks : min(first_block + per, blocks);
        int32_t tok[RT];
        int64_t at[RT];                                               // row of out, -1: none
        Frag q[RT][ST][QR];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const uint32_t r = r0 + 16 * rt + row, rr = min(r, rows - 1);
            tok[rt] = (int32_t)(rr / group);
            const int head = hk * (int)group + (int)(rr - (uint32_t)tok[rt] * group);
            at[rt] = r < rows ? (int64_t)(sq.first + tok[rt]) * a.heads + head : -1;
            const T *qr = static_cast<const T *>(a.q) + (int64_t)(sq.first + tok[rt]) * a.q_ts + head * a.q_hs;
#pragma unroll
            for (int st = 0; st < ST; ++st) {
                if constexpr (DT == DT_BF16) {
                    *reinterpret_cast<kv_u32x4 *>(q[rt][st][0].u) = *reinterpret_cast<const kv_u32x4 *>(qr + Block::key_elem(g, st));
#pragma unroll
                    for (int j = 0; j < 4; ++j) q[rt][st][0].u[j] = (q[rt][st][0].u[j] & qkeep) ^ qflip;
                } else {
                    float x[8];
                    load_row<DT, true>(qr + Block::key_elem(g, st), x);
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] *= csign;
                    if constexpr (QLOW) {
                        Frag f[QP];
                        split_planes<false>(x, f);
                        q[rt][st][0] = f[0];
                        if (wave == 0) qlow[(rt * ST + st) * 64 + lane] = *reinterpret_cast<const kv_u32x4 *>(f[1].u);
                    } else split_planes<false>(x, q[rt][st]);
                }
            }
        }
        if constexpr (QLOW) __syncthreads();

        ta_f32x4 o[RT][NB];
        float m[RT], l[RT];                                           // m: of the raw scores (x csign); l: this lane's keys only
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            m[rt] = -INFINITY;
            l[rt] = 0.f;
#pragma unroll
            for (int t = 0; t < NB; ++t) o[rt][t] = (ta_f32x4){0.f, 0.f, 0.f, 0.f};
        }
        // A block's keys are requested as soon as the registers of the last one's are free, behind its scores, and its values behind its sums;
        // the page ids of the block after that are on their way meanwhile.
        const ScalarInts pages = (ScalarInts)table;
        auto page_ids = [&](int32_t b, int32_t (&id)[2]) {            // (a block without keys: any entry of the table)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int32_t key = (int32_t)min(((uint32_t)b << 5) + 16u * h, (uint32_t)sq.len - 1u);
                id[h] = pages[key >> a.page_shift];                   // (len <= max_pages * page_size)
            }
        };
        auto place = [&](int32_t b, const int32_t (&id)[2], int64_t (&base)[2], uint32_t &there) {
            const int32_t key0 = b << 5;
            there = low_bits(sq.len - key0);                          // keys that exist at all
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bool good = (uint32_t)id[h] < (uint32_t)a.num_pages;
                const int32_t page = good ? id[h] : 0;
                base[h] = (((int64_t)page * a.kv_heads + hk) << a.page_shift) + ((key0 + 16 * h) & ((1 << a.page_shift) - 1));
                if (!good) there &= h ? 0x0000ffffu : 0xffff0000u;
            }
        };
        Block kv;
        int64_t base[2];
        int32_t ids[2];
        uint32_t there = 0;
        if (first_block + wave < end_block) {
            page_ids(first_block + wave, ids);
            place(first_block + wave, ids, base, there);
            kv.load_keys(a, base, lane);
            __builtin_amdgcn_sched_barrier(0);                        // (in the loop's order, or its waits would cover both)
            kv.load_values(a, base, lane);
            page_ids(first_block + wave + NW, ids);
        }
        for (int32_t b = first_block + wave; b < end_block; b += NW) {
                const int32_t key0 = b << 5;
                int64_t next[2];
                uint32_t next_there = 0;
                // (behind the last block it is requested again, from the cache: a load that a branch may skip would have to be waited for with
                // all younger ones)
                place(b + NW, ids, next, next_there);
                if (b + NW >= end_block) {
                    next[0] = base[0];
                    next[1] = base[1];
                }
                const bool edge = there != ~0u || key0 + 31 >= ctx;   // some key is not seen by every row
                ta_f32x4 sc[RT][2];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) sc[rt][0] = sc[rt][1] = (ta_f32x4){0.f, 0.f, 0.f, 0.f};
                uint32_t low_at = lane;
                if constexpr (QLOW) asm volatile("" : "+v"(low_at));  // (or it would be read ahead of the loop, into registers again)
                if constexpr (Block::STAGED) {
                    wave_order();
                    kv.stage_keys(stage, lane);
                    wave_order();
                }
#pragma unroll
                for (int c = 0; c < Block::PIECES; ++c) {
                    Frag low[Block::STEPS][RT];
                    if constexpr (QLOW) {
#pragma unroll
                        for (int st = 0; st < Block::STEPS; ++st)
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt) *reinterpret_cast<kv_u32x4 *>(low[st][rt].u) = qlow[(rt * ST + c * Block::STEPS + st) * 64 + low_at];
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        Frag kf[Block::STEPS];
                        kv.keys(stage, h, c, lane, kf);
#pragma unroll
                        for (int st = 0; st < Block::STEPS; ++st)
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt) {
                                if constexpr (QLOW) sc[rt][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[st].b, low[st][rt].b, sc[rt][h], 0, 0, 0);
#pragma unroll
                                for (int pl = QR - 1; pl >= 0; --pl)
                                    sc[rt][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[st].b, q[rt][c * Block::STEPS + st][pl].b, sc[rt][h], 0, 0, 0);
                            }
                    }
                }
                kv.load_keys(a, next, lane);
                page_ids(b + 2 * NW, ids);                            // (not earlier: a wait for LDS is one for these too)
                float p[RT][8];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) p[rt][j] = sc[rt][j >> 2][j & 3];
                    if (edge) {
                        int32_t d0 = key0 - ctx;
                        asm volatile("" : "+s"(d0));                  // (nothing of this is worth computing ahead)
                        const uint32_t vis = there & tree_window(a.mask ? a.mask + (int64_t)(sq.first + tok[rt]) * a.mask_stride : nullptr, a.mask_words, tok[rt], d0);
#pragma unroll
                        for (int j = 0; j < 8; ++j) p[rt][j] = vis >> ((j >> 2) * 16 + 4 * g + (j & 3)) & 1 ? p[rt][j] : -INFINITY;
                    }
                    float mx = p[rt][0];
#pragma unroll
                    for (int j = 1; j < 8; ++j) mx = fmaxf(mx, p[rt][j]);
                    // the reference moves only when a score passes it by more than 2^8: the sums hold that, and the lanes need not meet otherwise
                    if (__ballot((mx - m[rt]) * cabs > 8.f)) {
                        mx = fmaxf(m[rt], row_max(mx));
                        const float alpha = m[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m[rt] - mx) * cabs);
                        l[rt] *= alpha;
#pragma unroll
                        for (int t = 0; t < NB; ++t) o[rt][t] *= alpha;
                        m[rt] = mx;
                    }
                    // (2^-inf is 0; without a reference yet it is 0)
                    const float mc = m[rt] == -INFINITY ? 0.f : m[rt] * cabs;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        p[rt][j] = __builtin_amdgcn_exp2f(fmaf(p[rt][j], cabs, -mc));
                        l[rt] += p[rt][j];
                    }
                }
                if (there != ~0u) kv.drop_values(there, g);
                Frag pf[RT][PP];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) split_planes<PP == 2>(p[rt], pf[rt]);          // (three are exact either way)
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
                __builtin_amdgcn_sched_barrier(0);
                kv.load_values(a, next, lane);
                base[0] = next[0];
                base[1] = next[1];
                there = next_there;
        }
        float odd = 0.f;                                              // NaN if a sum is not finite
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int t = 0; t < NB; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) odd = fmaf(o[rt][t][r], 0.f, odd);
        float share[RT];                                              // what o is to be weighted with: 1, or the wave's sum where o is an average already
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) share[rt] = 1.f;
        if (__ballot(odd != odd)) {                                          // key by key, each row only with what it sees: its sum first, then the average
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                m[rt] = -INFINITY;
                share[rt] = 0.f;
#pragma unroll
                for (int t = 0; t < NB; ++t) o[rt][t] = (ta_f32x4){0.f, 0.f, 0.f, 0.f};
                const uint32_t rr = min(r0 + 16 * rt + row, rows - 1);
                const T *qr = static_cast<const T *>(a.q) + (int64_t)(sq.first + tok[rt]) * a.q_ts + (hk * (int)group + (int)(rr - (uint32_t)tok[rt] * group)) * a.q_hs;
#pragma unroll 1
                for (int turn = 0; turn < 2; ++turn) {
                    const float inv = share[rt] == 0.f ? 0.f : 1.f / share[rt];
                    for (int32_t b = first_block + wave; b < end_block; b += NW)
                        for (int32_t key = b << 5, n = min(32, sq.len - key); n > 0; --n, ++key) {
                            const int64_t kr = kv_row_base(table, a.max_pages, a.num_pages, a.kv_heads, hk, a.page_shift, key);
                            if (kr < 0) continue;                     // (the same for all lanes)
                            float dot = 0.f;
#pragma unroll 1
                            for (int d = g * (D / 4); d < (g + 1) * (D / 4); ++d) dot += (float)qr[d] * csign * kv_element<FMT>(a.k, a.k_exp, kr, D, d);
                            dot = row_sum(dot);
                            const bool sees = tree_window(a.mask ? a.mask + (int64_t)(sq.first + tok[rt]) * a.mask_stride : nullptr, a.mask_words, tok[rt], key - ctx) & 1;
                            if (!sees) continue;
                            const float mx = fmaxf(m[rt], dot), mc = mx == -INFINITY ? 0.f : mx * cabs, p = __builtin_amdgcn_exp2f(fmaf(dot, cabs, -mc));
                            if (turn == 0) {
                                share[rt] = share[rt] * (m[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m[rt] - mx) * cabs)) + p;
                                m[rt] = mx;
                            } else {
#pragma unroll
                                for (int t = 0; t < NB; ++t)
#pragma unroll
                                    for (int e = 0; e < 4; ++e) o[rt][t][e] += p * inv * kv_element<FMT>(a.v, a.v_exp, kr, D, g * (D / 4) + e * NB + t);
                            }
                        }
                }
                l[rt] = g == 0 ? share[rt] : 0.f;
            }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) l[rt] = row_sum(l[rt]);
        // ---- the waves' sums meet in LDS: one maximum per row, then every thread adds its share of the outputs in a fixed order and writes it
        // in whole lines
        if (g == 0) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                stat[wave][16 * rt + row][0] = m[rt];
                stat[wave][16 * rt + row][1] = l[rt];
                if (wave == 0) place_of[16 * rt + row] = at[rt];
            }
        }
        __syncthreads();
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float mm = -INFINITY, ll = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) mm = fmaxf(mm, stat[w][16 * rt + row][0]);
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float mw = stat[w][16 * rt + row][0];
                ll += stat[w][16 * rt + row][1] * (mw == mm || mw == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((mw - mm) * cabs));      // (no maximum: 0 or NaN)
            }
            // (averages: of finite values they are finite, however many there are)
            const float f = (m[rt] == mm || m[rt] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m[rt] - mm) * cabs)) * share[rt] * (ll == 0.f ? 0.f : 1.f / ll);
            float *dst = &osum[wave][16 * rt + row][g * (D / 4)];
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int t = 0; t < NB; t += 2) *reinterpret_cast<kv_f32x2 *>(dst + r * NB + t) = (kv_f32x2){o[rt][t][r] * f, o[rt][t + 1][r] * f};
            if (wave == 0 && g == 0) {
                whole[16 * rt + row][0] = mm == -INFINITY ? 0.f : mm * cabs;                  // (in units of log2)
                whole[16 * rt + row][1] = ll;
            }
        }
        __syncthreads();
#pragma unroll 1
        for (int e = tid; e < RT * 16 * (D / 4); e += 64 * NW) {
            const int rr = e / (D / 4), d = e % (D / 4) * 4;
            const int64_t to = place_of[rr];
            if (to < 0) continue;
            ta_f32x4 v = *reinterpret_cast<const ta_f32x4 *>(&osum[0][rr][d]);
#pragma unroll
            for (int w = 1; w < NW; ++w) v += *reinterpret_cast<const ta_f32x4 *>(&osum[w][rr][d]);
            const float mc = whole[rr][0], ll = whole[rr][1];
            if (a.nsplit > 1 && !whole_tile) {
                const int64_t pr = (int64_t)split * a.part_rows + part_row(a, s, hk, r0 + (uint32_t)rr, to);
                *reinterpret_cast<ta_f32x4 *>(a.part + pr * D + d) = v;
                if (d == 0) {
                    float *ml = a.part + (int64_t)a.nsplit * a.part_rows * D + pr * 2;
                    ml[0] = ll == 0.f ? -INFINITY : mc;
                    ml[1] = ll;
                }
            } else {
                alignas(16) T x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = (T)(ll == 0.f ? 0.f : v[j]);
                T *po = static_cast<T *>(a.out) + to * D + d;
                if constexpr (sizeof(T) == 4) *reinterpret_cast<kv_u32x4 *>(po) = *reinterpret_cast<const kv_u32x4 *>(x);
                else *reinterpret_cast<kv_u32x2 *>(po) = *reinterpret_cast<const kv_u32x2 *>(x);
                if (a.lse && d == 0) a.lse[to] = ll == 0.f ? -INFINITY : (mc + __builtin_amdgcn_logf(ll)) * 0.693147180559945f;
            }
        }
        __syncthreads();                                              // (the sums have been read: their place is the next rows' keys')
    }
}

// The splits' averages of one row meet: a wave per (token, head) of a sequence.  Rows of no sequence are left to the kernel above.  A chain of three round
// trips to memory: 4 us for 1056 rows of 6 splits.
constexpr int TA_MAX_SPLITS = 128;

template <int DT, int D>
__global__ __launch_bounds__(256) void tree_attention_join_kernel(TreeAttnArgs a) {
    using T = typename ElemOf<DT>::type;
    constexpr int E = D < 64 ? 1 : D / 64;                            // neighbouring elements of a lane
    const int lane = threadIdx.x & 63;
    // grid: tile_rows / 4, key heads, sequences; or all rows / 4
    const uint32_t total = a.part_rows, r = blockIdx.x * 4 + (threadIdx.x >> 6), at = (blockIdx.z * (uint32_t)a.kv_heads + blockIdx.y) * a.tile_rows + r;
    if (at >= total) return;
    const float *ml = a.part + (int64_t)a.nsplit * total * D + (int64_t)at * 2;
    float ms[2], ls[2];                                               // splits lane and lane + 64
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int s = lane + 64 * i;
        ms[i] = s < a.nsplit ? ml[(int64_t)s * total * 2] : -INFINITY;
        ls[i] = s < a.nsplit ? ml[(int64_t)s * total * 2 + 1] : 0.f;
    }
    int64_t to = at;                                                  // row of out
    if (a.tile_rows) {                                                // (asked behind the loads above, which stay within `part` also where the row is nobody's)
        const uint32_t group = (uint32_t)a.heads / (uint32_t)a.kv_heads, tok = r / group;
        const TreeSeq sq = tree_seq(a, (int)blockIdx.z);
        if (tok >= (uint32_t)sq.n) return;
        to = (int64_t)(sq.first + (int32_t)tok) * a.heads + blockIdx.y * group + (r - tok * group);
    } else {
        const int32_t token = (int32_t)(at / (uint32_t)a.heads);
        const ScalarInts starts = (ScalarInts)a.starts;
        if (token < starts[0] || token >= starts[a.seqs]) return;
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
#pragma unroll
    for (int i = 0; i < 2; ++i) f[i] = l == 0.f ? 0.f : f[i] * ls[i] / l;          // a split's share of the row
    const float *po = a.part + (int64_t)at * D + (D < 64 ? lane & (D - 1) : lane * E);
    auto add = [&](auto width) {                                      // sums on their way at once: a launch of few rows is a chain of round trips
        constexpr int U = decltype(width)::value;
        for (int s0 = 0; s0 < a.nsplit; s0 += U) {
            float x[U][E];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < E; ++e) x[u][e] = po[(int64_t)min(s0 + u, a.nsplit - 1) * total * D + e];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int s = s0 + u;
                const float fs = __shfl(s < 64 ? f[0] : f[1], s & 63, 64);
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] += s < a.nsplit ? fs * x[u][e] : 0.f;
            }
        }
    };
    if (a.nsplit <= 4) add(std::integral_constant<int, 4>());
    else add(std::integral_constant<int, 16>());
    T *out = static_cast<T *>(a.out) + to * D + lane * E;
    if (lane * E < D) {
#pragma unroll
        for (int e = 0; e < E; ++e) out[e] = (T)(l == 0.f ? 0.f : acc[e]);
    }
    if (a.lse && lane == 0) a.lse[to] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.693147180559945f;
}

}  // namespace pocr
