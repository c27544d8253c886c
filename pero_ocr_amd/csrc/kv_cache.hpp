// kv_cache.hpp — paged cache of attention keys and values, in bfloat16 or in 8 bits with one scale per row: quantise on write,
// restore on read.  The rows an attention kernel reads are found through kv_row_base().
//
// Layout: [page][kv_head][page_size][head_dim], k and v apart, so that the keys of one head in one page are one contiguous piece
// (page_size * head_dim bytes in 8 bits: 8 KB for 64 x 128) and a kernel that serves one head streams whole 128-byte lines.  Slot s is
// row s % page_size of page s / page_size.
//
// 8 bits: a row x (one token, one head) is stored as e4m3 codes c and ONE power of two, x ~= c * 2^(exp - 127):
//   s = min { s >= -100 : max |x| <= 448 * 2^s },  exp = s + 127,  c = round_to_nearest_even(x * 2^-s)
// A power of two costs no relative precision (e4m3's is the same in every binade; an arbitrary scale would buy at most one bit at the
// far lower end of its 18 binades) and makes every step but the one rounding exact: x * 2^-s, c * 2^s, and - what the attention
// kernel lives on - any product of a code with 2^s in bfloat16 (4 significant bits).  The rounding is off by at most half a step,
// 2^-4 relative to the value, or 2^-10 * 2^s below 2^-6 * 2^s.  An element that is not finite becomes NaN and does not count for s.
#pragma once
#include <stdint.h>
#ifdef __HIP__
#include <hip/hip_runtime.h>
#define POCR_HD __host__ __device__ __forceinline__
#else
#define POCR_HD inline              // (the index arithmetic is compiled by a host test too)
#endif

namespace pocr {

// Row number (in units of head_dim elements, also the index of the row's exponent) of position `pos` of a sequence for head `head`,
// or -1 when its page is absent: a table entry outside the cache, or a position outside the table, is never followed.
POCR_HD int64_t kv_row_base(const int32_t *table, int32_t max_pages, int32_t num_pages, int32_t kv_heads, int32_t head, int page_shift, int64_t pos) {
    const int64_t e = pos >> page_shift;
    if (pos < 0 || e >= max_pages) return -1;
    const int32_t page = table[e];
    if (page < 0 || page >= num_pages) return -1;
    return ((((int64_t)page * kv_heads + head) << page_shift) + (pos & (((int64_t)1 << page_shift) - 1)));
}

// The same for a slot number of the whole cache.
POCR_HD int64_t kv_slot_row(int64_t slot, int32_t num_pages, int32_t kv_heads, int32_t head, int page_shift) {
    const int64_t page = slot >> page_shift;
    if (slot < 0 || page >= num_pages) return -1;
    return ((page * kv_heads + head) << page_shift) + (slot & (((int64_t)1 << page_shift) - 1));
}

}  // namespace pocr

#ifdef __HIP__
namespace pocr {

enum { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };          // = POCR_F32, POCR_BF16, POCR_F16
enum { KV_BF16 = 0, KV_FP8 = 1 };                      // = POCR_KV_BF16, POCR_KV_FP8

template <int DT> struct ElemOf;
template <> struct ElemOf<DT_F32> { using type = float; };
template <> struct ElemOf<DT_BF16> { using type = __bf16; };
template <> struct ElemOf<DT_F16> { using type = _Float16; };

typedef float kv_f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t kv_u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t kv_u32x4 __attribute__((ext_vector_type(4)));

// E consecutive elements as floats; VEC: the address is a multiple of 16 bytes
template <int DT, bool VEC, int E> __device__ __forceinline__ void load_row(const void *p, float (&x)[E]) {
    using T = typename ElemOf<DT>::type;
    const T *e = static_cast<const T *>(p);
    if constexpr (VEC) {
        alignas(16) T t[E];
        constexpr int N = sizeof(t) / 16;
#pragma unroll
        for (int i = 0; i < N; ++i) reinterpret_cast<kv_u32x4 *>(t)[i] = reinterpret_cast<const kv_u32x4 *>(p)[i];
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = (float)t[i];
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = (float)e[i];
    }
}

template <int DT, int E> __device__ __forceinline__ void store_row(void *p, const float (&x)[E]) {
    using T = typename ElemOf<DT>::type;
    alignas(16) T t[E];
#pragma unroll
    for (int i = 0; i < E; ++i) t[i] = (T)x[i];
    constexpr int N = sizeof(t) / 16;
#pragma unroll
    for (int i = 0; i < N; ++i) reinterpret_cast<kv_u32x4 *>(p)[i] = reinterpret_cast<const kv_u32x4 *>(t)[i];
}

__device__ __forceinline__ float kv_scale(uint8_t exp) { return __uint_as_float((uint32_t)exp << 23); }

// exp of a row whose largest finite |value| is a (see the head of this file): 448 = 1.75 * 2^8
__device__ __forceinline__ int kv_exponent(float a) {
    const uint32_t u = __float_as_uint(a);
    const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < 27 ? 27 : e;
}

struct KvWriteArgs {
    void *k, *v;
    uint8_t *k_exp, *v_exp;
    const void *k_in, *v_in;
    const void *slots;
    int64_t k_ts, k_hs, v_ts, v_hs;          // element strides of a token and of a head
    int32_t num_pages, kv_heads, page_shift;
    uint32_t rows;                           // tokens * 2 * kv_heads
    int32_t slots64;
};

// D / 16 lanes own a row, 16 elements each (16384 tokens x 8 heads x 128 in bfloat16: 19.2 us = 5.2 TB/s, as a large copy reaches; with 8 elements
// a lane 23.4 us).  Rows in the order (token, k or v, head), as the projection that made them lies in memory.
constexpr int KV_WRITE_ELEMS = 16, KV_READ_ELEMS = 8;

template <int DT, int FMT, int D, bool VEC>
__global__ __launch_bounds__(256) void kv_write_kernel(KvWriteArgs a) {
    constexpr int LPR = D / KV_WRITE_ELEMS, RPB = 256 / LPR;
    const uint32_t r = blockIdx.x * RPB + threadIdx.x / LPR;
    if (r >= a.rows) return;
    const int c = (threadIdx.x % LPR) * KV_WRITE_ELEMS;
    const uint32_t hk = (uint32_t)a.kv_heads;
    const uint32_t t2 = r / hk, head = r - t2 * hk, token = t2 >> 1, is_v = t2 & 1;
    const int64_t slot = a.slots64 ? static_cast<const int64_t *>(a.slots)[token] : static_cast<const int32_t *>(a.slots)[token];
    const int64_t row = kv_slot_row(slot, a.num_pages, a.kv_heads, (int32_t)head, a.page_shift);
    using T = typename ElemOf<DT>::type;
    const T *in = static_cast<const T *>(is_v ? a.v_in : a.k_in) + (int64_t)token * (is_v ? a.v_ts : a.k_ts) + (int64_t)head * (is_v ? a.v_hs : a.k_hs) + c;
    float x[KV_WRITE_ELEMS];
    load_row<DT, VEC>(in, x);
    if constexpr (FMT == KV_BF16) {
        if (row >= 0) store_row<DT_BF16>(static_cast<__bf16 *>(is_v ? a.v : a.k) + row * D + c, x);
    } else {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < KV_WRITE_ELEMS; ++i) {
            const float ax = fabsf(x[i]);
            m = fmaxf(m, ax <= 3.402823466e38f ? ax : 0.f);          // (false for NaN and infinities)
        }
#pragma unroll
        for (int off = LPR / 2; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
        const int exp = kv_exponent(m);
        const float inv = __uint_as_float((uint32_t)(254 - exp) << 23);
#pragma unroll
        for (int i = 0; i < KV_WRITE_ELEMS; ++i) {
            const float y = x[i] * inv;
            x[i] = fabsf(x[i]) <= 3.402823466e38f ? y : __builtin_nanf("");
        }
        kv_u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
            w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], lo, true);
        }
        if (row >= 0) {
            *reinterpret_cast<kv_u32x4 *>(static_cast<uint8_t *>(is_v ? a.v : a.k) + row * D + c) = w;
            if (c == 0) (is_v ? a.v_exp : a.k_exp)[row] = (uint8_t)exp;
        }
    }
}

struct KvReadArgs {
    const void *k, *v;
    const uint8_t *k_exp, *v_exp;
    void *k_out, *v_out;                     // [tokens][kv_heads][D]
    const void *slots;
    int32_t num_pages, kv_heads, page_shift;
    uint32_t rows;                           // tokens * 2 * kv_heads
    int32_t slots64;
};

// D / 8 lanes own a row (the same 16384 tokens: 18.6 us = 5.4 TB/s; 16 elements a lane: 19.0).
template <int DT, int FMT, int D>
__global__ __launch_bounds__(256) void kv_read_kernel(KvReadArgs a) {
    constexpr int LPR = D / KV_READ_ELEMS, RPB = 256 / LPR;
    const uint32_t r = blockIdx.x * RPB + threadIdx.x / LPR;
    if (r >= a.rows) return;
    const int c = (threadIdx.x % LPR) * KV_READ_ELEMS;
    const uint32_t hk = (uint32_t)a.kv_heads;
    const uint32_t t2 = r / hk, head = r - t2 * hk, token = t2 >> 1, is_v = t2 & 1;
    const int64_t slot = a.slots64 ? static_cast<const int64_t *>(a.slots)[token] : static_cast<const int32_t *>(a.slots)[token];
    const int64_t row = kv_slot_row(slot, a.num_pages, a.kv_heads, (int32_t)head, a.page_shift);
    float x[KV_READ_ELEMS] = {};
    if (row >= 0) {
        if constexpr (FMT == KV_BF16) {
            load_row<DT_BF16, true>(static_cast<const __bf16 *>(is_v ? a.v : a.k) + row * D + c, x);
        } else {
            const kv_u32x2 w = *reinterpret_cast<const kv_u32x2 *>(static_cast<const uint8_t *>(is_v ? a.v : a.k) + row * D + c);
            const float s = kv_scale((is_v ? a.v_exp : a.k_exp)[row]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const kv_f32x2 p = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false), q = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
                x[4 * i] = p[0] * s; x[4 * i + 1] = p[1] * s; x[4 * i + 2] = q[0] * s; x[4 * i + 3] = q[1] * s;
            }
        }
    }
    using T = typename ElemOf<DT>::type;
    store_row<DT>(static_cast<T *>(is_v ? a.v_out : a.k_out) + ((int64_t)token * hk + head) * D + c, x);
}

}  // namespace pocr
#endif  // __HIP__
