// decode_ops.hip — C entries (include/pocr.h "decoding operators") of the stand-alone operators on device memory of the caller:
// the paged key / value cache, attention of drafted tokens over it, scores of given tokens.  No engine, no host copies, no
// allocation and no synchronisation: every call checks its arguments, enqueues on the caller's stream and returns.
#include <hip/hip_runtime.h>
#include <cstdarg>
#include <cstdio>
#include <algorithm>
#include <type_traits>

#include "../../include/pocr.h"
#include "kv_cache.hpp"
#include "token_logprobs.hpp"
#include "tree_attention.hpp"

namespace pocr {
int set_error(const char *text);          // pocr_hip.hip: what pocr_last_error() returns on this thread; 1
}

using namespace pocr;

static_assert((int)POCR_F32 == DT_F32 && (int)POCR_BF16 == DT_BF16 && (int)POCR_F16 == DT_F16, "element types");
static_assert((int)POCR_KV_BF16 == KV_BF16 && (int)POCR_KV_FP8 == KV_FP8, "cache formats");

namespace {

int refuse(const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return set_error(buf);
}

// The caller's device for the length of a call (a thread's current device is left as it was).
struct OnDevice {
    int was = -1;
    bool changed = false;
    int enter(int device_id) {
        static const int n = [] { int c = 0; return hipGetDeviceCount(&c) == hipSuccess ? c : 0; }();
        if (n == 0) return refuse("no HIP device available: this library has no CPU fallback");
        if (device_id < 0 || device_id >= n) return refuse("device_id %d out of range (%d devices)", device_id, n);
        if (hipGetDevice(&was) != hipSuccess) return refuse("hipGetDevice failed");
        if (was != device_id) {
            if (hipSetDevice(device_id) != hipSuccess) return refuse("hipSetDevice(%d) failed", device_id);
            changed = true;
        }
        return 0;
    }
    ~OnDevice() { if (changed) (void)hipSetDevice(was); }
};

// the launch's own status: an error that some earlier call of the process left behind is not taken for this one's
template <class Args> int launch(const char *what, void (*kernel)(Args), dim3 grid, dim3 block, void *stream, Args args) {
    void *p[1] = {&args};
    const hipError_t e = hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, p, 0, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : refuse("%s: launch failed: %s", what, hipGetErrorString(e));
}

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
int elem_size(int dtype) { return dtype == POCR_F32 ? 4 : 2; }
bool known_dtype(int dtype) { return dtype == POCR_F32 || dtype == POCR_BF16 || dtype == POCR_F16; }

int page_shift(const pocr_kv_pages *c) { int s = 0; while ((1 << s) < c->page_size) ++s; return s; }

int check_pages(const pocr_kv_pages *c) {
    if (!c || !c->k || !c->v) return refuse("NULL cache");
    if (c->format != POCR_KV_BF16 && c->format != POCR_KV_FP8) return refuse("cache format %d: POCR_KV_BF16 or POCR_KV_FP8", c->format);
    if (c->format == POCR_KV_FP8 && (!c->k_exp || !c->v_exp)) return refuse("an 8-bit cache needs k_exp and v_exp");
    if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return refuse("head_dim %d: 32, 64, 128 or 256", c->head_dim);
    if (c->page_size < 16 || (c->page_size & (c->page_size - 1)) || c->page_size > 1 << 30) return refuse("page_size %d: a power of two from 16 on", c->page_size);
    if (c->num_pages < 1 || c->kv_heads < 1) return refuse("num_pages and kv_heads must be positive (got %d, %d)", c->num_pages, c->kv_heads);
    if (!aligned(c->k, 16) || !aligned(c->v, 16)) return refuse("the cache must start at a multiple of 16 bytes");
    if (c->format == POCR_KV_FP8 && (!aligned(c->k_exp, 4) || !aligned(c->v_exp, 4))) return refuse("k_exp and v_exp must start at a multiple of 4 bytes");
    return 0;
}

int check_rows(const pocr_kv_pages *c, int64_t tokens, const char *what) {
    if (tokens < 0) return refuse("%s: tokens %lld", what, (long long)tokens);
    if (tokens > ((int64_t)1 << 31) / (2 * (int64_t)c->kv_heads) - 128) return refuse("%s: 2 * tokens * kv_heads must stay below 2^31", what);
    // (8 elements a thread, and a launch has fewer than 2^32 threads)
    if (tokens * 2 * c->kv_heads * (c->head_dim / 8) > (int64_t)1 << 31) return refuse("%s: 2 * tokens * kv_heads * head_dim must not exceed 2^34", what);
    return 0;
}

template <int DT, int FMT, bool VEC> int write_by_dim(dim3 (*grid)(uint32_t, int), int D, void *stream, const KvWriteArgs &a) {
    const char *w = "pocr_kv_write";
    switch (D) {
        case 32: return launch(w, kv_write_kernel<DT, FMT, 32, VEC>, grid(a.rows, 32), dim3(256), stream, a);
        case 64: return launch(w, kv_write_kernel<DT, FMT, 64, VEC>, grid(a.rows, 64), dim3(256), stream, a);
        case 128: return launch(w, kv_write_kernel<DT, FMT, 128, VEC>, grid(a.rows, 128), dim3(256), stream, a);
        default: return launch(w, kv_write_kernel<DT, FMT, 256, VEC>, grid(a.rows, 256), dim3(256), stream, a);
    }
}

template <int DT, int FMT> int read_by_dim(dim3 (*grid)(uint32_t, int), int D, void *stream, const KvReadArgs &a) {
    const char *w = "pocr_kv_read";
    switch (D) {
        case 32: return launch(w, kv_read_kernel<DT, FMT, 32>, grid(a.rows, 32), dim3(256), stream, a);
        case 64: return launch(w, kv_read_kernel<DT, FMT, 64>, grid(a.rows, 64), dim3(256), stream, a);
        case 128: return launch(w, kv_read_kernel<DT, FMT, 128>, grid(a.rows, 128), dim3(256), stream, a);
        default: return launch(w, kv_read_kernel<DT, FMT, 256>, grid(a.rows, 256), dim3(256), stream, a);
    }
}

// workgroups for `rows` rows of D elements, E of them a lane
template <int E> dim3 row_grid(uint32_t rows, int D) { const uint32_t per = 256 / (D / E); return dim3((rows + per - 1) / per); }

// 32 rows a wave where their queries and sums leave room for two waves in a SIMD's registers
constexpr bool two_tiles(int dtype, int D) { return D <= 64 || (D == 128 && dtype != POCR_F32); }

// How the work of one attention call is cut.
struct AttendPlan { int rt, tiles, nsplit, waves; int64_t slots, run, groups, part_rows, tile_rows; };

AttendPlan attend_plan(const pocr_kv_pages *c, const pocr_tree_attention_args *t) {
    AttendPlan p;
    const int64_t average = (t->tokens + t->seqs - 1) / t->seqs, group = t->heads / c->kv_heads, known = std::min(t->max_queries, t->tokens);
    p.rt = (known > 0 ? known : average) * group > 16 && two_tiles(t->dtype, c->head_dim) ? 2 : 1;
    // Slots for row tiles: the same number for each sequence where that is not more than what their rows could need together (then nothing has to
    // be looked up: 2048 sequences of 8 tokens 510 us, looked up 615 us), or as many as its rows need (15 single tokens next to one of
    // 512: 82 us, slots for 512 in each 114 us; 256 single tokens of which nobody said so 53 us, slots for all of them in each 295 us).
    const int64_t all = t->tokens * group / (16 * p.rt), most = known > 0 ? (known * group + 16 * p.rt - 1) / (16 * p.rt) : all + 1;
    p.tiles = most * t->seqs <= all + t->seqs ? (int)most : 0;
    p.slots = p.tiles ? p.tiles * (int64_t)t->seqs : all + t->seqs;
    const int64_t units = (p.tiles ? p.slots : all + (t->seqs + 1) / 2) * c->kv_heads, blocks = (((int64_t)t->max_pages << page_shift(c)) + 31) / 32;
    // Splits for one workgroup on each CU, of 10 blocks of 32 keys or more: a workgroup costs about 4 us to start and to end (single tokens, 8 key
    // heads of 128, 8 query heads each; in brackets the rule's: 500 keys [1] 8.6 us, 2 splits 10.0; 2000 keys 1 split 17.3, 3 12.9, [6] 11.4;
    // 8 sequences of 4000 keys 1 split 29.8, 2 21.8, [4] 19.0, 6 20.6; 32 sequences [1] 47, 2 49).  Two workgroups on each where a split still is
    // 256 blocks, so that sequences of different lengths end together (60 to 131 thousand keys: 256 workgroups 186 us, 512 169 us, 768 172 us).
    // The lengths are on the device: the table's width stands for them.  In a table of 131072 positions one sequence of 500 keys takes 10.5 to 11 us (its
    // own width 8.5), of 2000 keys 10.7 to 11.2 (11.4), 8 of 500 keys 11.0 to 11.9 (8.6), 8 of 4000 keys 19.5 (19.1): where one split is best the join's
    // launch is lost, elsewhere more splits do as well.  A caller who knows the lengths passes the table's first columns.
    p.nsplit = (int)std::min<int64_t>(std::max({std::min(256 / units, blocks / 10), std::min(512 / units, blocks / 256), (int64_t)1}), TA_MAX_SPLITS);
    // Room for the splits of the rows that the slots hold (units * nsplit <= 512: at most 17 MB), not of all that a batch is padded to.
    p.tile_rows = p.tiles * (int64_t)(16 * p.rt);
    p.part_rows = p.tile_rows * t->seqs * c->kv_heads;
    if (p.tiles == 0 || p.part_rows >= t->tokens * t->heads) {
        p.tile_rows = 0;
        p.part_rows = t->tokens * t->heads;
    }
    // A wave alone where there are enough of them for 8 on a CU: nothing to join (512 single tokens over 40 to 272 keys 25.2 us, four waves 33.8;
    // 256 over 2000 keys 183 and 195).
    p.waves = p.rt == 1 && units >= 2048 ? 1 : 4;
    // Lists of slots, one for every key head and split: each on one XCD where 8 XCDs share them evenly (24 trees of 28 to 256 rows: 202 us, in runs of 8
    // slots 227, of 2 292, of 1 375), in runs of up to 16 where not.
    const int64_t lists = (int64_t)c->kv_heads * p.nsplit, work = p.slots * lists;
    p.run = p.tiles == 1 || lists % 8 ? 1 : 0;
    while (p.tiles != 1 && p.run > 0 && p.run < 16 && work / p.run >= 128) p.run *= 2;
    p.groups = p.run ? (work + 8 * p.run - 1) / (8 * p.run) * (8 * p.run) : work;
    return p;
}

int64_t attend_workspace(const pocr_kv_pages *c, const AttendPlan &p) { return p.nsplit == 1 ? 0 : p.nsplit * p.part_rows * (c->head_dim + 2) * 4; }

template <int DT, int FMT, int D> int attend(const AttendPlan &p, void *stream, const TreeAttnArgs &a) {
    const char *w = "pocr_tree_attention";
    const dim3 grid((unsigned)p.groups), block(64 * p.waves);
    constexpr int RT = two_tiles(DT, D) ? 2 : 1;
    const int rc = p.waves == 1 ? launch(w, tree_attention_kernel<DT, FMT, D, 1, 1>, grid, block, stream, a)
                   : p.rt == 1  ? launch(w, tree_attention_kernel<DT, FMT, D, 1, 4>, grid, block, stream, a)
                                : launch(w, tree_attention_kernel<DT, FMT, D, RT, 4>, grid, block, stream, a);
    if (rc || p.nsplit == 1) return rc;
    return launch(w, tree_attention_join_kernel<DT, D>, p.tile_rows ? dim3(a.tile_rows / 4, a.kv_heads, a.seqs) : dim3((unsigned)((p.part_rows + 3) / 4)), dim3(256), stream, a);
}

template <int DT, int FMT> int attend_by_dim(int D, const AttendPlan &p, void *stream, const TreeAttnArgs &a) {
    switch (D) {
        case 32: return attend<DT, FMT, 32>(p, stream, a);
        case 64: return attend<DT, FMT, 64>(p, stream, a);
        case 128: return attend<DT, FMT, 128>(p, stream, a);
        default: return attend<DT, FMT, 256>(p, stream, a);
    }
}

int check_attention(const pocr_kv_pages *c, const pocr_tree_attention_args *t) {
    if (check_pages(c)) return 1;
    if (!t) return refuse("pocr_tree_attention: NULL arguments");
    if (!known_dtype(t->dtype)) return refuse("pocr_tree_attention: dtype %d", t->dtype);
    if (t->tokens < 0 || t->tokens > 0x7fffffff || t->seqs < 0) return refuse("pocr_tree_attention: tokens %lld, seqs %d", (long long)t->tokens, t->seqs);
    if (t->heads < 1 || t->heads % c->kv_heads) return refuse("pocr_tree_attention: heads %d must be a multiple of the cache's %d key heads", t->heads, c->kv_heads);
    if (t->max_pages < 0) return refuse("pocr_tree_attention: max_pages %d", t->max_pages);
    if (t->tokens > 0 && t->seqs == 0) return refuse("pocr_tree_attention: tokens without a sequence");
    if ((int64_t)t->seqs * c->kv_heads > 1 << 20 || t->tokens * t->heads > 1 << 27)
        return refuse("pocr_tree_attention: seqs * kv_heads exceeds 2^20 or tokens * heads 2^27");
    return 0;
}

// Rows of one call: HIP's limit of 2^32 threads to a launch, for what a row of so many classes may take.
int64_t score_rows(int classes) { return ((int64_t)1 << 32) / (classes <= 512 ? 16 : classes <= 4096 ? 64 : classes <= 32768 ? 256 : 1024); }

int check_scores(const pocr_token_logprobs_args *t) {
    if (!t) return refuse("pocr_token_logprobs: NULL arguments");
    if (!known_dtype(t->dtype)) return refuse("pocr_token_logprobs: dtype %d", t->dtype);
    if (t->rows < 0 || t->rows > 0x7fffffff) return refuse("pocr_token_logprobs: rows %lld", (long long)t->rows);
    if (t->classes < 1 || t->classes > 1 << 30) return refuse("pocr_token_logprobs: classes %d", t->classes);
    if (t->rows >= score_rows(t->classes))
        return refuse("pocr_token_logprobs: rows %lld: with %d classes fewer than %lld", (long long)t->rows, t->classes, (long long)score_rows(t->classes));
    if (t->given < 0) return refuse("pocr_token_logprobs: given %d", t->given);
    if (t->top < 0 || t->top > LP_MAX_TOP || t->top > t->classes) return refuse("pocr_token_logprobs: top %d must be in 0..%d and at most the classes", t->top, LP_MAX_TOP);
    return 0;
}

// Workgroups of a row: more than one where rows are too few to fill the chip and so long that one workgroup (36 GB/s) takes longer than
// the second launch and the join (time on the GPU: 9 rows of 151003 in fp32, top 8: whole 16.0 us, in slices 11.6; 64 of 152000 in bf16 16.1 and 12.9;
// 100 of 152000 19.5 and 19.2.  Between 65536 and 98304 classes it depends on top: 8 rows of 80000, top 5, 11.5 and 10.6, top 64 13.7 and 15.7;
// there a row stays whole, which needs no scratch memory), up to four on each CU (64 rows of 400000 in fp32: 256 workgroups 41 us,
// 512 28.3, 1024 27.4, whole 39), of 8192 classes or more.
int score_slices(const pocr_token_logprobs_args *t) {
    if (t->classes <= 98304 || t->rows >= 128) return 1;
    return (int)std::min<int64_t>({(1024 + t->rows - 1) / t->rows, t->classes / 8192, 64, LP_CAND / std::max(t->top, 1)});
}

int64_t score_workspace(const pocr_token_logprobs_args *t) {
    const int64_t parts = t->rows * score_slices(t);
    return parts == t->rows ? 0 : parts * (16 + 8 * (int64_t)t->top);
}

// Few classes in registers: 16 lanes a row where there are rows enough for every SIMD (36864 rows of 232 in fp32, top 4: 12.3 us, with 64 lanes
// 23.9), 64 lanes where not (600 rows: 4.1 us, with 16 4.8; even at 2400).  An alternative costs a pass over the registers, so above 256 classes only
// to 8 of them (500 classes, fp32: top 4 22.7 us against 33.5 by a wave that looks among the largest, top 8 32 and 35, top 20 62 and 47), and
// with 16-bit logits, whose single loads are half as wide, only for few rows (500 classes, top 8: 48 us against 39).
// Otherwise a wave (rows enough, and a row too short for more: 2000 classes in fp32, top 4 86 us, with 256 threads 110; 4000 classes 170 and
// 156; and few enough alternatives for a threshold among the maxima of 64 lanes to leave a short list, without which every alternative is a pass over
// the row: 16384 rows of 1200 in fp32, top 26 41.7 us and 46.8, top 28 91.7 and 47.6, top 32 377 and 48.3, top 64 734 and 57.7), 256 threads (600 rows of 1000 classes, top 20: 7.2 us, a wave 12.1), or 1024 (1024 rows of 131072 in bf16, top 20: 52.7 us, with 256
// 67.3; 3000 rows of 32000 68.5 and 52.6).
template <int DT> int score(void *stream, const LogprobArgs &a) {
    const char *w = "pocr_token_logprobs";
    const int64_t rows = a.rows;
    auto few = [&](void (*kernel)(LogprobArgs), int lanes) { return launch(w, kernel, dim3((unsigned)((rows * lanes + 255) / 256)), dim3(256), stream, a); };
    auto row = [&](void (*kernel)(LogprobArgs), int threads) {
        return launch(w, kernel, dim3((unsigned)std::min<int64_t>(rows, LP_GRID), (unsigned)((rows + LP_GRID - 1) / LP_GRID)), dim3(threads), stream, a);
    };
    if (a.C <= 256) return rows > 2048 ? few(token_logprobs_few_kernel<DT, 16, 16>, 16) : few(token_logprobs_few_kernel<DT, 64, 4>, 64);
    if (a.C <= 1024 && a.top <= 8 && rows <= 4096) return a.C <= 512 ? few(token_logprobs_few_kernel<DT, 64, 8>, 64) : few(token_logprobs_few_kernel<DT, 64, 16>, 64);
    if constexpr (DT == DT_F32)
        if (a.C <= 512 && a.top <= 8) return few(token_logprobs_few_kernel<DT, 16, 32>, 16);
    if (a.C <= 2048 && rows > 2048 && a.top <= LP_WAVE_TOP) return row(token_logprobs_kernel<DT, 64>, 64);
    if (a.C <= 32768) return row(token_logprobs_kernel<DT, 256>, 256);
    if (a.slices == 1) return row(token_logprobs_kernel<DT, 1024>, 1024);
    if (launch(w, token_logprobs_kernel<DT, 256, true>, dim3((unsigned)(rows * a.slices)), dim3(256), stream, a)) return 1;
    return launch(w, token_logprobs_join_kernel<DT>, dim3((unsigned)rows), dim3(256), stream, a);
}

}  // namespace

extern "C" {

int pocr_kv_write(int device_id, void *stream, const pocr_kv_pages *c, const pocr_kv_rows *t) {
    if (check_pages(c)) return 1;
    if (!t) return refuse("pocr_kv_write: NULL arguments");
    if (check_rows(c, t->tokens, "pocr_kv_write")) return 1;
    if (!known_dtype(t->dtype)) return refuse("pocr_kv_write: dtype %d", t->dtype);
    if (t->tokens == 0) return 0;
    if (!t->k || !t->v || !t->slots) return refuse("pocr_kv_write: NULL pointer");
    const int es = elem_size(t->dtype), dtype = t->dtype;
    if (!aligned(t->k, es) || !aligned(t->v, es) || !aligned(t->slots, t->slots64 ? 8 : 4)) return refuse("pocr_kv_write: a pointer is not aligned to its element");
    OnDevice dev;
    if (dev.enter(device_id)) return 1;
    KvWriteArgs a{c->k, c->v, c->k_exp, c->v_exp, t->k, t->v, t->slots, t->k_token_stride, t->k_head_stride, t->v_token_stride, t->v_head_stride,
                  c->num_pages, c->kv_heads, page_shift(c), (uint32_t)(t->tokens * 2 * c->kv_heads), t->slots64};
    // 16-byte loads where every row starts at a multiple of 16 bytes, single elements otherwise
    const bool vec = aligned(t->k, 16) && aligned(t->v, 16) && (t->k_token_stride * es) % 16 == 0 && (t->k_head_stride * es) % 16 == 0 &&
                     (t->v_token_stride * es) % 16 == 0 && (t->v_head_stride * es) % 16 == 0;
    auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (c->format == POCR_KV_FP8) return vec ? write_by_dim<DT, KV_FP8, true>(row_grid<KV_WRITE_ELEMS>, c->head_dim, stream, a) : write_by_dim<DT, KV_FP8, false>(row_grid<KV_WRITE_ELEMS>, c->head_dim, stream, a);
        return vec ? write_by_dim<DT, KV_BF16, true>(row_grid<KV_WRITE_ELEMS>, c->head_dim, stream, a) : write_by_dim<DT, KV_BF16, false>(row_grid<KV_WRITE_ELEMS>, c->head_dim, stream, a);
    };
    if (dtype == POCR_F32) return go(std::integral_constant<int, DT_F32>());
    if (dtype == POCR_BF16) return go(std::integral_constant<int, DT_BF16>());
    return go(std::integral_constant<int, DT_F16>());
}

int pocr_kv_read(int device_id, void *stream, const pocr_kv_pages *c, const void *slots, int32_t slots64, int64_t tokens, void *k, void *v, int32_t dtype) {
    if (check_pages(c) || check_rows(c, tokens, "pocr_kv_read")) return 1;
    if (!known_dtype(dtype)) return refuse("pocr_kv_read: dtype %d", dtype);
    if (tokens == 0) return 0;
    if (!k || !v || !slots) return refuse("pocr_kv_read: NULL pointer");
    if (!aligned(k, 16) || !aligned(v, 16) || !aligned(slots, slots64 ? 8 : 4)) return refuse("pocr_kv_read: k and v must start at a multiple of 16 bytes");
    OnDevice dev;
    if (dev.enter(device_id)) return 1;
    KvReadArgs a{c->k, c->v, c->k_exp, c->v_exp, k, v, slots, c->num_pages, c->kv_heads, page_shift(c), (uint32_t)(tokens * 2 * c->kv_heads), slots64};
    auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        return c->format == POCR_KV_FP8 ? read_by_dim<DT, KV_FP8>(row_grid<KV_READ_ELEMS>, c->head_dim, stream, a) : read_by_dim<DT, KV_BF16>(row_grid<KV_READ_ELEMS>, c->head_dim, stream, a);
    };
    if (dtype == POCR_F32) return go(std::integral_constant<int, DT_F32>());
    if (dtype == POCR_BF16) return go(std::integral_constant<int, DT_BF16>());
    return go(std::integral_constant<int, DT_F16>());
}

int64_t pocr_tree_attention_workspace(const pocr_kv_pages *c, const pocr_tree_attention_args *t) {
    if (check_attention(c, t)) return -1;
    if (t->tokens == 0) return 0;
    return attend_workspace(c, attend_plan(c, t));
}

int pocr_tree_attention(int device_id, void *stream, const pocr_kv_pages *c, const pocr_tree_attention_args *t) {
    if (check_attention(c, t)) return 1;
    if (t->mask && t->mask_words < 1) return refuse("pocr_tree_attention: mask_words %d", t->mask_words);
    if (t->tokens == 0) return 0;
    if (!t->q || !t->out || !t->lengths || !t->q_start || (t->max_pages > 0 && !t->page_table)) return refuse("pocr_tree_attention: NULL pointer");
    const int es = elem_size(t->dtype);
    if (!aligned(t->q, 16) || (t->q_token_stride * es) % 16 || (t->q_head_stride * es) % 16) return refuse("pocr_tree_attention: rows of q must start at multiples of 16 bytes");
    if (!aligned(t->out, 16) || !aligned(t->lse, 4) || !aligned(t->mask, 8) || !aligned(t->lengths, 4) || !aligned(t->q_start, 4) || !aligned(t->page_table, 4))
        return refuse("pocr_tree_attention: a pointer is not aligned to its element (out: to 16 bytes)");
    const AttendPlan p = attend_plan(c, t);
    const int64_t need = attend_workspace(c, p);
    if (need > 0 && (!t->workspace || !aligned(t->workspace, 16) || t->workspace_bytes < need))
        return refuse("pocr_tree_attention: a workspace of %lld bytes, aligned to 16, is needed (pocr_tree_attention_workspace)", (long long)need);
    OnDevice dev;
    if (dev.enter(device_id)) return 1;
    TreeAttnArgs a{t->q, c->k, c->v, c->k_exp, c->v_exp, t->page_table, t->lengths, t->q_start, t->mask, t->out, t->lse, static_cast<float *>(t->workspace),
                   t->q_token_stride, t->q_head_stride, t->page_table_stride, t->mask_stride, t->tokens, t->seqs, t->heads, c->kv_heads, c->num_pages, page_shift(c),
                   t->max_pages, t->mask_words, t->zero_rest, p.nsplit, p.tiles, (uint32_t)p.slots, (uint32_t)p.run, (uint32_t)p.part_rows,
                   (uint32_t)p.tile_rows, t->scale};
    auto go = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        return c->format == POCR_KV_FP8 ? attend_by_dim<DT, KV_FP8>(c->head_dim, p, stream, a) : attend_by_dim<DT, KV_BF16>(c->head_dim, p, stream, a);
    };
    if (t->dtype == POCR_F32) return go(std::integral_constant<int, DT_F32>());
    if (t->dtype == POCR_BF16) return go(std::integral_constant<int, DT_BF16>());
    return go(std::integral_constant<int, DT_F16>());
}

int64_t pocr_token_logprobs_workspace(const pocr_token_logprobs_args *t) {
    if (check_scores(t)) return -1;
    return t->rows == 0 ? 0 : score_workspace(t);
}

int pocr_token_logprobs(int device_id, void *stream, const pocr_token_logprobs_args *t) {
    if (check_scores(t)) return 1;
    if (t->rows == 0) return 0;
    if (!t->logits || !t->entropy || (t->given > 0 && (!t->tokens || !t->logprob)) || (t->top > 0 && (!t->top_logprob || !t->top_index)))
        return refuse("pocr_token_logprobs: NULL pointer");
    if (!aligned(t->logits, elem_size(t->dtype)) || !aligned(t->tokens, t->tokens64 ? 8 : 4)) return refuse("pocr_token_logprobs: a pointer is not aligned to its element");
    const int64_t need = score_workspace(t);
    if (need > 0 && (!t->workspace || !aligned(t->workspace, 16) || t->workspace_bytes < need))
        return refuse("pocr_token_logprobs: a workspace of %lld bytes, aligned to 16, is needed (pocr_token_logprobs_workspace)", (long long)need);
    OnDevice dev;
    if (dev.enter(device_id)) return 1;
    const int slices = score_slices(t), slice = ((t->classes + slices - 1) / slices + 63) / 64 * 64;
    LogprobArgs a{t->logits, t->row_stride, t->tokens, t->logprob, t->entropy, t->top_logprob, t->top_index, t->rows, t->classes, t->given, t->top, t->tokens64,
                  t->dtype, slices, slice, static_cast<float *>(t->workspace)};
    if (t->dtype == POCR_F32) return score<DT_F32>(stream, a);
    if (t->dtype == POCR_BF16) return score<DT_BF16>(stream, a);
    return score<DT_F16>(stream, a);
}

}  // extern "C"
