// What the kernels that serve many sequences share (rotary.hip, pages.hip, kv8.hip, prompt.hip): batches' runs, the cache's geometry, argument checks.
#pragma once
#include <hip/hip_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>
#include "dev.h"

namespace {

constexpr int PAGE = L3M_PAGE;                                       // positions of a page
constexpr int BLOCK = 32;                                            // positions that share a scale
constexpr int SCALES = PAGE / BLOCK;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------- device: integers and lanes

// x / d by d's multiplier (host: multiplier), exact while x d < 2^32; 0: d is 1, or too large for it.
__host__ inline uint32_t multiplier(uint32_t d, uint64_t most) {
    return d > 1 && most * d < 1ull << 32 ? (uint32_t)((1ull << 32) / d) + 1 : 0;
}
__device__ __forceinline__ uint32_t divide(uint32_t x, uint32_t d, uint32_t mul) { return mul ? __umulhi(x, mul) : d == 1 ? x : x / d; }
__device__ __forceinline__ int clamp(int x, int lo, int hi) { return max(lo, min(x, hi)); }

__device__ __forceinline__ float bf16_float(uint32_t u) { return __uint_as_float(u << 16); }
// Two float32 values as bf16, the first in the low half; to the nearest, ties to even; NaN stays NaN.
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

// Inclusive sum over the lanes of a wavefront: within rows of 16, then each row's last lane onto the row behind, and lane 31 onto the upper half. Lanes that
// nothing comes to add 0.
template <int CTRL, int ROWS> __device__ __forceinline__ int dpp_or_0(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false); }
__device__ __forceinline__ int scan_wave(int x) {
    x += dpp_or_0<0x111, 0xF>(x);                                    // row_shr 1, 2, 4, 8
    x += dpp_or_0<0x112, 0xF>(x);
    x += dpp_or_0<0x114, 0xF>(x);
    x += dpp_or_0<0x118, 0xF>(x);
    x += dpp_or_0<0x142, 0xA>(x);                                    // row_bcast 15 into rows 1 and 3
    x += dpp_or_0<0x143, 0xC>(x);                                    // row_bcast 31 into rows 2 and 3
    return x;
}

// The largest of a wavefront's, in all lanes: within rows of 16 by moves, then over the halves.
template <int CTRL> __device__ __forceinline__ float dpp_move(float x) { return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xF, 0xF, true)); }
__device__ __forceinline__ float max_wave(float x) {
    x = fmaxf(x, dpp_move<0xB1>(x));                                 // lane ^ 1, lane ^ 2, the half row and the row mirrored
    x = fmaxf(x, dpp_move<0x4E>(x));
    x = fmaxf(x, dpp_move<0x141>(x));
    x = fmaxf(x, dpp_move<0x140>(x));
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// The exponents of a softmax are fma(s, scale, -m), m the rounded product of the largest score: off by half a unit of m, alike for all of a row and so for no
// result's sake, while that is small. From here on it isn't, and both are rounded alike (x scale - m).
constexpr float LARGE_SCORE = 16777216.f;
__device__ __forceinline__ float scaled_less(float x, float scale, float m) {
#pragma clang fp contract(off)
    const float y = x * scale;
    return y - m;
}

// A batch as kernels take it: starts whatever they hold are brought into 0 .. n, in order.
struct Runs {
    const int32_t *ids, *starts;
    int seqs, n;
    __device__ __forceinline__ int id(int i) const { return ids ? ids[i] : i; }
    __device__ __forceinline__ int from(int i) const { return clamp(starts[i], 0, n); }
    __device__ __forceinline__ int to(int i, int first) const { return clamp(starts[i + 1], first, n); }
};
inline Runs runs_of(const l3m_batch *b) { return {b->ids, b->starts, b->seqs, b->n}; }
// The run that holds item `item` of the runs' items one behind the other, count(run, first row, rows) each, and the item's place in it. run < 0: there are
// fewer items. Up to 64 runs are counted by each wavefront for itself, a lane a run; of more the W wavefronts of a workgroup, which then all look for the same
// item, count 64 each and meet in LDS.
struct Found {
    int run, at, s0, rows;
};
constexpr int MOST_ITEMS = 1 << 26;                                  // of a wavefront's 64 runs; a call has fewer, unless its runs overlap
template <int W, class Count> __device__ __forceinline__ Found find_run(const Runs &b, int item, Count count) {
    __shared__ int   sums_s[2][W];
    __shared__ Found found_s;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool alone = b.seqs <= 64;
    int base = 0;
    for (int r0 = 0, turn = 0; r0 < b.seqs; r0 += 64 * W, turn ^= 1) {
        const int r = r0 + (alone ? 0 : 64 * wave) + lane;
        int s0 = 0, rows = 0, c = 0;
        if (r < b.seqs) {
            s0 = b.from(r);
            rows = b.to(r, s0) - s0;
            c = count(r, s0, rows);
        }
        const int sum = scan_wave(c);
        int upto = sum, all = __builtin_amdgcn_readlane(sum, 63);
        if (!alone) {
            if (lane == 0) sums_s[turn][wave] = min(all, MOST_ITEMS);
            __syncthreads();
            upto += base;
            all = base;
#pragma unroll
            for (int w = 0; w < W; w++) {
                const int x = sums_s[turn][w];
                upto += w < wave ? x : 0;
                all += x;
            }
        }
        if (all > item) {
            const uint64_t past = __ballot(upto > item && upto - c <= item);
            Found f = {r - lane, 0, 0, 0};
            if (past) {
                const int l = __builtin_ctzll(past);
                f = {f.run + l, item - __builtin_amdgcn_readlane(upto - c, l), __builtin_amdgcn_readlane(s0, l), __builtin_amdgcn_readlane(rows, l)};
            }
            if (alone) return f;
            if (past && lane == 0) found_s = f;
            __syncthreads();
            return {__builtin_amdgcn_readfirstlane(found_s.run), __builtin_amdgcn_readfirstlane(found_s.at), __builtin_amdgcn_readfirstlane(found_s.s0),
                    __builtin_amdgcn_readfirstlane(found_s.rows)};
        }
        base = all;
    }
    return {-1, 0, 0, 0};
}

// ---------------------------------------------------------------- the cache's geometry

__host__ __device__ constexpr int padded(int hd) { return (hd + 31) & ~31; }
__host__ __device__ inline size_t layer_bytes(int nkv, int hd) { return ((size_t)nkv * (2 * PAGE * padded(hd) + 2 * SCALES) + 255) & ~(size_t)255; }
// A (page, layer, kv head)'s planes: K codes [128][HP], V codes [HP][128], the scales' exponents of K [4] and of V [4].
struct Unit {
    uint8_t *k, *v, *s;
};
__device__ __forceinline__ Unit unit_of(const l3m_kv8 &c, int page, int layer, int h) {
    const int hp = padded(c.hd);
    uint8_t *at = c.mem + ((size_t)page * c.layers + layer) * layer_bytes(c.nkv, c.hd);
    uint8_t *k = at + (size_t)h * 2 * PAGE * hp;
    return {k, k + PAGE * hp, at + (size_t)c.nkv * 2 * PAGE * hp + 2 * SCALES * h};
}

// ---------------------------------------------------------------- host: argument checks

inline bool overlap(const void *a, size_t na, const void *b, size_t nb) {
    return a && b && na && nb && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}
// The stream of a call that names none: the library's, made now if this is its first call. False: there is no device, or it was shut down.
inline bool stream_of(void *s, hipStream_t &st) {
    if (!s && l3m_dev_init()) {
        l3m_dev_fail("no usable device, or the library was shut down");
        return false;
    }
    st = (hipStream_t)(s ? s : l3m_dev_stream());
    return true;
}
inline size_t value_bytes(int dtype) { return dtype == L3M_HIP_F32 ? 4 : dtype == L3M_HIP_BF16 ? 2 : 0; }
// The bytes of n rows of `width` values, `stride` values apart.
inline size_t rows_bytes(int n, long long stride, long long width, size_t size) { return n > 0 ? ((size_t)(n - 1) * stride + width) * size : 0; }
inline const char *batch_bad(const l3m_batch *b) {
    if (!b || b->seqs < 0 || b->n < 0 || b->seqs > 65536 || b->n > 1 << 28) return "batch: counts out of range";
    if (b->seqs && !b->starts) return "batch: no starts";
    if (((uintptr_t)b->ids | (uintptr_t)b->starts) % 4) return "batch: ids and starts must be 4-byte aligned";
    return nullptr;
}
inline bool on_batch(const l3m_batch *b, const void *p, size_t n) {
    return overlap(p, n, b->ids, 4 * (size_t)b->seqs) || overlap(p, n, b->starts, 4 * ((size_t)b->seqs + 1));
}
inline const char *kv8_bad(const l3m_kv8 *c) {
    if (!c || !l3m_kv8_bytes(c->pages, c->layers, c->nkv, c->hd)) return "kv8: not a cache: hd a multiple of 8 up to 256, pages up to 2^20, layers and kv heads up to 4096";
    if (!c->mem || (uintptr_t)c->mem % 256) return "kv8: a cache without memory, or not 256-byte aligned";
    return nullptr;
}
inline bool on_cache(const l3m_kv8 *c, const void *p, size_t n) { return overlap(p, n, c->mem, l3m_kv8_bytes(c->pages, c->layers, c->nkv, c->hd)); }
inline const char *pages_bad(const l3m_pages *p) {
    if (!p || !l3m_pages_bytes(p->pages, p->seqs, p->width)) return "pages: not tables: pages up to 2^20, sequences up to 65536, pages of a sequence up to 2^20, 2^28 entries in all";
    if (!p->refs || !p->table || !p->len || !p->state || !p->scratch) return "pages: tables without memory";
    if (((uintptr_t)p->refs | (uintptr_t)p->table | (uintptr_t)p->len | (uintptr_t)p->state | (uintptr_t)p->scratch) % 16) return "pages: tables must be 16-byte aligned";
    return nullptr;
}
constexpr size_t STATE_INTS = 64;
inline size_t scratch_ints(int pages, int seqs) { return 4 * (size_t)pages + 2 * (size_t)seqs; }
inline bool on_pages(const l3m_pages *p, const void *m, size_t n) {
    return overlap(m, n, p->refs, 4 * (size_t)p->pages) || overlap(m, n, p->table, 4 * (size_t)p->seqs * p->width) || overlap(m, n, p->len, 4 * (size_t)p->seqs) ||
           overlap(m, n, p->state, 4 * STATE_INTS) || overlap(m, n, p->scratch, 4 * scratch_ints(p->pages, p->seqs));
}
// What is wrong with a cache and tables that a call takes together, or NULL.
inline const char *paged_bad(const l3m_kv8 *c, const l3m_pages *p) {
    if (const char *why = kv8_bad(c)) return why;
    if (const char *why = pages_bad(p)) return why;
    if (p->pages > c->pages) return "pages: the tables count more pages than the cache has";
    if (on_pages(p, c->mem, l3m_kv8_bytes(c->pages, c->layers, c->nkv, c->hd))) return "pages: the tables overlap the cache";
    return nullptr;
}

}  // namespace
