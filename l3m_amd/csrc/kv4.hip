// A K/V cache of 4-bit blocks for CDNA4 (gfx950): the norm and rotation of query and key heads, the writer that stores K and V rows
// behind it in the same pass, the read-back, and the attention of one token or many over the cache.
//
// Layout. Per kv head, tiles of 32 positions; NB = ceil(hd / 32) blocks of 32 dimensions, a last block short of dimensions filled
// with zeros. A tile is laid out as the matrix cores' operands, so a lane's words are one contiguous load and no value crosses lanes:
// Half f of a tile is its positions 8 (m / 4) + 4 f + m % 4, m = 0 .. 15.
//   K codes   q4_0   [nkv][tile][half 2][lane 64][NB words]    lane 16 c + m: word b holds dimensions 32 b + 8 c .. + 7
//             mxfp4  [nkv][tile][half 2][NB][m 16][4 words]    a block as it is
//   V codes   q4_0   [nkv][tile][lane 64][2 NB words]          lane 16 g + j: word t holds dimension 16 t + j of positions 8 g .. 8 g + 7,
//                                                              position i at bit 4 (i / 2) + 16 (i % 2): pairs of f16 halves
//             mxfp4  the same shape                            word 2 b + u: dimensions 32 b + j (low nibbles) and 32 b + 16 + j of
//                                                              positions 8 g + 4 u .. + 3, a position's two in a byte
//   scales    q4_0   [nkv][tile][NB][32 positions]             f16 d, of K and of V
//             mxfp4  [nkv][tile][NB][m 16][half 2] of K, [nkv][tile][NB][32 positions] of V: a biased exponent byte, 0 of a block of zeros
// Both codes of a tile and head take 512 NB bytes. Dimension i of a word of K is the nibble at bit nib(dt, i): q4_0's masked bytes are then
// dimensions 0..3 and 4..7, mxfp4's come in order.
#include <hip/hip_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>
#include <type_traits>
#include "dev.h"
#include "format.h"

namespace {

constexpr int TILE = 32;                                             // positions of a tile
constexpr int HD_MAX = 256;
constexpr int E8M0_NAN = 255;                                        // reads as infinity times code 0

__host__ __device__ constexpr int sbytes(int dt) { return dt == L3M_Q4_0 ? 2 : 1; }
__host__ __device__ constexpr int nib(int dt, int i) { return dt == L3M_Q4_0 ? 8 * (i & 3) + (i & 4) : 4 * i; }

// One kv head's planes.
struct Head {
    uint32_t *kq, *vq;
    uint8_t  *ks, *vs;
};
__device__ __forceinline__ Head head_of(const l3m_kv4 &c, int nb, int sb, int h) {
    const size_t tiles = ((size_t)c.cap + TILE - 1) / TILE, words = tiles * 128 * nb, scales = tiles * TILE * nb * sb;
    return {(uint32_t *)c.kq + h * words, (uint32_t *)c.vq + h * words, c.ks + h * scales, c.vs + h * scales};
}
// The word of K that holds dimensions d .. d + 7 (d a multiple of 8) of position p; the word of V that holds dimension d of position p, and
// its bit; the element of the scale of position p's block b.
__device__ __forceinline__ int half_of(int p) { return (p >> 2) & 1; }
__device__ __forceinline__ int row_of(int p) { return ((p & 31) >> 3) * 4 + (p & 3); }
template <int DT> __device__ __forceinline__ size_t k_word(int nb, int p, int d) {
    const int b = d >> 5, c = (d & 31) >> 3;
    if constexpr (DT == L3M_Q4_0) return ((size_t)(p >> 5) * 128 + half_of(p) * 64 + c * 16 + row_of(p)) * nb + b;
    return ((((size_t)(p >> 5) * 2 + half_of(p)) * nb + b) * 16 + row_of(p)) * 4 + c;
}
template <int DT> __device__ __forceinline__ size_t v_word(int nb, int p, int d) {
    return ((size_t)(p >> 5) * 64 + ((p & 31) >> 3) * 16 + (d & 15)) * 2 * nb + (DT == L3M_Q4_0 ? d >> 4 : 2 * (d >> 5) + ((p >> 2) & 1));
}
template <int DT> __device__ __forceinline__ int v_bit(int p, int d) { return DT == L3M_Q4_0 ? 4 * ((p >> 1) & 3) + 16 * (p & 1) : 8 * (p & 3) + ((d >> 2) & 4); }
__device__ __forceinline__ size_t v_scale(int nb, int p, int b) { return ((size_t)(p >> 5) * nb + b) * TILE + (p & 31); }
template <int DT> __device__ __forceinline__ size_t k_scale(int nb, int p, int b) {
    if constexpr (DT == L3M_Q4_0) return v_scale(nb, p, b);
    return (((size_t)(p >> 5) * nb + b) * 16 + row_of(p)) * 2 + half_of(p);
}

template <int DT> __device__ __forceinline__ float scale_value(const uint8_t *s, size_t i) {
    if constexpr (DT == L3M_Q4_0) return (float)((const _Float16 *)s)[i];
    return __uint_as_float((uint32_t)s[i] << 23);                    // 0 (never written) is zero
}
// A code's value without its scale.
template <int DT> __device__ __forceinline__ float code_value(uint32_t c) {
    if constexpr (DT == L3M_Q4_0) return (float)((int)c - 8);
    const uint32_t m = c & 7;
    const float v = m < 2 ? 0.5f * (float)m : __uint_as_float(((m >> 1) + 126) << 23 | (m & 1) << 22);
    return c & 8 ? -v : v;
}

// ---------------------------------------------------------------- writer
template <int M> __device__ __forceinline__ uint32_t quad_xor(uint32_t x) {                 // lane ^ M's, M 1 or 2
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, M == 1 ? 0xB1 : 0x4E, 0xF, 0xF, true);
}
__device__ __forceinline__ void wave_sync() {                        // LDS values pass between a wavefront's lanes
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// x of another lane of the row of 16 (DPP), added.
template <int CTRL> __device__ __forceinline__ double dpp_add(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)u, CTRL, 0xF, 0xF, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, true);
    return x + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// The sum over each 1 << lg lanes, in all of them.
__device__ __forceinline__ double lanes_sum(double x, int lg) {
    if (lg > 0) x = dpp_add<0xB1>(x);                                // lane ^ 1
    if (lg > 1) x = dpp_add<0x4E>(x);                                // lane ^ 2
    if (lg > 2) x = dpp_add<0x141>(x);                               // the row's half mirrored: the other quad
    if (lg > 3) x = dpp_add<0x140>(x);                               // the row mirrored: the other half
    if (lg > 4) x += __shfl_xor(x, 16);
    return x;
}
// 1 / sqrt(x) by the hardware's estimate and two Newton steps, each of which squares the relative error: some 2^-52.
__device__ __forceinline__ double rsqrt64(double x) {
    double y = __builtin_amdgcn_rsq(x);
    if (!(x > 0 && x < 1e300)) return 1.0 / sqrt(x);
#pragma unroll
    for (int i = 0; i < 2; i++) y += 0.5 * y * (1.0 - x * y * y);
    return y;
}
// Codes in order, value i in bits 4 i .., as a word of K holds them.
template <int DT> __device__ __forceinline__ uint32_t in_order(uint32_t w) {
    if constexpr (DT != L3M_Q4_0) return w;
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) r |= (w >> 4 * i & 15u) << nib(DT, i);
    return r;
}
// Eight values of a block of 32 in each lane of a quad: their codes, value i in bits 4 i .., and the block's scale as it is stored (the
// same in the four). The file formats' rounding to the nearest (l3m_quantize_row), in the same float32 steps, so the stored bytes do not depend on
// where a row is quantized; a block holding a value that is not finite reads as NaN, a scale past f16 saturates, mxfp4 exponents end at
// 2^-126.
template <int DT> __device__ __forceinline__ uint32_t quantize(const float (&x)[8], uint32_t &stored) {
#pragma clang fp contract(off)
    float    top = x[0];
    uint32_t mag = __float_as_uint(x[0]) & 0x7FFFFFFFu;
#pragma unroll
    for (int i = 1; i < 8; i++) {
        const uint32_t m = __float_as_uint(x[i]) & 0x7FFFFFFFu;
        top = m > mag ? x[i] : top;                                  // the first of equal ones
        mag = max(mag, m);
    }
    uint32_t peak = max(mag, quad_xor<1>(mag));
    peak = max(peak, quad_xor<2>(peak));
    const bool bad = peak >= 0x7F800000u;
    uint32_t word = 0;
    if constexpr (DT == L3M_Q4_0) {
        const uint32_t first = (threadIdx.x & 60) + __builtin_ctz((uint32_t)(__ballot(mag == peak) >> (threadIdx.x & 60)) & 15u);
        const float d = __shfl(top, (int)first) * -0.125f, r = d != 0.f ? 1.0f / d : 0.f;
        stored = bad ? 0x7E00u : __builtin_bit_cast(uint16_t, (_Float16)fminf(fmaxf(d, -65504.f), 65504.f));
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float scaled = x[i] * r, v = floorf(scaled + 8.5f);
            word |= (uint32_t)(int)fminf(fmaxf(v, 0.f), 15.f) << 4 * i;
        }
    } else {
        const int   e = peak ? max((int)(peak >> 23) - 2, 1) : 0;    // a block of zeros: no value's exponent, so none is measured by it
        const float inv = __uint_as_float((uint32_t)(peak ? 254 - e : 127) << 23);
        stored = bad ? (uint32_t)E8M0_NAN : (uint32_t)e;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float    y = fabsf(x[i]) * inv;                    // exact
            const uint32_t c = (y > 0.25f) + (y > 0.75f) + (y > 1.25f) + (y > 1.75f) + (y > 2.5f) + (y > 3.5f) + (y > 5.f);
            word |= (c | (c && x[i] < 0.f ? 8u : 0u)) << 4 * i;
        }
        if (bad) word = 0;
    }
    return word;
}
template <int DT> __device__ __forceinline__ void put_scale(uint8_t *s, size_t i, uint32_t stored) {
    if constexpr (DT == L3M_Q4_0) ((uint16_t *)s)[i] = (uint16_t)stored;
    else s[i] = (uint8_t)stored;
}

struct RowsIn {
    const float *x, *wq, *wk, *table;
    float       *q, *k;
    long long    stride;
    int          n, nq, nkv, hd, halves, pos, lg;                    // 1 << lg lanes hold a head
    unsigned     qk_waves;
    float        eps;
};
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));   // floats need no alignment beyond their own

// A lane's four rotation pairs, pairs 4 i .. of a head row at x: first and second values. VEC: np a multiple of 4. Lanes past the head zeros.
template <bool VEC> __device__ __forceinline__ void load_pairs(const float *x, int i, int np, bool halves, float v0[4], float v1[4]) {
    if constexpr (VEC) {
        const bool in = 4 * i < np;
        const f32x4 a = *(const f32x4_a4 *)(x + (in ? (halves ? 4 * i : 8 * i) : 0)), b = *(const f32x4_a4 *)(x + (in ? (halves ? np + 4 * i : 8 * i + 4) : 0));
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v0[j] = !in ? 0.f : halves ? a[j] : j < 2 ? a[2 * j] : b[2 * j - 4];
            v1[j] = !in ? 0.f : halves ? b[j] : j < 2 ? a[2 * j + 1] : b[2 * j - 3];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int p = 4 * i + j;
            v0[j] = p < np ? x[halves ? p : 2 * p] : 0.f;
            v1[j] = p < np ? x[halves ? np + p : 2 * p + 1] : 0.f;
        }
    }
}
template <bool VEC> __device__ __forceinline__ void store_pairs(float *x, int i, int np, bool halves, const float v0[4], const float v1[4]) {
    if constexpr (VEC) {
        if (4 * i >= np) return;
        *(f32x4_a4 *)(x + (halves ? 4 * i : 8 * i)) = halves ? f32x4{v0[0], v0[1], v0[2], v0[3]} : f32x4{v0[0], v1[0], v0[1], v1[1]};
        *(f32x4_a4 *)(x + (halves ? np + 4 * i : 8 * i + 4)) = halves ? f32x4{v1[0], v1[1], v1[2], v1[3]} : f32x4{v0[2], v1[2], v0[3], v1[3]};
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int p = 4 * i + j;
            if (p < np) {
                x[halves ? p : 2 * p] = v0[j];
                x[halves ? np + p : 2 * p + 1] = v1[j];
            }
        }
    }
}

// Norm and rotation of query and key heads, eight values a lane and 64 >> lg heads a wavefront: x s w with s = 1 / sqrt(mean x^2 + eps), then
// the pairs turned by the table's angles. In 64 bits up to the one rounding of each result, because a key's 4-bit code hangs on which
// side of a border it lies: the row is the float32 nearest to the formula's, whatever the order of the sum. Then, DT < 0, keys
// go to a.k; else they are quantized, eight consecutive dimensions a lane (through LDS where the lane's own are two fours a half head
// apart). Wavefronts behind a.qk_waves take eight positions of 64 dimensions of V each: a lane quantizes eight dimensions of one
// position, and the words, which run along positions, are put together through LDS.
//
// Bound by the bytes for many tokens: the rotation of 2048 tokens, 40 heads of 128, takes 19.0 us, 4.4 TB/s of the 5.5 that a copy reaches (33.5
// with one value a lane and a head a wavefront); an append of 1000 tokens, 32 and 8 heads of 128, 12.7 us, 3.3 TB/s; one token 2.4 and
// 3.0 us, a launch and one chain of loads. Stores past the caches take 16.9 instead of 19.0 us, but the attention that reads the queries next
// loses more; fewer workgroups in a loop change nothing.
template <int DT, bool VEC> __global__ void __launch_bounds__(256) k_rows_in(RowsIn a, l3m_kv4 c) {
    __shared__ __align__(16) float row_s[4][512];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, heads = a.nq + a.nkv, nb = (a.hd + 31) >> 5, np = a.hd >> 1;
    const unsigned w = blockIdx.x * 4 + wave;
    if (w < a.qk_waves) {
        const int sub = lane >> a.lg, i = lane & ((1 << a.lg) - 1);
        const unsigned item = w * (64u >> a.lg) + sub, items = (unsigned)a.n * heads, at = min(item, items - 1), t = at / (unsigned)heads;
        const int h = (int)(at - t * heads);
        const bool key = h >= a.nq, halves = a.halves;
        const float *x = a.x + (long long)t * a.stride + (size_t)h * a.hd, *wt = key ? a.wk : a.wq;
        float v0[4], v1[4], g0[4], g1[4], cs0[4], cs1[4];
        load_pairs<VEC>(x, i, np, halves, v0, v1);
        const bool any_norm = a.wq || a.wk;
        if (any_norm) load_pairs<VEC>(wt ? wt : x, i, np, halves, g0, g1);
        if (a.table) load_pairs<VEC>(a.table + (size_t)(a.pos + (int)t) * a.hd, i, np, false, cs0, cs1);
        double s = 1;
        if (any_norm) {
            double ss = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) ss += (double)v0[j] * v0[j] + (double)v1[j] * v1[j];
            s = rsqrt64(lanes_sum(ss, a.lg) / a.hd + (double)a.eps);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            double y0 = v0[j], y1 = v1[j];
            if (any_norm && wt) {
                y0 *= s * (double)g0[j];
                y1 *= s * (double)g1[j];
            }
            if (a.table) {
                const double co = cs0[j], si = cs1[j], z = y0 * co - y1 * si;
                y1 = y0 * si + y1 * co;
                y0 = z;
            }
            v0[j] = (float)y0;
            v1[j] = (float)y1;
        }
        if (item < items && (DT < 0 || !key))
            store_pairs<VEC>(key ? a.k + ((size_t)t * a.nkv + h - a.nq) * a.hd : a.q + ((size_t)t * a.nq + h) * a.hd, i, np, halves, v0, v1);
        if constexpr (DT >= 0) {
            if (!__ballot(key)) return;                              // queries alone
            float k[8];
            if (halves) {
                float *row = row_s[wave] + (sub << a.lg) * 8;
                store_pairs<VEC>(row, i, np, true, v0, v1);
                wave_sync();
#pragma unroll
                for (int j = 0; j < 8; j++) k[j] = 8 * i < a.hd ? row[8 * i + j] : 0.f;
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    k[2 * j] = v0[j];
                    k[2 * j + 1] = v1[j];
                }
            }
            uint32_t stored;
            const uint32_t codes = quantize<DT>(k, stored);
            if (key && item < items && 8 * i < 32 * nb) {
                const Head H = head_of(c, nb, sbytes(DT), h - a.nq);
                const int p = a.pos + (int)t;
                H.kq[k_word<DT>(nb, p, 8 * i)] = in_order<DT>(codes);
                if ((i & 3) == 0) put_scale<DT>(H.ks, k_scale<DT>(nb, p, i >> 2), stored);
            }
        }
        return;
    }
    if constexpr (DT >= 0) {
        const unsigned vw = w - a.qk_waves, chunks = (unsigned)(nb + 1) >> 1, per = chunks * a.nkv;
        const unsigned o0 = (unsigned)a.pos >> 3, octets = ((unsigned)(a.pos + a.n - 1) >> 3) - o0 + 1, oi = vw / per;
        if (oi >= octets) return;
        const int h = (int)((vw - oi * per) / chunks), chunk = (int)((vw - oi * per) % chunks), p0 = (int)(o0 + oi) * 8;
        const int first = max(p0, a.pos), end = min(p0 + 8, a.pos + a.n);
        const Head H = head_of(c, nb, sbytes(DT), h);
        const int p = p0 + (lane >> 3), d = 64 * chunk + 8 * (lane & 7);
        const bool in = p >= first && p < end && d < a.hd;
        const float *v = a.x + (size_t)(heads + h) * a.hd + (in ? (p - a.pos) * a.stride + d : 0);
        const f32x4 v0 = *(const f32x4_a4 *)v, v1 = *(const f32x4_a4 *)(v + 4);
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = in ? j < 4 ? v0[j & 3] : v1[j & 3] : 0.f;
        uint32_t stored, *word_s = (uint32_t *)row_s[wave];
        word_s[lane] = quantize<DT>(x, stored);                      // [position][eight dimensions]
        if ((lane & 3) == 0 && p >= first && p < end && d < 32 * nb) put_scale<DT>(H.vs, v_scale(nb, p, d >> 5), stored);
        wave_sync();
        // lane's word: q4_0 dimension 64 chunk + lane of the eight positions; mxfp4 dimensions 64 chunk + 32 (lane / 32) + lane % 16 and 16 more
        // of four
        const int u = DT == L3M_Q4_0 ? 0 : lane >> 4 & 1, e = DT == L3M_Q4_0 ? lane : (lane & 32) + (lane & 15);
        uint32_t word = 0, mine = 0;
#pragma unroll
        for (int j = 0; j < (DT == L3M_Q4_0 ? 8 : 4); j++) {
            const int q = 4 * u + j;
            const bool has = p0 + q >= first && p0 + q < end;
            word |= (word_s[8 * q + (e >> 3)] >> 4 * (e & 7) & 15u) << v_bit<DT>(q, 0);
            if constexpr (DT != L3M_Q4_0) word |= (word_s[8 * q + (e >> 3) + 2] >> 4 * (e & 7) & 15u) << v_bit<DT>(q, 16);
            if (has) mine |= (DT == L3M_Q4_0 ? 15u : 255u) << v_bit<DT>(q, 0);
        }
        if (64 * chunk + e < 32 * nb && mine) {
            uint32_t *to = H.vq + v_word<DT>(nb, p0 + 4 * u, 64 * chunk + e);
            *to = mine == ~0u ? word : (*to & ~mine) | (word & mine);   // the word's other positions stay
        }
    }
}

// ---------------------------------------------------------------- read-back
// A thread a word of K (eight dimensions of a position), then one a dimension of V (its eight positions): stores are contiguous either way.
// Bound by the bytes it writes: 1000 positions of 8 heads of 128 (8.2 MB) q4_0 5.0 us, mxfp4 5.7, one 2.0.
template <int DT> __global__ void __launch_bounds__(256) k_kv4_rows(l3m_kv4 c, float *k, float *v, int pos, int n, unsigned k_threads) {
    const int nb = (c.hd + 31) >> 5;
    const unsigned id = blockIdx.x * 256 + threadIdx.x, nkv = c.nkv, hd = c.hd;
    if (id < k_threads) {
        const unsigned per = hd >> 3, row = id / per, d = 8 * (id - row * per), t = row / nkv, h = row - t * nkv;
        if (t >= (unsigned)n) return;
        const Head H = head_of(c, nb, sbytes(DT), (int)h);
        const int p = pos + (int)t;
        const uint32_t w = H.kq[k_word<DT>(nb, p, (int)d)];
        const float s = scale_value<DT>(H.ks, k_scale<DT>(nb, p, (int)d >> 5));
        f32x4 x[2];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i >> 2][i & 3] = code_value<DT>(w >> nib(DT, i) & 15) * s;
        float *to = k + (size_t)row * hd + d;
        *(f32x4_a4 *)to = x[0];
        *(f32x4_a4 *)(to + 4) = x[1];
        return;
    }
    const unsigned vi = id - k_threads, oh = vi / hd, d = vi - oh * hd, o = oh / nkv, h = oh - o * nkv, p0 = 8 * (((unsigned)pos >> 3) + o);
    if (!v || p0 >= (unsigned)(pos + n)) return;
    const Head H = head_of(c, nb, sbytes(DT), (int)h);
    const uint32_t w[2] = {H.vq[v_word<DT>(nb, (int)p0, (int)d)], H.vq[v_word<DT>(nb, (int)p0 + 4, (int)d)]};   // q4_0: the same
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int p = (int)p0 + i;
        if (p < pos || p >= pos + n) continue;
        v[((size_t)(p - pos) * nkv + h) * hd + d] = code_value<DT>(w[i >> 2] >> v_bit<DT>(i, (int)d) & 15) * scale_value<DT>(H.vs, v_scale(nb, p, (int)d >> 5));
    }
}

// ---------------------------------------------------------------- attention
// Rows: the n g (token, query head) pairs of a kv head, a token's heads side by side (g = nq / nkv); 16 are a product's columns. Per tile of
// 32 positions and wavefront, with the keys as the left operand so that lane 16 g4 + r holds the scores of row r for positions
// 8 g4 .. 8 g4 + 7, which is where the second product wants the weights:
//   S = K Q^T   16 positions x 16 rows, twice; q scaled by log2(e) / sqrt(hd) and held in parts (below)
//   P = 2^(S - m), m such that the largest weight lies between 2^7 and 2^15 (q4_0: times the largest scale): it moves only when one passes
//               that, and -m is what mxfp4's accumulators begin at (q4_0's scores get it with their unit, in one operation)
//   O^T += V^T P^T   16 dimensions x 16 rows x 32 positions (v_mfma_f32_16x16x32_f16), P in two f16 parts: 22 bits, and 2^-32 of the largest at the
//               least. A position's scale differs from block to block. q4_0's multiplies P, in 32 bits, before it is split (the range of
//               the weights then goes by the scales). mxfp4's goes into the conversion of its codes (a layout of its own), exactly where
//               it lies between 2^-23 and 2^13; other tiles' values and the accumulators take another unit. A row's range, and NaN, come
//               from positions that it sees, never from one behind it.
// All sums in 32 bits. A workgroup's four wavefronts share 16 CT rows and split the tiles; they meet in LDS, and the workgroups of a
// long cache (splits > 1) in the workspace, added in order by k_kv4_join.
//
// A few tokens are bound by latency (one token over 40 positions 3.6 us, 256: 4.2, 480 tokens of 9 heads over 3 of 64 6.1 us: one
// workgroup's tiles one after the other), long caches by the cache's bytes and the conversions together: one token over 131071 positions, 32
// heads over 8 of 128, q4_0 (151 MB) 37 us, 4.1 TB/s with the SIMDs issuing three quarters of the time; mxfp4 over 32768 (36 MB) 10.5 us; with
// the join, and caches past the Infinity Cache in turn, 44.1 and 14.8.
// Prompts by instruction issue: 1024 tokens behind 2999, the same heads, mxfp4, 98 us, 600 TFLOP/s: VALU and matrix instructions, some 256 and 52
// a tile of 32 rows, are issued for 157k of 212k cycles, the matrix unit is busy for 92k. q4_0, with every scale on the weights,
// 177 us. Tried without gain: eight wavefronts a workgroup, a tile requested ahead, values a tile ahead, raised wave priority around the
// products; a tile's scores beside the products of the one before has no registers.
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x6 __attribute__((ext_vector_type(6)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x32 __attribute__((ext_vector_type(32)));

constexpr int WAVES = 4;
constexpr int SPLIT_WGS = 512, SPLITS = 256;                         // workgroups up to which a cache is split; most parts of it
constexpr int NONE = -1000;                                          // a unit before the first: below every one by more than 60
constexpr float M0 = -3.40282347e38f;                                // the maximum of no score: float32's lowest, below every one

// A q4_0 K word's eight codes, 0 .. 15, in f16: a nibble alone in a byte is the e4m3 number 2^-9 times it.
__device__ __forceinline__ f16x8 widen(uint32_t w) {
    const int lo = (int)(w & 0x0F0F0F0Fu), hi = (int)(w >> 4 & 0x0F0F0F0Fu);
    const f16x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.f, false), p1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.f, true);
    const f16x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.f, false), p3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.f, true);
    return f16x8{p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
}
// Byte i of w as the power of two that it is the exponent of: one instruction, a product with 2^23 that takes the byte where it lies; as a shift,
// or a product that the compiler sees to be one, it is a shift and a mask.
__device__ __forceinline__ float pow2_byte(uint32_t w, int i) {
    uint32_t unit = 1u << 23;
    asm("" : "+s"(unit));
    return __uint_as_float(__umul24(w >> 8 * i & 255u, unit));
}
__device__ __forceinline__ float max8(const float (&s)[8]) {
    return fmaxf(fmaxf(fmaxf(fmaxf(fmaxf(fmaxf(fmaxf(s[0], s[1]), s[2]), s[3]), s[4]), s[5]), s[6]), s[7]);
}
__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// Eight float32 values as the sum of two f16 ones each: 22 bits, 2^-25 at the least; below 65520. The rests by the instruction that takes a
// half as it lies in its pair (v_fma_mix_f32; a difference is a conversion first, so the compiler does not see the factor).
__device__ __forceinline__ void two_parts(const float (&w)[8], f16x8 &hi, f16x8 &lo) {
    float minus1 = -1.f;
    asm("" : "+s"(minus1));
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const f16x2 h = __builtin_convertvector((f32x2{w[i], w[i + 1]}), f16x2);
        const float r0 = fmaf((float)h.x, minus1, w[i]), r1 = fmaf((float)h.y, minus1, w[i + 1]);
        const f16x2 l = __builtin_convertvector((f32x2{r0, r1}), f16x2);
        hi[i] = h.x; hi[i + 1] = h.y;
        lo[i] = l.x; lo[i + 1] = l.y;
    }
}
// A q4_0 V word's values -8 .. 7 in f16: 1024 + code is the half 0x6400 | code, 1032 less is exact.
__device__ __forceinline__ f16x8 widen_f16(uint32_t w) {
    uint32_t r[4], codes = 0x000F000Fu;
    asm("" : "+v"(codes));                                           // in a vector register: the and and the or are one instruction
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const _Float16 c = (_Float16)-1032.f;
        r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, (w >> 4 * i & codes) | 0x64006400u) + f16x2{c, c});
    }
    return __builtin_bit_cast(f16x8, u32x4{r[0], r[1], r[2], r[3]});
}
// mxfp4 V words of a block, eight positions of dimensions j and 16 + j, a position's scale each, as the two operands.
__device__ __forceinline__ void widen_v(const uint32_t w[2], const float d[8], f16x8 &v0, f16x8 &v1) {
    uint32_t r[8], a[4], b[4];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        r[4 * u] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[u], d[4 * u], 0));
        r[4 * u + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[u], d[4 * u + 1], 1));
        r[4 * u + 2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[u], d[4 * u + 2], 2));
        r[4 * u + 3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[u], d[4 * u + 3], 3));
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        a[i] = __builtin_amdgcn_perm(r[2 * i + 1], r[2 * i], 0x05040100u);
        b[i] = __builtin_amdgcn_perm(r[2 * i + 1], r[2 * i], 0x07060302u);
    }
    v0 = __builtin_bit_cast(f16x8, u32x4{a[0], a[1], a[2], a[3]});
    v1 = __builtin_bit_cast(f16x8, u32x4{b[0], b[1], b[2], b[3]});
}
// Whether the four exponents of w lie in 104 .. 140, where e2m1 codes with them are f16 numbers (k 2^-24 .. 6 2^13).
__device__ __forceinline__ bool f16_range(uint32_t w) {
    const uint32_t a = w & 0x7F7F7F7Fu, from104 = a + 0x18181818u, from141 = a + 0x73737373u;   // bit 7: of 104 .. 127, of 141 ..
    return ((from104 ^ w) & ~(from141 & w) & 0x80808080u) == 0x80808080u;
}

// The maximum and the sum of a row of 16 lanes' (DPP), over lane ^ 16 and lane ^ 32.
__device__ __forceinline__ float other16(float x, float &y) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    y = __uint_as_float(r[1]);
    return __uint_as_float(r[0]);
}
__device__ __forceinline__ float other32(float x, float &y) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    y = __uint_as_float(r[1]);
    return __uint_as_float(r[0]);
}
__device__ __forceinline__ float max_g4(float x) {
    float y;
    x = other16(x, y); x = fmaxf(x, y);
    x = other32(x, y); return fmaxf(x, y);
}
__device__ __forceinline__ float sum_g4(float x) {
    float y;
    x = other16(x, y); x += y;
    x = other32(x, y); return x + y;
}

// The scores of one half of a tile, 16 positions x 16 rows, from the queries of a row held in parts (Queries) and what a lane reads of the
// keys (KeysIn).
//
// q4_0: 16x16x32 f16 products of a block's codes 0 .. 15 with q in two f16 parts, begun at -8 sum q; a block's sum times d, which belongs to
// a position, in 32 bits. A row of q is scaled by a power of two to a largest value of 2^13 .. 2^14: 22 bits of each value, and 2^-38 of
// the largest at the least.
//
// mxfp4: 16x16x128 products of the codes as they lie with their scales (v_mfma_scale_f32_16x16x128_f8f6f4, fp4 operand): lane 16 c + m gives
// block c of position m, and q is the fp6 (e2m3) operand, a block in five parts with scales of their own. A part takes five bits of
// the block's largest magnitude: with a in [2, 4) units, rounded to 1/4 at most, 1/8 unit is left, which is 4 of the next part's, 32
// times smaller. Five leave 2^-24 of the largest magnitude. Where a head has one or two blocks, the lane groups past them take
// other parts of the same blocks.
template <int DT, int NB> struct KeysIn;
template <int DT, int NB> struct Queries;

template <int NB> struct KeysIn<L3M_Q4_0, NB> {
    uint32_t q[2][NB];
    f16x8    d[NB];                                                  // of positions 8 g4 .. + 7
    __device__ __forceinline__ void load(const Head &H, int tile, int lane) {
        const size_t T = (size_t)tile;
        __builtin_memcpy(q[0], __builtin_assume_aligned(H.kq + (T * 128 + lane) * NB, 4), 4 * NB);
        __builtin_memcpy(q[1], __builtin_assume_aligned(H.kq + (T * 128 + 64 + lane) * NB, 4), 4 * NB);
#pragma unroll
        for (int b = 0; b < NB; b++) d[b] = *(const f16x8 *)(H.ks + 2 * ((T * NB + b) * TILE + 8 * (lane >> 4)));
    }
};
template <int NB> struct Queries<L3M_Q4_0, NB> {
    f16x8 part[NB][2];
    f32x4 off[NB];                                                   // -8 sum of a block's q
    float unit;                                                      // of the scores
    __device__ __forceinline__ void load(const float *q, int hd, float scale, int lane) {
        float x[NB][8];
        uint32_t peak = 0;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const int d = 32 * b + 8 * (lane >> 4);
            const bool in = d < hd;
            const f32x4 x0 = *(const f32x4_a4 *)(q + (in ? d : 0)), x1 = *(const f32x4_a4 *)(q + (in ? d + 4 : 4));
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[b][i] = in ? (i < 4 ? x0[i & 3] : x1[i & 3]) * scale : 0.f;
                peak = max(peak, __float_as_uint(x[b][i]) & 0x7FFFFFFFu);
            }
        }
        peak = __float_as_uint(max_g4(__uint_as_float(min(peak, 0x7F7FFFFFu))));
        const int e = 140 - (int)(peak >> 23);
        unit = ldexpf(1.f, -e);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float y = ldexpf(x[b][i], e);
                const _Float16 hi = (_Float16)y, lo = (_Float16)(y - (float)hi);
                part[b][0][i] = hi;
                part[b][1][i] = lo;
                sum += y;
            }
            sum = -8.f * sum_g4(sum);
            off[b] = f32x4{sum, sum, sum, sum};
        }
    }
};
template <int NB, int CT> __device__ __forceinline__ void scores(const KeysIn<L3M_Q4_0, NB> &k, const Queries<L3M_Q4_0, NB> (&q)[CT], int f, f32x4 (&c)[CT]) {
#pragma unroll
    for (int b = 0; b < NB; b++) {
        const f16x8 w = widen(k.q[f][b]);
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            const f32x4 x = mfma(w, q[ct].part[b][1], mfma(w, q[ct].part[b][0], q[ct].off[b]));
#pragma unroll
            for (int r = 0; r < 4; r++) c[ct][r] = fmaf(x[r], (float)k.d[b][4 * f + r], c[ct][r]);
        }
    }
}

constexpr int Q_PARTS = 5;
// Blocks by fours (a product's lane groups); parts that one product takes; products a four.
template <int NB> struct Mx {
    static constexpr int fours = (NB + 3) / 4, at_once = NB == 1 ? 4 : NB == 2 ? 2 : 1, times = (Q_PARTS + at_once - 1) / at_once;
    static __device__ __forceinline__ int block(int four, int group) { return NB <= 2 ? group % NB : min(4 * four + group, NB - 1); }
};
template <int NB> struct KeysIn<L3M_MXFP4, NB> {
    u32x4    q[2][Mx<NB>::fours];
    uint32_t e[Mx<NB>::fours];                                       // the two halves' exponents
    uint32_t four;                                                   // of the tile's 32 NB values' exponents, which are looked over first: 4 lane ..
    __device__ __forceinline__ void load(const Head &H, int tile, int lane) {
        const size_t T = (size_t)tile;
        four = ((const uint32_t *)(H.vs + T * NB * TILE))[min(lane, 8 * NB - 1)];
#pragma unroll
        for (int i = 0; i < Mx<NB>::fours; i++) {
            const int b = Mx<NB>::block(i, lane >> 4), m = lane & 15;
            q[0][i] = ((const u32x4 *)H.kq)[(T * 2 * NB + b) * 16 + m];
            q[1][i] = ((const u32x4 *)H.kq)[((T * 2 + 1) * NB + b) * 16 + m];
            e[i] = ((const uint16_t *)H.ks)[(T * NB + b) * 16 + m];
        }
    }
};
template <int NB> struct Queries<L3M_MXFP4, NB> {
    u32x6 part[Mx<NB>::fours][Mx<NB>::times];
    int   e[Mx<NB>::fours][(Mx<NB>::times + 3) / 4];                 // the parts' exponents, a byte each
    __device__ __forceinline__ void load(const float *q, int hd, float scale, int lane) {
        const int c = lane >> 4;
#pragma unroll
        for (int i = 0; i < Mx<NB>::fours; i++) {
            const int b = Mx<NB>::block(i, c), first = NB == 1 ? c : NB == 2 ? c >> 1 : 0;       // this lane's part of the first product
            const bool used = NB <= 2 || 4 * i + c < NB;
            float x[32];
            uint32_t peak = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int d = 32 * b + 4 * j;
                const bool in = d < hd;
                const f32x4 v = *(const f32x4_a4 *)(q + (in ? d : 0));
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    x[4 * j + r] = in ? v[r] * scale : 0.f;
                    peak = max(peak, __float_as_uint(x[4 * j + r]) & 0x7FFFFFFFu);
                }
            }
            const bool bad = peak >= 0x7F800000u;                    // a scale of NaN for a row that is not finite
            // The conversions of 32 values take several cycles and may not write over what they read (with results on their sources, now and then
            // wrong last parts). The compiler does not know it of its builtins, so they are written out with results that it keeps apart (=&);
            // the wait behind each is for a product that reads its result next. No product is under way here that they could meet.
#pragma unroll
            for (int t = 0; t < Mx<NB>::times; t++) {
                part[i][t] = u32x6{0, 0, 0, 0, 0, 0};
                e[i][t / 4] = 0x7F7F7F7F;
            }
#pragma unroll
            for (int p = 0; p < Q_PARTS; p++) {
                const int ex = max((int)(peak >> 23) - 1 - 5 * p, 1);
                const float unit = __uint_as_float((uint32_t)ex << 23);
                f32x16 even, odd;
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    even[j] = x[2 * j];
                    odd[j] = x[2 * j + 1];
                }
                u32x6 w;
                f32x32 back;
                asm("v_cvt_scalef32_2xpk16_fp6_f32 %0, %1, %2, %3\n\ts_nop 1" : "=&v"(w) : "v"(even), "v"(odd), "v"(unit));
                asm("v_cvt_scalef32_pk32_f32_fp6 %0, %1, %2\n\ts_nop 1" : "=&v"(back) : "v"(w), "v"(unit));
#pragma unroll
                for (int j = 0; j < 32; j++) x[j] -= back[j];
                const int t = p / Mx<NB>::at_once, at = p - t * Mx<NB>::at_once;
                if (used && (Mx<NB>::at_once == 1 || first == at)) {
                    part[i][t] = w;
                    e[i][t / 4] ^= ((bad ? E8M0_NAN : ex) ^ 127) << 8 * (t % 4);
                }
            }
        }
    }
};
template <int NB, int CT> __device__ __forceinline__ void scores(const KeysIn<L3M_MXFP4, NB> &k, const Queries<L3M_MXFP4, NB> (&q)[CT], int f, f32x4 (&c)[CT]) {
#pragma unroll
    for (int i = 0; i < Mx<NB>::fours; i++) {
        const i32x8 a = {(int)k.q[f][i].x, (int)k.q[f][i].y, (int)k.q[f][i].z, (int)k.q[f][i].w, 0, 0, 0, 0};
        auto part = [&](auto which, auto half) {
            constexpr int t = decltype(which)::value, F = decltype(half)::value;
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                const u32x6 &w = q[ct].part[i][t];
                const i32x8 b = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], (int)w[4], (int)w[5], 0, 0};
                c[ct] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c[ct], 4, 2, F, (int)k.e[i], t % 4, q[ct].e[i][t / 4]);
            }
        };
        auto parts = [&](auto half) {
            part(std::integral_constant<int, 0>{}, half);
            if constexpr (Mx<NB>::times > 1) part(std::integral_constant<int, 1>{}, half);
            if constexpr (Mx<NB>::times > 2) part(std::integral_constant<int, 2>{}, half);
            if constexpr (Mx<NB>::times > 3) part(std::integral_constant<int, 3>{}, half);
            if constexpr (Mx<NB>::times > 4) part(std::integral_constant<int, 4>{}, half);
        };
        if (f == 0) parts(std::integral_constant<int, 0>{});
        else parts(std::integral_constant<int, 1>{});
    }
}

// Of its values: its dimensions' words, and the scales of its positions.
template <int DT, int NB> struct ValuesIn {
    uint32_t q[2 * NB], e[NB][2];
    f16x8    d[DT == L3M_Q4_0 ? NB : 1];
    __device__ __forceinline__ void load(const Head &H, int tile, int lane) {
        const size_t T = (size_t)tile;
        __builtin_memcpy(q, __builtin_assume_aligned(H.vq + (T * 64 + lane) * 2 * NB, 4), 8 * NB);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            if constexpr (DT == L3M_Q4_0) d[b] = *(const f16x8 *)(H.vs + 2 * ((T * NB + b) * TILE + 8 * (lane >> 4)));
            else __builtin_memcpy(e[b], __builtin_assume_aligned(H.vs + (T * NB + b) * TILE + 8 * (lane >> 4), 8), 8);
        }
    }
};

struct AttendIn {
    float       *out, *ml, *parts;                                   // ml, parts: [row of out][split] maximum and sum, output
    const float *q;
    l3m_kv4      c;
    int          n, nq, g, pos, groups, group0, splits;
    uint32_t     g_mul, quad_mul, of_mul;                            // of g, hd / 4 and splits WAVES (divide)
};
// x / d by d's multiplier, exact while x d < 2^32; 0: d is 1, or too large for it.
__host__ inline uint32_t multiplier(uint32_t d, uint32_t most) {
    return d > 1 && (uint64_t)most * d < 1ull << 32 ? (uint32_t)((1ull << 32) / d) + 1 : 0;
}
__device__ __forceinline__ uint32_t divide(uint32_t x, uint32_t d, uint32_t mul) { return mul ? __umulhi(x, mul) : d == 1 ? x : x / d; }
template <int CTRL> __device__ __forceinline__ float dpp(float x) { return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xF, 0xF, true)); }
__device__ __forceinline__ float max_wave(float x) {
    x = fmaxf(x, dpp<0xB1>(x)); x = fmaxf(x, dpp<0x4E>(x)); x = fmaxf(x, dpp<0x141>(x)); x = fmaxf(x, dpp<0x140>(x));
    return max_g4(x);
}
__device__ __forceinline__ float sum_wave(float x) {
    x += dpp<0xB1>(x); x += dpp<0x4E>(x); x += dpp<0x141>(x); x += dpp<0x140>(x);
    return sum_g4(x);
}

template <int DT, int NB, int CT> __global__ void __launch_bounds__(64 * WAVES) k_kv4_attend(AttendIn a) {
    constexpr int ROWS = 16 * CT, OS = 32 * NB + 4;                  // OS: a row's stride in LDS
    constexpr int O_WAVES = WAVES * ROWS * OS * 4 <= 60000 ? WAVES : WAVES / 2;   // wavefronts whose outputs LDS holds at once
    __shared__ float o_s[O_WAVES][ROWS][OS], m_s[WAVES][ROWS], l_s[WAVES][ROWS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, g4 = lane >> 4, hd = a.c.hd, g = a.g;
    // kv heads fastest: consecutive workgroups go to different XCDs, so 8 heads keep to an L2 each. The longest rows first.
    const int h = (int)blockIdx.x, split = (int)blockIdx.y, group = a.groups - 1 - a.group0 - (int)blockIdx.z;
    const int R = a.n * g, row0 = group * ROWS, rows = min(R - row0, ROWS);
    const int first = (int)divide(row0, g, a.g_mul), last = (int)divide(row0 + rows - 1, g, a.g_mul);   // the rows' tokens
    const unsigned tiles = (unsigned)(a.pos + last + TILE) / TILE, whole = (unsigned)(a.pos + first + 1) / TILE;   // tiles seen; those with nothing masked
    const unsigned part = (unsigned)(split * WAVES + wave), of = (unsigned)a.splits * WAVES, share = divide(tiles, of, a.of_mul), more = tiles - share * of;
    const int t0 = (int)(part * share + min(part, more)), t1 = t0 + (int)(share + (part < more));
    const Head H = head_of(a.c, NB, sbytes(DT), h);
    KeysIn<DT, NB> keys;
    ValuesIn<DT, NB> vals;
    keys.load(H, min(t0, (int)tiles - 1), lane);
    vals.load(H, min(t0, (int)tiles - 1), lane);

    Queries<DT, NB> qs[CT];
    int seen[CT];                                                    // positions a row sees
    const float scale = 1.44269504f / sqrtf((float)hd);
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        const unsigned r = (unsigned)min(row0 + 16 * ct + r16, R - 1), t = divide(r, g, a.g_mul);   // columns past the last row repeat it
        seen[ct] = a.pos + (int)t + 1;
        qs[ct].load(a.q + ((size_t)t * a.nq + h * g + (r - t * (unsigned)g)) * hd, hd, scale, lane);
    }

    f32x4 acc[CT][2 * NB];
    float m[CT], lim[CT], l[CT];                                     // what scores are less by; the weight that moves it; sum of weights
    float base[CT];                                                  // log2 of the weight a new maximum gets; q4_0: of its product with the largest scale 7
    constexpr float RISE = DT == L3M_Q4_0 ? 7.98f : 8.f;             // how far weights pass 2^base before it moves (q4_0: 2^16 less f16's room for products)
    int   unit = 0, high = NONE;                                     // mxfp4: acc counts 2^unit; the largest unit that fit_unit chose or found
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        base[ct] = 7.f;
        m[ct] = 0.f;
        lim[ct] = -1.f;                                              // a row's first score always does
        l[ct] = 0.f;
#pragma unroll
        for (int t = 0; t < 2 * NB; t++) acc[ct][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if constexpr (DT == L3M_Q4_0)                                    // the first tile's, of those that the row sees, of every eighth position: larger ones lower base
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            uint32_t most = 1;                                       // 2^-24, the smallest scale there is
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const _Float16 d = vals.d[b][0];
                const uint32_t u = __builtin_bit_cast(uint16_t, d) & 0x7FFFu;
                most = max(most, u < 0x7C00u && t0 * TILE + 8 * g4 < seen[ct] ? u : 0u);
            }
            const float d = max_g4((float)__builtin_bit_cast(_Float16, (uint16_t)most));
            base[ct] -= (float)((int)(__float_as_uint(d) >> 23) - 127);
        }
    auto scale_acc = [&](int ct, float f) {
#pragma unroll
        for (int t = 0; t < 2 * NB; t++) acc[ct][t] *= f;
    };
    // mxfp4, a tile whose exponents are not all f16's (or one behind it): its values in a unit of their own, the largest 2^10 to 2^13 and values of
    // 2^-33 of it exact, and its exponents in that unit. What the accumulators are to be multiplied by, exactly: they hold less than 2^61 times
    // the largest unit so far, and the unit never lies 60 below that (values that much smaller have no part in the sums). Tiles that were
    // not brought here counted as unit 0; where the first has no value, the next is brought here too.
    auto fit_unit = [&](int tile, uint32_t four) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t e = four >> 8 * i & 255u;
            top = e == E8M0_NAN ? top : max(top, e);
        }
        const int most = __builtin_amdgcn_readfirstlane((int)max_wave((float)top)), was = unit;
        if (tile != t0 && unit == 0 && high == NONE) high = 0;
        const bool first = high == NONE;
        if (most) {
            unit = max(most - 137, high - 60);
            high = max(high, unit);
        } else if (first) unit = -1;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                uint32_t to = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int e = (int)(vals.e[b][j] >> 8 * i & 255u);
                    to |= (uint32_t)(e == E8M0_NAN ? e : min(max(e - unit, 0), 254)) << 8 * i;
                }
                vals.e[b][j] = to;
            }
        return first ? 1.f : ldexpf(1.f, was - unit);
    };

    // mxfp4: the bytes of a lane's four exponents whose positions lie at `end` or behind; whether all others of the tile are f16's; whether they are f16's
    // or zeros', and not zeros' alone.
    auto behind = [&](int tile, int end) {
        const int left = end - (tile * TILE + 4 * (min(lane, 8 * NB - 1) & 7));
        return left >= 4 ? 0u : left <= 0 ? ~0u : ~0u << 8 * left;
    };
    auto narrow = [&](uint32_t four, uint32_t none) { return !__ballot(!f16_range((four & ~none) | (0x7F7F7F7Fu & none))); };
    auto narrow_or_zero = [&](uint32_t four, uint32_t none) {
        const uint32_t w = four & ~none, some = (((w & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) | w) & 0x80808080u;   // bytes that are not 0
        return narrow(w | ((some ^ 0x80808080u) >> 7) * 0x7Fu, none) && __ballot(w != 0) != 0;
    };
    // A tile (masked: the positions before `end`; each: for the rows that see just those, alone). Then the words of tile `next`.
    auto step = [&](const int tile, const int next, const int end, const bool each, auto masked) {
        constexpr bool MASK = decltype(masked)::value;
        const int p0 = tile * TILE + 8 * g4;
        int upto[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ct++) upto[ct] = each && seen[ct] != end ? 0 : seen[ct];
        float p[CT][8];
#pragma unroll
        for (int f = 0; f < 2; f++) {
            f32x4 c[CT];
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                const float from = DT == L3M_Q4_0 ? 0.f : -m[ct];
                c[ct] = f32x4{from, from, from, from};
            }
            scores<NB, CT>(keys, qs, f, c);
            if constexpr (DT == L3M_Q4_0)
#pragma unroll
                for (int ct = 0; ct < CT; ct++)
#pragma unroll
                    for (int r = 0; r < 4; r++) c[ct][r] = fmaf(c[ct][r], qs[ct].unit, -m[ct]);
#pragma unroll
            for (int ct = 0; ct < CT; ct++)
#pragma unroll
                for (int r = 0; r < 4; r++) p[ct][4 * f + r] = !MASK || p0 + 4 * f + r < upto[ct] ? c[ct][r] : -INFINITY;
        }
        uint32_t four = 0;
        if constexpr (DT != L3M_Q4_0) four = keys.four;
        uint32_t none = 0;                                           // exponents of positions that no row sees do not count
        if constexpr (DT != L3M_Q4_0 && MASK) none = behind(tile, end);
        const bool fits = DT == L3M_Q4_0 || narrow(four, none);
        keys.load(H, next, lane);
        float to_unit = 1.f;
        uint32_t nan[CT];                                            // blocks whose value is NaN at a position the row sees
#pragma unroll
        for (int ct = 0; ct < CT; ct++) nan[ct] = 0;
        if constexpr (DT != L3M_Q4_0) {
            if ((unit || !fits) && (unit || !narrow_or_zero(four, none))) {
                to_unit = fit_unit(tile, four | none);
                if constexpr (MASK)                                  // NaN for the rows that see it, and for no other: 0 here, put in below
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            if ((vals.e[b][i >> 2] >> 8 * (i & 3) & 255u) == E8M0_NAN) {
                                vals.e[b][i >> 2] ^= 128u << 8 * (i & 3);   // 127; a NaN block's codes are 0
#pragma unroll
                                for (int ct = 0; ct < CT; ct++) nan[ct] |= p0 + i < upto[ct] ? 1u << b : 0u;
                            }
            }
        }
        f16x8 hi[CT], lo[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; i++) e[i] = __builtin_amdgcn_exp2f(p[ct][i]);
            if (__ballot(max8(e) > lim[ct]) || to_unit != 1.f) {
                const float top = max_g4(max8(p[ct]));
                const bool move = top > (lim[ct] < 0.f ? -INFINITY : base[ct] + RISE);
                // a row's first maximum scales nothing: 2^-up of one below -121 is infinite, and the sums are zeros
                const float up = move ? top - base[ct] : 0.f, f = lim[ct] < 0.f ? 1.f : __builtin_amdgcn_exp2f(-up);
                if (move) lim[ct] = __builtin_amdgcn_exp2f(base[ct] + RISE);
                m[ct] += up;
                l[ct] *= f;
                scale_acc(ct, f * (each && seen[ct] != end ? 1.f : to_unit));
#pragma unroll
                for (int i = 0; i < 8; i++) e[i] = __builtin_amdgcn_exp2f(p[ct][i] - up);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                p[ct][i] = e[i];
                l[ct] += e[i];
            }
            if constexpr (DT != L3M_Q4_0) two_parts(p[ct], hi[ct], lo[ct]);
        }
        if constexpr (DT == L3M_Q4_0) {
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                float w[NB][8], most = 0.f;
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        w[b][i] = fmaf(p[ct][i], (float)vals.d[b][i], 0.f);
                        if constexpr (MASK) w[b][i] = p0 + i < upto[ct] ? w[b][i] : 0.f;   // a masked position's scale may be anything
                        if (i & 1) most = fmaxf(fmaxf(most, fabsf(w[b][i - 1])), fabsf(w[b][i]));
                    }
                // past f16 soon, so a scale of more than 2^(8 - base): base goes by the largest one here, and 2^(base + RISE) times it is below
                // 2^16 again. It goes by the scale, not by the product, whose weight may lie anywhere above 2^base: the next maximum's weight is 2^base,
                // and times the largest scale still 2^7. An infinite scale, which only memory that was never written holds, has no part in that
                most = most < INFINITY ? most : 0.f;
                if (__ballot(most > 65000.f)) {
                    const float top = max_g4(most);
                    uint32_t u = 0;
                    for (int b = 0; b < NB; b++) {                   // read again: the registers are the weights' by now
                        const f16x8 at = *(const f16x8 *)(H.vs + 2 * (((size_t)tile * NB + b) * TILE + 8 * g4));
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const _Float16 d = at[i];
                            const uint32_t x = __builtin_bit_cast(uint16_t, d) & 0x7FFFu;
                            u = max(u, x < 0x7C00u && (!MASK || p0 + i < upto[ct]) ? x : 0u);
                        }
                    }
                    const float d = max_g4((float)__builtin_bit_cast(_Float16, (uint16_t)u));
                    const int   k = top > 65000.f ? (int)base[ct] - 134 + (int)(__float_as_uint(d) >> 23) : 0;
                    const float f = __uint_as_float((uint32_t)(127 - k) << 23);
                    scale_acc(ct, f);
                    l[ct] *= f;
                    m[ct] += (float)k;
                    lim[ct] *= lim[ct] < 0.f ? 1.f : f;
                    base[ct] -= (float)k;
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int i = 0; i < 8; i++) w[b][i] *= f;
                }
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const f16x8 v0 = widen_f16(vals.q[2 * b]), v1 = widen_f16(vals.q[2 * b + 1]);
                    two_parts(w[b], hi[ct], lo[ct]);
                    acc[ct][2 * b] = mfma(v0, lo[ct], mfma(v0, hi[ct], acc[ct][2 * b]));
                    acc[ct][2 * b + 1] = mfma(v1, lo[ct], mfma(v1, hi[ct], acc[ct][2 * b + 1]));
                }
            }
        } else {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                float d[8];
                f16x8 v0, v1;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    d[i] = pow2_byte(vals.e[b][i >> 2], i & 3);
                    if constexpr (MASK) d[i] = p0 + i < end ? d[i] : 1.f;
                }
                widen_v(&vals.q[2 * b], d, v0, v1);
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    acc[ct][2 * b] = mfma(v0, lo[ct], mfma(v0, hi[ct], acc[ct][2 * b]));
                    acc[ct][2 * b + 1] = mfma(v1, lo[ct], mfma(v1, hi[ct], acc[ct][2 * b + 1]));
                }
            }
            if constexpr (MASK)
#pragma unroll
                for (int ct = 0; ct < CT; ct++)
                    if (__ballot(nan[ct] != 0))
#pragma unroll
                        for (int b = 0; b < NB; b++)
                            if (max_g4((float)(nan[ct] >> b & 1u)) != 0.f) acc[ct][2 * b] = acc[ct][2 * b + 1] = f32x4{NAN, NAN, NAN, NAN};
        }
        vals.load(H, next, lane);
    };
    int tile = t0;
    for (; tile < min(t1, (int)whole); tile++) step(tile, min(tile + 1, t1 - 1), INT_MAX, false, std::false_type{});
    // mxfp4 exponents of a masked tile that are not all f16's: a token at a time, in a unit of its own, so that no token's output hangs on
    // positions behind it
    int range[CT];                                                   // of a row's token: high, unit (16 bits each)
    auto pack = [&] { return high * 65536 | (unit & 0xFFFF); };
#pragma unroll
    for (int ct = 0; ct < CT; ct++) range[ct] = pack();
    for (; tile < t1; tile++) {
        const int end = a.pos + last + 1;
        bool each = false;
        if constexpr (DT != L3M_Q4_0) {
            each = !narrow_or_zero(keys.four, behind(tile, end));
#pragma unroll
            for (int ct = 0; ct < CT; ct++) each = each || __ballot((range[ct] & 0xFFFF) != 0);
        }
        for (int to = each ? a.pos + first + 1 : end; to <= end; to++) {
            if (each)
#pragma unroll
                for (int ct = 0; ct < CT; ct++)
                    if (const uint64_t rows_of = __ballot(seen[ct] == to)) {
                        const int r = __builtin_amdgcn_readlane(range[ct], __builtin_ctzll(rows_of));
                        unit = (int16_t)r;
                        high = r >> 16;
                    }
            step(tile, to < end ? tile : min(tile + 1, t1 - 1), to, each, std::true_type{});
#pragma unroll
            for (int ct = 0; ct < CT; ct++) range[ct] = each && seen[ct] == to ? pack() : range[ct];
        }
    }
    if constexpr (DT != L3M_Q4_0) {
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            const int u = (int16_t)range[ct];
            const bool far = range[ct] >> 16 > 60;                   // sums of values near float32's end: weights 2^-48 of what they were
            if (__ballot(u != 0 || far)) {
                scale_acc(ct, ldexpf(1.f, far ? u - 48 : u));
                l[ct] *= far ? 0x1p-48f : 1.f;
                m[ct] += far ? 48.f : 0.f;
            }
        }
    }

    // the wavefronts' parts at their common maximum; where LDS has no room for all, the second half first and the first half onto them
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        l[ct] = sum_g4(l[ct]);
        if (lim[ct] < 0.f) m[ct] = M0;                               // nothing seen
        if (g4 == 0) {
            m_s[wave][16 * ct + r16] = m[ct];
            l_s[wave][16 * ct + r16] = l[ct];
        }
    }
    auto put_acc = [&](int at, auto add, const float (&f)[CT]) {
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
#pragma unroll
            for (int t = 0; t < 2 * NB; t++) {
                f32x4 &to = *(f32x4 *)&o_s[at][16 * ct + r16][16 * t + 4 * g4];
                if constexpr (decltype(add)::value) to += acc[ct][t] * f[ct];
                else to = acc[ct][t] * f[ct];
            }
    };
    float f[CT];
    if constexpr (O_WAVES == WAVES) {
#pragma unroll
        for (int ct = 0; ct < CT; ct++) f[ct] = 1.f;
        put_acc(wave, std::false_type{}, f);
        __syncthreads();
    } else {
        __syncthreads();
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            float top = m_s[0][16 * ct + r16];
#pragma unroll
            for (int w = 1; w < WAVES; w++) top = fmaxf(top, m_s[w][16 * ct + r16]);
            f[ct] = __builtin_amdgcn_exp2f(m[ct] - top);
        }
        if (wave >= O_WAVES) put_acc(wave - O_WAVES, std::false_type{}, f);
        __syncthreads();
        if (wave < O_WAVES) put_acc(wave, std::true_type{}, f);
        __syncthreads();
    }
    const unsigned quads = (unsigned)hd >> 2;
    for (unsigned i = threadIdx.x; i < rows * quads; i += 64 * WAVES) {
        const unsigned r = __umulhi(i, a.quad_mul), d = 4 * (i - r * quads);
        float top = m_s[0][r], sum = 0.f;
#pragma unroll
        for (int w = 1; w < WAVES; w++) top = fmaxf(top, m_s[w][r]);
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const float e = __builtin_amdgcn_exp2f(m_s[w][r] - top);
            sum = fmaf(l_s[w][r], e, sum);
            if constexpr (O_WAVES == WAVES) x += *(const f32x4 *)&o_s[w][r][d] * e;
            else if (w < O_WAVES) x += *(const f32x4 *)&o_s[w][r][d];
        }
        const unsigned row = row0 + r, t = divide(row, g, a.g_mul);
        const size_t at = (size_t)t * a.nq + h * g + (row - t * (unsigned)g);
        if (a.splits == 1) *(f32x4_a4 *)(a.out + at * hd + d) = x / sum;
        else {
            const size_t to = at * a.splits + split;
            *(f32x4 *)(a.parts + to * hd + d) = x;
            if (d == 0) *(f32x2 *)(a.ml + 2 * to) = f32x2{top, sum};
        }
    }
}

// The splits' parts of a row, one workgroup a (token, query head): groups of hd / 4 lanes take every so many splits, 16 bytes a lane and
// eight loads in flight while every wavefront makes the splits' factors for itself; they meet in LDS in a fixed order. Bound by latency: 2.4 us
// for 32 rows of 32 parts, 3.8 of 64. As the last workgroup's work in the launch before (tickets in memory) it took as long.
__global__ void __launch_bounds__(256) k_kv4_join(AttendIn a) {
    __shared__ float f_s[4][SPLITS];
    __shared__ f32x4 o_s[256];
    const unsigned tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hd = a.c.hd, S = a.splits, quads = hd >> 2;
    const unsigned mine = __umulhi(tid, a.quad_mul), groups = __umulhi(256, a.quad_mul), d = 4 * (tid - mine * quads);
    const float *part = a.parts + (size_t)blockIdx.x * S * hd + d, *ml = a.ml + (size_t)blockIdx.x * S * 2;
    f32x2 v[SPLITS / 64];
#pragma unroll
    for (int i = 0; i < SPLITS / 64; i++) v[i] = i == 0 || 64u * i < S ? *(const f32x2 *)(ml + 2 * min(lane + 64 * i, S - 1)) : f32x2{M0, 0.f};
    f32x4 x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = *(const f32x4 *)(part + (size_t)min(mine + i * groups, S - 1) * hd);
    float top = v[0].x, sum = 0.f;
#pragma unroll
    for (int i = 1; i < SPLITS / 64; i++) top = fmaxf(top, v[i].x);
    top = max_wave(top);
#pragma unroll
    for (int i = 0; i < SPLITS / 64; i++) {
        const float f = __builtin_amdgcn_exp2f(v[i].x - top);
        if (lane + 64 * i < S) {
            sum = fmaf(v[i].y, f, sum);
            f_s[wave][lane + 64 * i] = f;
        }
    }
    sum = sum_wave(sum);
    wave_sync();
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (mine < groups)
        for (unsigned s = mine; s < S; s += 8 * groups) {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (s + i * groups < S) o += x[i] * f_s[wave][s + i * groups];
            if (s + 8 * groups < S)
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = *(const f32x4 *)(part + (size_t)min(s + (8 + i) * groups, S - 1) * hd);
        }
    o_s[tid] = o;
    __syncthreads();
    if (tid < quads) {
        for (unsigned i = 1; i < groups; i++) o += o_s[i * quads + tid];
        *(f32x4_a4 *)(a.out + (size_t)blockIdx.x * hd + d) = o / sum;
    }
}

// ---------------------------------------------------------------- argument checks

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
bool kv4_dtype(int dt) { return dt == L3M_Q4_0 || dt == L3M_MXFP4; }
bool kv4_shape(int dt, int nkv, int hd, int cap) {
    return kv4_dtype(dt) && nkv >= 1 && nkv <= 65536 && hd >= 8 && hd <= HD_MAX && hd % 8 == 0 && cap >= 1 && cap <= 1 << 30;
}
size_t codes_bytes(int nkv, int hd, int cap) { return (size_t)nkv * ((cap + TILE - 1) / TILE) * 512 * ((hd + 31) / 32); }
size_t scales_bytes(int dt, int nkv, int hd, int cap) { return (size_t)nkv * ((cap + TILE - 1) / TILE) * TILE * ((hd + 31) / 32) * sbytes(dt); }
bool overlap(const void *a, size_t na, const void *b, size_t nb) {
    return na && nb && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}
// Whether n bytes at p (NULL: none) lie on the cache's memory.
bool on_cache(const l3m_kv4 *c, const void *p, size_t n) {
    const size_t q = codes_bytes(c->nkv, c->hd, c->cap), s = scales_bytes(c->dtype, c->nkv, c->hd, c->cap);
    return p && (overlap(p, n, c->kq, q) || overlap(p, n, c->ks, s) || overlap(p, n, c->vq, q) || overlap(p, n, c->vs, s));
}
const char *kv4_bad(const l3m_kv4 *c) {
    if (!c || !kv4_shape(c->dtype, c->nkv, c->hd, c->cap)) return "kv4: not a cache of q4_0 or mxfp4 blocks, hd a multiple of 8 up to 256";
    if (!c->kq || !c->ks || !c->vq || !c->vs) return "kv4: a cache without memory";
    if (((uintptr_t)c->kq | (uintptr_t)c->vq | (uintptr_t)c->ks | (uintptr_t)c->vs) % 16) return "kv4: planes must be 16-byte aligned";
    const size_t q = codes_bytes(c->nkv, c->hd, c->cap), s = scales_bytes(c->dtype, c->nkv, c->hd, c->cap);
    if (overlap(c->kq, q, c->vq, q) || overlap(c->ks, s, c->vs, s) || overlap(c->kq, q, c->ks, s) || overlap(c->kq, q, c->vs, s) ||
        overlap(c->vq, q, c->ks, s) || overlap(c->vq, q, c->vs, s))
        return "kv4: planes overlap";
    return nullptr;
}
bool span_ok(const l3m_kv4 *c, int pos, int n) { return pos >= 0 && n >= 1 && pos <= c->cap && n <= c->cap - pos; }
// The stream of a call that names none: the library's, made now if this is its first call. False: there is no device, or it was shut down.
bool stream_of(void *s, hipStream_t &st) {
    if (!s && l3m_dev_init()) {
        l3m_dev_fail("no usable device, or the library was shut down");
        return false;
    }
    st = (hipStream_t)(s ? s : l3m_dev_stream());
    return true;
}

// The rows of the table that a call reads, n of hd floats.
const float *table_rows(const RowsIn &a) { return a.table ? a.table + (size_t)a.pos * a.hd : nullptr; }
// What is wrong with a call's rows and outputs, or NULL. An output may be the rows' own heads only where a token's are dense: one token.
const char *rows_bad(const RowsIn &a, bool floats) {
    const long long width = (long long)(a.nq + (floats ? 1 : 2) * (long long)a.nkv) * a.hd;
    if (a.n < 1 || a.nq < 0 || a.nq > 65536 || a.nkv < 0 || a.nkv > 65536 || a.nq + a.nkv < 1 || a.pos < 0 || a.pos > 0x7FFFFFFF - a.n) return "rows: counts out of range";
    if (!a.x || a.stride < width) return "rows: a row holds fewer values than its heads";
    if ((a.nq && !a.q) || (floats && a.nkv && !a.k)) return "rows: no output";
    if ((a.wq || a.wk) && !(a.eps >= 0.f)) return "rows: eps is negative or NaN";
    if (((uintptr_t)a.x | (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.wq | (uintptr_t)a.wk | (uintptr_t)a.table) % 4) return "rows: floats must be 4-byte aligned";
    const size_t in = 4 * ((size_t)(a.n - 1) * a.stride + width), nqb = 4 * (size_t)a.n * a.nq * a.hd, nkb = floats ? 4 * (size_t)a.n * a.nkv * a.hd : 0;
    const bool one = a.n == 1;
    if (overlap(a.q, nqb, a.x, in) && !(one && a.q == a.x)) return "rows: q overlaps the rows";
    if (overlap(a.k, nkb, a.x, in) && !(one && a.k == a.x + (size_t)a.nq * a.hd)) return "rows: k overlaps the rows";
    if (overlap(a.q, nqb, a.k, nkb)) return "rows: q overlaps k";
    const size_t w = 4 * (size_t)a.hd;
    const float *turn = table_rows(a);
    auto read = [&](const float *to, size_t n) {
        return (a.wq && overlap(to, n, a.wq, w)) || (a.wk && overlap(to, n, a.wk, w)) || (turn && overlap(to, n, turn, w * a.n));
    };
    if (read(a.q, nqb) || read(a.k, nkb)) return "rows: q or k overlaps the weights or the table";
    return nullptr;
}
template <int DT> void launch_rows_in(RowsIn a, const l3m_kv4 &c, hipStream_t st) {
    a.lg = DT >= 0 ? 2 : 0;                                          // a block's four lanes at least
    while (8 << a.lg < a.hd) a.lg++;
    const unsigned per = 64u >> a.lg, items = (unsigned)((long long)a.n * (a.nq + a.nkv));
    a.qk_waves = (items + per - 1) / per;
    unsigned waves = a.qk_waves;
    if (DT >= 0) waves += (unsigned)(((a.pos + a.n - 1) >> 3) - (a.pos >> 3) + 1) * a.nkv * (((a.hd + 31) / 32 + 1) / 2);
    const dim3 grid((waves + 3) / 4);
    if (a.hd % 8 == 0) hipLaunchKernelGGL((k_rows_in<DT, true>), grid, dim3(256), 0, st, a, c);
    else if constexpr (DT < 0) hipLaunchKernelGGL((k_rows_in<DT, false>), grid, dim3(256), 0, st, a, c);
}
// Columns of 16 rows a workgroup takes of each kv head's `rows`. Two share a tile's conversions, which pays for mxfp4 heads of 33 to 128
// where every CU has two workgroups all the same and a last turn of them is not nearly empty: 1024 tokens behind 2999, 32 heads over 8,
// hd 128: 98 us, one column 115 (96: 86 and 100, 64: 67 and 77); 128 tokens behind 2000: 22 us, one column 15; 564 workgroups (1500
// tokens, 12 heads of 128) 28.8 and 25.4, 640 (1024 behind 2000, 20 heads over 5) 55.4 and 56. q4_0's do not pay: hd 128 has no registers
// (228 us with two, 177 with one), hd 64 96 and 95.
int tile_columns(int dt, int nb, int nkv, long long rows) {
    const long long two = nkv * ((rows + 31) / 32), turns = (two + 511) / 512;
    return dt == L3M_MXFP4 && nb >= 2 && nb <= 4 && two >= 512 && 5 * two >= 3 * 512 * turns ? 2 : 1;
}
template <int DT> void launch_attend(AttendIn a, int ct, hipStream_t st) {
    for (; a.group0 < a.groups; a.group0 += 65535) {                 // a grid's last dimension
        const dim3 grid(a.c.nkv, a.splits, a.groups - a.group0 < 65535 ? a.groups - a.group0 : 65535), wg(64 * WAVES);
#define ATTEND(NB, CT) hipLaunchKernelGGL((k_kv4_attend<DT, NB, CT>), grid, wg, 0, st, a)
        if constexpr (DT == L3M_MXFP4)
            if (ct == 2) {
                if (a.c.hd <= 64) ATTEND(2, 2);
                else if (a.c.hd <= 96) ATTEND(3, 2);
                else ATTEND(4, 2);
                continue;
            }
        switch ((a.c.hd + 31) / 32) {
        case 1: ATTEND(1, 1); break;
        case 2: ATTEND(2, 1); break;
        case 3: ATTEND(3, 1); break;
        case 4: ATTEND(4, 1); break;
        case 5: ATTEND(5, 1); break;
        case 6: ATTEND(6, 1); break;
        case 7: ATTEND(7, 1); break;
        default: ATTEND(8, 1); break;
        }
#undef ATTEND
    }
}
// Workgroups that share the positions of 16 rows, with `alone` workgroups unsplit. A split costs the join, 2.5 us and more with the rows'
// parts; a tile costs a wavefront 0.2 us and 0.2 (q4_0) or 0.1 (mxfp4) a block. Unsplit against split over 78 shapes of 1 to 64 tokens and 128
// to 2048 positions, heads of 32 to 256 (the rule is at most 5% off the better one, 0.15% on average), one token of 32 heads over 8 of 128:
// q4_0 over 256 positions 5.5 and 7.2 us, 512: 7.6 and 7.3, 1024: 11.5 and 7.4; mxfp4 over 512: 6.0 and 6.9, 1024: 8.3 and 6.9; 64 tokens of
// 2048: mxfp4 14.7 and 15.1, q4_0 21 and 19. Down to a tile a wavefront: against two tiles, one token over 1024 (q4_0) 7.3 and 8.3 us. Up to
// one workgroup a CU, two where a wavefront has six tiles all the same (then they hide each other's loads; between the two some CUs
// are left with half): one token over 32768 (mxfp4, 32 heads over 8 of 128; caches past the Infinity Cache in turn) 15.0 us with one, 16.1 with
// two; 131071: 38.4 and 34.6, q4_0 49.4 and 46.9; 16 tokens behind 2000 9.6 and 11.9.
int split_count(int dt, long long alone, int tiles, int nb, long long rows) {
    const bool q4 = dt == L3M_Q4_0;
    if ((long long)tiles * (nb + (q4 ? 1 : 2)) <= (q4 ? 66 : 120) + rows / 10) return 1;
    const long long two = SPLIT_WGS / alone, most = (tiles + WAVES - 1) / WAVES, room = most >= 6 * two ? two : two / 2, splits = room < most ? room : most;
    return splits < 2 ? 1 : splits < SPLITS ? (int)splits : SPLITS;
}
constexpr long long MAX_ITEMS = (1ll << 26) - 4;                     // wavefronts of a launch (its threads are counted in 32 bits)

}  // namespace

extern "C" {

size_t l3m_kv4_bytes(int dtype, int nkv, int hd, int cap) {
    if (!kv4_shape(dtype, nkv, hd, cap)) return 0;
    return 2 * (up256(codes_bytes(nkv, hd, cap)) + up256(scales_bytes(dtype, nkv, hd, cap)));
}

int l3m_kv4_init(l3m_kv4 *c, int dtype, int nkv, int hd, int cap, void *mem) {
    if (!c || !mem || (uintptr_t)mem % 16) return l3m_dev_fail("kv4: memory must be 16-byte aligned");
    if (!kv4_shape(dtype, nkv, hd, cap)) return l3m_dev_fail("kv4: q4_0 or mxfp4, at least one kv head and position, hd a multiple of 8 up to 256");
    const size_t q = up256(codes_bytes(nkv, hd, cap)), s = up256(scales_bytes(dtype, nkv, hd, cap));
    uint8_t *m = (uint8_t *)mem;
    *c = l3m_kv4{m, m + q, m + q + s, m + 2 * q + s, nkv, hd, cap, dtype};
    return 0;
}

int l3m_k_qk_norm_rope(float *q, float *k, const float *rows, int stride, int n, int nq, int nkv, int hd, const float *wq, const float *wk,
                       float eps, int halves, int pos, const float *table, void *stream) {
    if (hd < 2 || hd > HD_MAX || hd % 2) return l3m_dev_fail("qk_norm_rope: hd must be even and at most 256");
    const RowsIn a = {rows, wq, wk, table, q, k, stride, n, nq, nkv, hd, halves != 0, pos, 0, 0, eps};
    if (const char *why = rows_bad(a, true)) return l3m_dev_fail(why);
    if ((long long)n * (nq + nkv) > MAX_ITEMS) return l3m_dev_fail("qk_norm_rope: too many rows for one call");
    hipStream_t st;
    if (!stream_of(stream, st)) return -1;
    launch_rows_in<-1>(a, l3m_kv4{}, st);
    return l3m_dev_launched("k_qk_norm_rope");
}

int l3m_k_kv4_append(const l3m_kv4 *c, float *q, const float *rows, int stride, int n, int nq, const float *wq, const float *wk, float eps,
                     int halves, int pos, const float *table, void *stream) {
    if (const char *why = kv4_bad(c)) return l3m_dev_fail(why);
    if (!span_ok(c, pos, n)) return l3m_dev_fail("kv4_append: positions past the cache's end");
    const RowsIn a = {rows, wq, wk, table, q, nullptr, stride, n, nq, c->nkv, c->hd, halves != 0, pos, 0, 0, eps};
    if (const char *why = rows_bad(a, false)) return l3m_dev_fail(why);
    const size_t w = 4 * (size_t)c->hd;
    if (on_cache(c, q, w * n * nq) || on_cache(c, rows, 4 * ((size_t)(n - 1) * stride + (size_t)(nq + 2 * c->nkv) * c->hd)) || on_cache(c, wq, w) ||
        on_cache(c, wk, w) || on_cache(c, table_rows(a), w * n))
        return l3m_dev_fail("kv4_append: rows, queries, weights or table overlap the cache");
    if ((long long)n * (nq + 2 * c->nkv) > MAX_ITEMS) return l3m_dev_fail("kv4_append: too many rows for one call");
    hipStream_t st;
    if (!stream_of(stream, st)) return -1;
    if (c->dtype == L3M_Q4_0) launch_rows_in<L3M_Q4_0>(a, *c, st);
    else launch_rows_in<L3M_MXFP4>(a, *c, st);
    return l3m_dev_launched("k_kv4_append");
}

int l3m_k_kv4_rows(const l3m_kv4 *c, float *k, float *v, int pos, int n, void *stream) {
    if (const char *why = kv4_bad(c)) return l3m_dev_fail(why);
    if (!span_ok(c, pos, n)) return l3m_dev_fail("kv4_rows: positions past the cache's end");
    if ((!k && !v) || ((uintptr_t)k | (uintptr_t)v) % 4) return l3m_dev_fail("kv4_rows: no output, or one that is not 4-byte aligned");
    const size_t vals = (size_t)n * c->nkv * c->hd;
    if (vals > (size_t)MAX_ITEMS * 64) return l3m_dev_fail("kv4_rows: too many rows for one call");
    if (k && v && overlap(k, 4 * vals, v, 4 * vals)) return l3m_dev_fail("kv4_rows: k overlaps v");
    if (on_cache(c, k, 4 * vals) || on_cache(c, v, 4 * vals)) return l3m_dev_fail("kv4_rows: k or v overlaps the cache");
    const unsigned k_threads = k ? (unsigned)((vals / 8 + 255) / 256 * 256) : 0;
    const size_t v_threads = v ? (size_t)(((pos + n - 1) >> 3) - (pos >> 3) + 1) * c->nkv * c->hd : 0;
    const dim3 grid((unsigned)((k_threads + v_threads + 255) / 256));
    hipStream_t st;
    if (!stream_of(stream, st)) return -1;
    if (c->dtype == L3M_Q4_0) hipLaunchKernelGGL(k_kv4_rows<L3M_Q4_0>, grid, dim3(256), 0, st, *c, k, v, pos, n, k_threads);
    else hipLaunchKernelGGL(k_kv4_rows<L3M_MXFP4>, grid, dim3(256), 0, st, *c, k, v, pos, n, k_threads);
    return l3m_dev_launched("k_kv4_rows");
}

size_t l3m_kv4_work_bytes(const l3m_kv4 *c, int n, int nq) {
    if (kv4_bad(c) || n < 1 || n > c->cap || nq < 1 || nq > 65536 || nq % c->nkv) return 0;
    const size_t rows = (size_t)n * (nq / c->nkv);                   // a workgroup's of a split: 16 at most
    return 4 * (size_t)SPLIT_WGS * (rows < 16 ? rows : 16) * (c->hd + 2) + 16;
}

int l3m_k_kv4_attend(float *out, const float *q, const l3m_kv4 *c, int n, int nq, int pos, void *work, size_t work_bytes, void *stream) {
    if (const char *why = kv4_bad(c)) return l3m_dev_fail(why);
    if (!span_ok(c, pos, n)) return l3m_dev_fail("kv4_attend: positions past the cache's end");
    if (nq < 1 || nq > 65536 || nq % c->nkv) return l3m_dev_fail("kv4_attend: query heads must be a multiple of the kv heads");
    const size_t rows = (size_t)n * nq, bytes = 4 * rows * c->hd;
    if (!out || !q || ((uintptr_t)out | (uintptr_t)q) % 4 || (out != q && overlap(out, bytes, q, bytes)))
        return l3m_dev_fail("kv4_attend: q and out must be floats, the same or apart");
    const size_t need = l3m_kv4_work_bytes(c, n, nq);
    if (!work || (uintptr_t)work % 16 || work_bytes < need) return l3m_dev_fail("kv4_attend: the workspace is too small (l3m_kv4_work_bytes) or not 16-byte aligned");
    if (overlap(work, need, q, bytes) || overlap(work, need, out, bytes)) return l3m_dev_fail("kv4_attend: the workspace overlaps q or out");
    if (on_cache(c, out, bytes) || on_cache(c, work, need)) return l3m_dev_fail("kv4_attend: out or the workspace overlaps the cache");
    if (rows > (size_t)MAX_ITEMS) return l3m_dev_fail("kv4_attend: too many rows for one call");
    const long long R = (long long)n * (nq / c->nkv);
    const int ct = tile_columns(c->dtype, (c->hd + 31) / 32, c->nkv, R), per = 16 * ct, groups = (int)((R + per - 1) / per), tiles = (pos + n + TILE - 1) / TILE;
    const long long alone = (long long)c->nkv * groups;
    const int splits = split_count(c->dtype, alone, tiles, (c->hd + 31) / 32, (long long)rows);
    const int g = nq / c->nkv;
    float *ml = (float *)work;
    const AttendIn a = {out, ml, ml + (2 * rows * splits + 3) / 4 * 4, q, *c, n, nq, g, pos, groups, 0, splits, multiplier(g, (uint32_t)R), multiplier(c->hd / 4, 4096),
                        multiplier(splits * WAVES, (uint32_t)tiles)};
    hipStream_t st;
    if (!stream_of(stream, st)) return -1;
    if (c->dtype == L3M_Q4_0) launch_attend<L3M_Q4_0>(a, ct, st);
    else launch_attend<L3M_MXFP4>(a, ct, st);
    if (splits > 1) hipLaunchKernelGGL(k_kv4_join, dim3((unsigned)rows), dim3(256), 0, st, a);
    return l3m_dev_launched("k_kv4_attend");
}

}
