// A K/V cache of 4-bit blocks for CDNA4 (gfx950): the norm and rotation of query and key heads, the writer that stores K and V rows
// behind it in the same pass, the read-back, and the attention of one token or many over the cache.
//
// Layout. Per kv head, tiles of 32 positions; NB = ceil(hd / 32) blocks of 32 dimensions, a last block short of dimensions filled
// with zeros. A tile is laid out as the matrix cores' operands, so a lane's words are one contiguous load and no value crosses lanes:
//   K codes  [nkv][tile][half 2][lane 64][NB words]   lane 16 c + m, half f: position 8 (m / 4) + 4 f + m % 4, word b its dimensions
//                                                     32 b + 8 c .. + 7
//   V codes  [nkv][tile][lane 64][2 NB words]         lane 16 g + j: word t holds dimension 16 t + j of positions 8 g .. 8 g + 7
//   scales   [nkv][tile][NB][32 positions]            of K and of V: f16 d (q4_0), a biased exponent byte (mxfp4)
// Both codes of a tile and head take 512 NB bytes. Element i of a word's eight (a dimension of K, a position of V) is the nibble at
// bit nib(dt, i): q4_0's masked bytes are then elements 0..3 and 4..7, mxfp4's byte pairs come in order.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
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
// The word of K that holds dimensions d .. d + 7 (d a multiple of 8) of position p, of V that holds dimension d of p's eight positions,
// and the element of the scale of position p's block b.
__device__ __forceinline__ size_t k_word(int nb, int p, int d) {
    const int w = p & 31, lane = ((d & 31) >> 3) * 16 + (w >> 3) * 4 + (w & 3);
    return ((size_t)(p >> 5) * 128 + ((w >> 2) & 1) * 64 + lane) * nb + (d >> 5);
}
__device__ __forceinline__ size_t v_word(int nb, int p, int d) {
    return ((size_t)(p >> 5) * 64 + ((p & 31) >> 3) * 16 + (d & 15)) * 2 * nb + (d >> 4);
}
__device__ __forceinline__ size_t scale_at(int nb, int p, int b) { return ((size_t)(p >> 5) * nb + b) * TILE + (p & 31); }

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
// Blocks of 32 values, one a lane of half a wavefront: this lane's code, and the block's scale as it is stored (the same in every
// lane). The file formats' rounding to the nearest (l3m_quantize_row), in the same float32 steps, so the stored bytes do not depend on
// where a row is quantized; a block holding a value that is not finite reads as NaN, a scale past f16 saturates, mxfp4 exponents end at
// 2^-126.
template <int DT> __device__ __forceinline__ uint32_t quantize(float x, uint32_t &stored) {
#pragma clang fp contract(off)
    const uint32_t mag = __float_as_uint(x) & 0x7FFFFFFFu;
    uint32_t peak = mag;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) peak = max(peak, (uint32_t)__shfl_xor((int)peak, m));
    const bool bad = peak >= 0x7F800000u;
    if constexpr (DT == L3M_Q4_0) {
        const uint64_t held = __ballot(mag == peak) >> (threadIdx.x & 32) & 0xFFFFFFFFu;     // the first of equal ones gives the sign
        const float top = __shfl(x, (int)(threadIdx.x & 32) + __builtin_ctzll(held | 1ull << 32), 64);
        const float d = top * -0.125f, r = d != 0.f ? 1.0f / d : 0.f, scaled = x * r, v = floorf(scaled + 8.5f);
        stored = bad ? 0x7E00u : __builtin_bit_cast(uint16_t, (_Float16)fminf(fmaxf(d, -65504.f), 65504.f));
        return bad ? 8u : v <= 0.f ? 0u : v >= 15.f ? 15u : (uint32_t)(int)v & 15u;
    } else {
        const int e = max((int)(peak >> 23) - 2, 1);
        const float y = fabsf(x) * __uint_as_float((uint32_t)(254 - e) << 23);               // exact
        const uint32_t c = (y > 0.25f) + (y > 0.75f) + (y > 1.25f) + (y > 1.75f) + (y > 2.5f) + (y > 3.5f) + (y > 5.f);
        stored = bad ? (uint32_t)E8M0_NAN : (uint32_t)e;
        return bad || !c ? 0u : c | (x < 0.f ? 8u : 0u);
    }
}
template <int DT> __device__ __forceinline__ void put_scale(uint8_t *s, size_t i, uint32_t stored) {
    if constexpr (DT == L3M_Q4_0) ((uint16_t *)s)[i] = (uint16_t)stored;
    else s[i] = (uint8_t)stored;
}

struct RowsIn {
    const float *x, *wq, *wk, *table;
    float       *q, *k;
    long long    stride;
    int          n, nq, nkv, hd, halves, pos;
    float        eps;
};

// Norm and rotation of one head row by one wavefront: pair i of the rotation in lane i % 64, x s w with s = 1 / sqrt(mean x^2 + eps),
// then the pair turned by the table's angle. In 64 bits up to the one rounding of each result, because a key's 4-bit code hangs on which
// side of a border it lies: the row is the float32 nearest to the formula's, whatever the order of the sum.
constexpr int PAIRS = HD_MAX / 2 / 64;
__device__ __forceinline__ void norm_rope(const RowsIn &a, const float *x, const float *w, const float *cs, float out[PAIRS][2]) {
    const int lane = threadIdx.x & 63, np = a.hd >> 1, second = a.halves ? np : 1, step = a.halves ? 1 : 2;
    double v[PAIRS][2], ss = 0;
#pragma unroll
    for (int i = 0; i < PAIRS; i++) {
        const int p = lane + 64 * i;
        v[i][0] = p < np ? (double)x[step * p] : 0;
        v[i][1] = p < np ? (double)x[step * p + second] : 0;
        ss += v[i][0] * v[i][0] + v[i][1] * v[i][1];
    }
    double s = 1;
    if (w) {
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) ss += __shfl_xor(ss, m);
        s = 1.0 / sqrt(ss / a.hd + (double)a.eps);
    }
#pragma unroll
    for (int i = 0; i < PAIRS; i++) {
        const int p = lane + 64 * i;
        if (p >= np) continue;
        double y0 = v[i][0], y1 = v[i][1];
        if (w) {
            y0 *= s * (double)w[step * p];
            y1 *= s * (double)w[step * p + second];
        }
        if (cs) {
            const double c = (double)cs[2 * p], t = (double)cs[2 * p + 1], z = y0 * c - y1 * t;
            y1 = y0 * t + y1 * c;
            y0 = z;
        }
        out[i][0] = (float)y0;
        out[i][1] = (float)y1;
    }
}

// One wavefront a (token, query or key head), then one a (eight positions, kv head) of V. DT < 0: keys go to a.k as floats and V is
// left alone.
template <int DT> __global__ void __launch_bounds__(256) k_rows_in(RowsIn a, l3m_kv4 c) {
    __shared__ float row_s[4][HD_MAX];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, heads = a.nq + a.nkv, nb = (a.hd + 31) >> 5;
    const long long item = (long long)blockIdx.x * 4 + wave, qk = (long long)a.n * heads;
    if (item < qk) {
        const int t = (int)(item / heads), h = (int)(item % heads), np = a.hd >> 1, second = a.halves ? np : 1, step = a.halves ? 1 : 2;
        const bool key = h >= a.nq;
        float y[PAIRS][2];
        norm_rope(a, a.x + t * a.stride + (size_t)h * a.hd, key ? a.wk : a.wq, a.table ? a.table + (size_t)(a.pos + t) * a.hd : nullptr, y);
        float *to = row_s[wave];
        if (!key) to = a.q + ((size_t)t * a.nq + h) * a.hd;
        else if (DT < 0) to = a.k + ((size_t)t * a.nkv + h - a.nq) * a.hd;
#pragma unroll
        for (int i = 0; i < PAIRS; i++) {
            const int p = lane + 64 * i;
            if (p < np) {
                to[step * p] = y[i][0];
                to[step * p + second] = y[i][1];
            }
        }
        if constexpr (DT >= 0) {
            if (!key) return;
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            const Head H = head_of(c, nb, sbytes(DT), h - a.nq);
            const int p = a.pos + t;
            for (int d = lane; d < 32 * ((nb + 1) & ~1); d += 64) {  // both halves run as long as one has a block
                const int b = d >> 5;
                uint32_t stored, code = quantize<DT>(d < a.hd ? row_s[wave][d] : 0.f, stored) << nib(DT, d & 7);
#pragma unroll
                for (int m = 1; m < 8; m <<= 1) code |= (uint32_t)__shfl_xor((int)code, m);
                if (b < nb) {
                    if ((d & 7) == 0) H.kq[k_word(nb, p, d)] = code;
                    if ((d & 31) == 0) put_scale<DT>(H.ks, scale_at(nb, p, b), stored);
                }
            }
        }
        return;
    }
    if constexpr (DT >= 0) {
        const long long vi = item - qk;
        const int o0 = a.pos >> 3, octets = ((a.pos + a.n - 1) >> 3) - o0 + 1;
        if (vi >= (long long)octets * a.nkv) return;
        const int o = o0 + (int)(vi / a.nkv), h = (int)(vi % a.nkv), first = max(8 * o, a.pos), end = min(8 * o + 8, a.pos + a.n);
        const Head H = head_of(c, nb, sbytes(DT), h);
        const float *v = a.x + (size_t)(heads + h) * a.hd;
        for (int d = lane; d < 32 * ((nb + 1) & ~1); d += 64) {
            const int b = d >> 5;
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int p = 8 * o + i;
                x[i] = p >= first && p < end && d < a.hd ? v[(p - a.pos) * a.stride + d] : 0.f;
            }
            uint32_t word = 0, mine = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int p = 8 * o + i;
                if (p < first || p >= end) continue;                 // the same in every lane
                uint32_t stored;
                word |= quantize<DT>(x[i], stored) << nib(DT, i);
                mine |= 15u << nib(DT, i);
                if ((d & 31) == 0 && b < nb) put_scale<DT>(H.vs, scale_at(nb, p, b), stored);
            }
            if (b < nb) {
                uint32_t *to = H.vq + v_word(nb, 8 * o, d);
                *to = mine == ~0u ? word : (*to & ~mine) | word;     // the word's other positions stay
            }
        }
    }
}

// ---------------------------------------------------------------- read-back
template <int DT> __global__ void __launch_bounds__(256) k_kv4_rows(l3m_kv4 c, float *k, float *v, int pos, int n) {
    const int nb = (c.hd + 31) >> 5;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, row = i / c.hd;
    if (row >= (size_t)n * c.nkv) return;
    const int d = (int)(i % c.hd), h = (int)(row % c.nkv), p = pos + (int)(row / c.nkv), b = d >> 5;
    const Head H = head_of(c, nb, sbytes(DT), h);
    if (k) k[i] = code_value<DT>(H.kq[k_word(nb, p, d & ~7)] >> nib(DT, d & 7) & 15) * scale_value<DT>(H.ks, scale_at(nb, p, b));
    if (v) v[i] = code_value<DT>(H.vq[v_word(nb, p, d)] >> nib(DT, p & 7) & 15) * scale_value<DT>(H.vs, scale_at(nb, p, b));
}

// ---------------------------------------------------------------- attention
// One wavefront a (token, query head): 64 positions at a time, a lane scores one, then holds dimensions lane, lane + 64, .. of the
// output; running maximum and sum.
template <int DT> __global__ void __launch_bounds__(64) k_kv4_attend(float *out, const float *q, l3m_kv4 c, int nq, int pos) {
    __shared__ float q_s[HD_MAX], p_s[64];
    const int lane = threadIdx.x, hd = c.hd, nb = (hd + 31) >> 5, t = (int)(blockIdx.x / nq), hq = (int)(blockIdx.x % nq), seen = pos + t + 1;
    const Head H = head_of(c, nb, sbytes(DT), hq / (nq / c.nkv));
    for (int d = lane; d < HD_MAX; d += 64) q_s[d] = d < hd ? q[(size_t)blockIdx.x * hd + d] / sqrtf((float)hd) : 0.f;
    float m = -INFINITY, l = 0.f, o[HD_MAX / 64] = {};
    __syncthreads();
    for (int p0 = 0; p0 < seen; p0 += 64) {
        const int p = p0 + lane;
        float s = -INFINITY;
        if (p < seen) {
            s = 0.f;
            for (int b = 0; b < nb; b++) {
                float dot = 0.f;
                for (int ch = 0; ch < 4; ch++) {
                    const uint32_t w = H.kq[k_word(nb, p, 32 * b + 8 * ch)];
                    for (int i = 0; i < 8; i++) dot = fmaf(q_s[32 * b + 8 * ch + i], code_value<DT>(w >> nib(DT, i) & 15), dot);
                }
                s = fmaf(dot, scale_value<DT>(H.ks, scale_at(nb, p, b)), s);
            }
        }
        float top = s;
        for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
        const float nm = fmaxf(m, top), base = nm == -INFINITY ? 0.f : nm, f = expf(m - base), e = p < seen ? expf(s - base) : 0.f;
        float sum = e;
        for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x);
        l = l * f + sum;
        m = nm;
        p_s[lane] = e;
        __syncthreads();
        const int cnt = min(64, seen - p0);
        for (int i = 0; i < HD_MAX / 64; i++) {
            const int d = lane + 64 * i;
            if (d >= hd) break;
            o[i] *= f;
            for (int j = 0; j < cnt; j++)
                o[i] = fmaf(p_s[j], code_value<DT>(H.vq[v_word(nb, p0 + j, d)] >> nib(DT, (p0 + j) & 7) & 15) * scale_value<DT>(H.vs, scale_at(nb, p0 + j, d >> 5)), o[i]);
        }
        __syncthreads();
    }
    for (int i = 0; i < HD_MAX / 64; i++)
        if (lane + 64 * i < hd) out[(size_t)blockIdx.x * hd + lane + 64 * i] = o[i] / l;
}

// ---------------------------------------------------------------- argument checks

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
bool kv4_dtype(int dt) { return dt == L3M_Q4_0 || dt == L3M_MXFP4; }
bool kv4_shape(int dt, int nkv, int hd, int cap) {
    return kv4_dtype(dt) && nkv >= 1 && nkv <= 65536 && hd >= 8 && hd <= HD_MAX && hd % 8 == 0 && cap >= 1 && cap <= 1 << 30;
}
size_t codes_bytes(int nkv, int hd, int cap) { return (size_t)nkv * ((cap + TILE - 1) / TILE) * 512 * ((hd + 31) / 32); }
size_t scales_bytes(int dt, int nkv, int hd, int cap) { return (size_t)nkv * ((cap + TILE - 1) / TILE) * TILE * ((hd + 31) / 32) * sbytes(dt); }
const char *kv4_bad(const l3m_kv4 *c) {
    if (!c || !kv4_shape(c->dtype, c->nkv, c->hd, c->cap)) return "kv4: not a cache of q4_0 or mxfp4 blocks, hd a multiple of 8 up to 256";
    if (!c->kq || !c->ks || !c->vq || !c->vs) return "kv4: a cache without memory";
    if (((uintptr_t)c->kq | (uintptr_t)c->vq | (uintptr_t)c->ks | (uintptr_t)c->vs) % 16) return "kv4: planes must be 16-byte aligned";
    return nullptr;
}
bool span_ok(const l3m_kv4 *c, int pos, int n) { return pos >= 0 && n >= 1 && pos <= c->cap && n <= c->cap - pos; }
bool overlap(const void *a, size_t na, const void *b, size_t nb) {
    return (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}
hipStream_t as_stream(void *s) { return (hipStream_t)(s ? s : l3m_dev_stream()); }

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
    if (nqb && overlap(a.q, nqb, a.x, in) && !(one && a.q == a.x)) return "rows: q overlaps the rows";
    if (nkb && overlap(a.k, nkb, a.x, in) && !(one && a.k == a.x + (size_t)a.nq * a.hd)) return "rows: k overlaps the rows";
    if (nqb && nkb && overlap(a.q, nqb, a.k, nkb)) return "rows: q overlaps k";
    return nullptr;
}
template <int DT> void launch_rows_in(const RowsIn &a, const l3m_kv4 &c, hipStream_t st) {
    long long items = (long long)a.n * (a.nq + a.nkv);
    if (DT >= 0) items += (long long)(((a.pos + a.n - 1) >> 3) - (a.pos >> 3) + 1) * a.nkv;
    hipLaunchKernelGGL(k_rows_in<DT>, dim3((unsigned)((items + 3) / 4)), dim3(256), 0, st, a, c);
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
    const RowsIn a = {rows, wq, wk, table, q, k, stride, n, nq, nkv, hd, halves, pos, eps};
    if (const char *why = rows_bad(a, true)) return l3m_dev_fail(why);
    if ((long long)n * (nq + nkv) > MAX_ITEMS) return l3m_dev_fail("qk_norm_rope: too many rows for one call");
    launch_rows_in<-1>(a, l3m_kv4{}, as_stream(stream));
    return l3m_dev_launched("k_qk_norm_rope");
}

int l3m_k_kv4_append(const l3m_kv4 *c, float *q, const float *rows, int stride, int n, int nq, const float *wq, const float *wk, float eps,
                     int halves, int pos, const float *table, void *stream) {
    if (const char *why = kv4_bad(c)) return l3m_dev_fail(why);
    if (!span_ok(c, pos, n)) return l3m_dev_fail("kv4_append: positions past the cache's end");
    const RowsIn a = {rows, wq, wk, table, q, nullptr, stride, n, nq, c->nkv, c->hd, halves, pos, eps};
    if (const char *why = rows_bad(a, false)) return l3m_dev_fail(why);
    if ((long long)n * (nq + 2 * c->nkv) > MAX_ITEMS) return l3m_dev_fail("kv4_append: too many rows for one call");
    if (c->dtype == L3M_Q4_0) launch_rows_in<L3M_Q4_0>(a, *c, as_stream(stream));
    else launch_rows_in<L3M_MXFP4>(a, *c, as_stream(stream));
    return l3m_dev_launched("k_kv4_append");
}

int l3m_k_kv4_rows(const l3m_kv4 *c, float *k, float *v, int pos, int n, void *stream) {
    if (const char *why = kv4_bad(c)) return l3m_dev_fail(why);
    if (!span_ok(c, pos, n)) return l3m_dev_fail("kv4_rows: positions past the cache's end");
    if ((!k && !v) || ((uintptr_t)k | (uintptr_t)v) % 4) return l3m_dev_fail("kv4_rows: no output, or one that is not 4-byte aligned");
    const size_t vals = (size_t)n * c->nkv * c->hd;
    if (vals > (size_t)MAX_ITEMS * 64) return l3m_dev_fail("kv4_rows: too many rows for one call");
    const dim3 grid((unsigned)((vals + 255) / 256));
    if (c->dtype == L3M_Q4_0) hipLaunchKernelGGL(k_kv4_rows<L3M_Q4_0>, grid, dim3(256), 0, as_stream(stream), *c, k, v, pos, n);
    else hipLaunchKernelGGL(k_kv4_rows<L3M_MXFP4>, grid, dim3(256), 0, as_stream(stream), *c, k, v, pos, n);
    return l3m_dev_launched("k_kv4_rows");
}

size_t l3m_kv4_work_bytes(const l3m_kv4 *c, int n, int nq) {
    if (kv4_bad(c) || n < 1 || n > c->cap || nq < 1 || nq % c->nkv) return 0;
    return 256;
}

int l3m_k_kv4_attend(float *out, const float *q, const l3m_kv4 *c, int n, int nq, int pos, void *work, size_t work_bytes, void *stream) {
    if (const char *why = kv4_bad(c)) return l3m_dev_fail(why);
    if (!span_ok(c, pos, n)) return l3m_dev_fail("kv4_attend: positions past the cache's end");
    if (nq < 1 || nq > 65536 || nq % c->nkv) return l3m_dev_fail("kv4_attend: query heads must be a multiple of the kv heads");
    const size_t rows = (size_t)n * nq, bytes = 4 * rows * c->hd;
    if (!out || !q || ((uintptr_t)out | (uintptr_t)q) % 4 || (out != q && overlap(out, bytes, q, bytes)))
        return l3m_dev_fail("kv4_attend: q and out must be floats, the same or apart");
    if (!work || (uintptr_t)work % 16 || work_bytes < l3m_kv4_work_bytes(c, n, nq)) return l3m_dev_fail("kv4_attend: the workspace is too small (l3m_kv4_work_bytes)");
    if (rows > (size_t)MAX_ITEMS) return l3m_dev_fail("kv4_attend: too many rows for one call");
    if (c->dtype == L3M_Q4_0) hipLaunchKernelGGL(k_kv4_attend<L3M_Q4_0>, dim3((unsigned)rows), dim3(64), 0, as_stream(stream), out, q, *c, nq, pos);
    else hipLaunchKernelGGL(k_kv4_attend<L3M_MXFP4>, dim3((unsigned)rows), dim3(64), 0, as_stream(stream), out, q, *c, nq, pos);
    return l3m_dev_launched("k_kv4_attend");
}

}
