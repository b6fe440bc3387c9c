// A paged K/V cache of 8-bit codes for CDNA4 (gfx950): the writer, the read-back, and the attention of a batch's last tokens over it.
//
// Layout. A page's unit of a layer and kv head: K codes [128 positions][HP] and V codes [HP][128 positions], HP hd rounded up to 32 (zeros), so that a lane's
// 16 bytes of either are columns of the matrix cores' operands as they lie. A block of 32 positions has one scale of a kv head's K and one of its V, a power
// of two, which the conversion of the codes takes.
#include <type_traits>
#include "serve.h"

namespace {

constexpr int TILE = 64;                                             // positions that a wavefront takes at once
constexpr int E4M3_NAN = 0x7F;
constexpr float M0 = -3.40282347e38f;                                // the maximum of no score: float32's lowest

typedef float f32x2 __attribute__((ext_vector_type(2)));

// ---------------------------------------------------------------- writer

// The exponent byte of a block by its largest finite magnitude: the smallest power of two, 2^-126 at least, by which it is at most 448 = 1.75 2^8.
__device__ __forceinline__ int exponent_for(float most) {
    const uint32_t u = __float_as_uint(most);
    return max((int)(u >> 23) - 8 + ((u & 0x7FFFFFu) > 0x600000u), 1);
}
// Sizes as whole numbers: of finite values in order, from FINITE up; of others, as the sum wraps, less.
constexpr uint32_t FINITE = 0x01000000u;
__device__ __forceinline__ uint32_t size_of(float x) { return (__float_as_uint(x) << 1) + FINITE; }
__device__ __forceinline__ float value_of(uint32_t size) { return size < FINITE ? 0.f : __uint_as_float((size - FINITE) >> 1); }
// Four values times 2^(127 - exponent) as codes, to the nearest, ties to even; what is not finite (FINITE_ONLY: there is none) is NaN.
template <bool FINITE_ONLY> __device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, float up) {
    uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a * up, b * up, 0, false);
    w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c * up, d * up, (int)w, true);
    if constexpr (FINITE_ONLY) return w;
    const float x[4] = {a, b, c, d};
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (!(fabsf(x[i]) < INFINITY)) w = (w & ~(255u << 8 * i)) | (uint32_t)E4M3_NAN << 8 * i;
    return w;
}
// Four codes times `by`, as codes.
__device__ __forceinline__ uint32_t recode4(uint32_t w, float by) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return encode4<false>(a.x, a.y, b.x, b.y, by);
}
__device__ __forceinline__ float pow2_byte(int e) { return __uint_as_float((uint32_t)e << 23); }   // 2^(e - 127), e 1 .. 254

// Bytes i of four words as word i.
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    w[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
    w[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    w[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
    w[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// Eight values as they lie in memory.
template <class T> struct Raw8 {
    u32x4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T *p) {
        typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
        typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
        typedef std::conditional_t<sizeof(T) == 4, u32x4_a4, u32x4_a2> u32x4_at;
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) w[i] = *(const u32x4_at *)(p + 16 / sizeof(T) * i);
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) w[i] = u32x4{0, 0, 0, 0};
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i >> 2][i & 3]);
        else return __uint_as_float(i & 1 ? w[0][i >> 1] & 0xFFFF0000u : w[0][i >> 1] << 16);
    }
};

struct RowsIn {
    l3m_kv8    c;
    Runs       b;
    const void *k, *v;                                               // rows in
    float      *ok, *ov;                                             // rows out (read-back)
    long long  stride;
    const int32_t *table, *len, *state;
    int        layer, pages, seqs, width, per;                       // per: workgroups of a block of positions
    uint32_t   per_mul;
};
// The blocks of 32 positions that a run's rows, the last ones of its sequence, lie in.
__device__ __forceinline__ int length_of(const RowsIn &a, int id) { return (unsigned)id < (unsigned)a.seqs ? clamp(a.len[id], 0, a.width * PAGE) : 0; }
__device__ __forceinline__ int blocks_of(const RowsIn &a, int run, int rows) {
    const int len = length_of(a, a.b.id(run)), first = len - rows;
    return rows && first >= 0 ? (len - 1) / BLOCK - first / BLOCK + 1 : 0;
}

// The new rows of a block of 32 positions of one kv head, K or V: a wavefront each. Their largest magnitude and the scale of what the block holds already make the
// block's scale; where that rises, the old codes are rounded again. Bound by latency for single rows (48 sequences, 8 heads of 128: 5.0 us, of which a launch is 1.6:
// lengths, page, scale, codes, each behind the last), by bytes for prompts.
template <class T, int NB> __global__ void __launch_bounds__(256) k_kv8_append(RowsIn a) {
    constexpr int HP = 32 * NB, PER = 4 * NB, IT = 2 * NB;           // eight values a lane: chunks of a row, turns for 32 rows
    __shared__ __align__(16) uint8_t code_s[4][BLOCK * (HP + 4)];
    const int failed = a.state[0];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nkv = a.c.nkv;
    const int item = (int)divide(blockIdx.x, a.per, a.per_mul), which = 4 * ((int)blockIdx.x - item * a.per) + wave, h = which >> 1;
    const bool value = which & 1;
    const Found f = find_run<4>(a.b, item, [&](int r, int, int rows) { return blocks_of(a, r, rows); });
    if (f.run < 0 || h >= nkv) return;
    const int id = a.b.id(f.run), len = length_of(a, id), first = len - f.rows, block = first / BLOCK + f.at;
    const int page = a.table[(size_t)id * a.width + block / SCALES];
    const int sub = block % SCALES, p0 = block * BLOCK, before = max(first - p0, 0), end = min(len - p0, BLOCK);
    const T *rows = (const T *)(value ? a.v : a.k) + (size_t)h * a.c.hd;
    // turn i: rows 64 i / PER .. (64 i + 63) / PER of the block; a row to a turn is the rule of steps, so turns without new rows are left out as a whole
    auto has = [&](int i) { return 64 * i / PER < end && (64 * i + 63) / PER >= before; };
    Raw8<T> x[IT];
#pragma unroll
    for (int i = 0; i < IT; i++) {
        const int at = 64 * i + lane, r = at / PER, d = 8 * (at - r * PER);
        if (has(i)) x[i].load(rows + (long long)(f.s0 + p0 + clamp(r, before, end - 1) - first) * a.stride + (d < a.c.hd ? d : 0));
    }
    if (failed || (unsigned)page >= (unsigned)a.pages) return;       // behind a failed call on the tables nothing is written
    const Unit u = unit_of(a.c, page, a.layer, h);
    uint8_t *scale = u.s + (value ? SCALES : 0) + sub;
    // V's words, four positions 4 q .. of a dimension: a lane's are of one q and the dimensions 4 (8 i + lane / 8) .. + 3. Those that hold earlier positions
    // beside new ones:
    const int q = lane & 7, dq = lane >> 3;
    uint32_t *const words = (uint32_t *)(u.v + (size_t)(4 * dq) * PAGE + sub * BLOCK) + q, shared[NB][4] = {};
    auto read_shared = [&] {
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) shared[i][j] = words[(32 * i + j) * (PAGE / 4)];
    };
    if (value && before % 4 && q == before >> 2) read_shared();
    const int had = before ? max((int)*scale, 1) : 0;
    uint32_t most = 0, least = ~0u;
#pragma unroll
    for (int i = 0; i < IT; i++) {
        const int at = 64 * i + lane, r = at / PER, d = 8 * (at - r * PER);
        if (!has(i)) continue;
        if (d >= a.c.hd) x[i].clear();                               // the head's end; rows beside the new ones are the first or last again
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t size = size_of(x[i].value(j));
            most = max(most, size);
            least = min(least, size);
        }
    }
    const bool finite = !__ballot(least < FINITE);
    const int e = max(exponent_for(max_wave(value_of(most))), had);
    const float up = pow2_byte(254 - e), down = had && had < e ? (e - had < 127 ? pow2_byte(127 - (e - had)) : 0.f) : 1.f;
    if (lane == 0) *scale = (uint8_t)e;                              // read by no other lane by now
    auto encode = [&](const Raw8<T> &x) {
        auto four = [&](int i) {
            return finite ? encode4<true>(x.value(i), x.value(i + 1), x.value(i + 2), x.value(i + 3), up)
                          : encode4<false>(x.value(i), x.value(i + 1), x.value(i + 2), x.value(i + 3), up);
        };
        return u32x2{four(0), four(4)};
    };
    if (!value) {
#pragma unroll
        for (int i = 0; i < IT; i++) {
            const int at = 64 * i + lane, r = at / PER, d = 8 * (at - r * PER);
            u32x2 *to = (u32x2 *)(u.k + (size_t)(sub * BLOCK + r) * HP + d);
            if (has(i) && r >= before && r < end) *to = encode(x[i]);
            else if (r < before && down != 1.f) {
                const u32x2 was = *to;
                *to = u32x2{recode4(was.x, down), recode4(was.y, down)};
            }
        }
    } else {
        // codes through LDS to words along positions
        uint8_t *row_s = code_s[wave];
#pragma unroll
        for (int i = 0; i < IT; i++) {
            const int at = 64 * i + lane, r = at / PER, d = 8 * (at - r * PER);
            uint32_t *to = (uint32_t *)(row_s + r * (HP + 4) + d);
            if (!has(i) || r < before || r >= end) continue;
            const u32x2 w = encode(x[i]);
            to[0] = w.x;
            to[1] = w.y;
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (4 * q >= end || (4 * q + 4 <= before && down == 1.f)) return;
        if (down != 1.f && 4 * q < before) {
            if (4 * q + 4 <= before) read_shared();
#pragma unroll
            for (int i = 0; i < NB; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) shared[i][j] = recode4(shared[i][j], down);
        }
        const uint32_t keep = before <= 4 * q ? 0u : before - 4 * q >= 4 ? ~0u : ~(~0u << 8 * (before - 4 * q));    // positions that were there
        const uint32_t gone = 4 * q + 4 > end ? ~0u << 8 * (end - 4 * q) : 0u;                                      // behind the sequence: zeros
#pragma unroll
        for (int i = 0; i < NB; i++) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; j++) w[j] = *(const uint32_t *)(row_s + (4 * q + j) * (HP + 4) + 32 * i + 4 * dq);
            transpose4(w);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                words[(32 * i + j) * (PAGE / 4)] = (shared[i][j] & keep) | (w[j] & ~keep & ~gone);
            }
        }
    }
}

// ---------------------------------------------------------------- read-back
// A block of 32 positions of one kv head, K or V, to a wavefront: float32 rows of the run's last positions. Bound by what it writes; 4 x 2000 rows of 8 heads of
// 128 stored and read back, 131 MB: 36.3 us, 3.6 TB/s for the two.
template <int NB> __global__ void __launch_bounds__(256) k_kv8_rows(RowsIn a) {
    constexpr int HP = 32 * NB;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nkv = a.c.nkv, hd = a.c.hd;
    const int item = (int)divide(blockIdx.x, a.per, a.per_mul), which = 4 * ((int)blockIdx.x - item * a.per) + wave, h = which >> 1;
    const bool value = which & 1;
    float *out = value ? a.ov : a.ok;
    const Found f = find_run<4>(a.b, item, [&](int r, int, int rows) { return blocks_of(a, r, rows); });
    if (f.run < 0 || h >= nkv || !out) return;
    const int id = a.b.id(f.run), len = length_of(a, id), first = len - f.rows, block = first / BLOCK + f.at;
    const int page = a.table[(size_t)id * a.width + block / SCALES];
    const bool lost = (unsigned)page >= (unsigned)a.pages;
    const Unit u = unit_of(a.c, lost ? 0 : page, a.layer, h);
    const int sub = block % SCALES, p0 = block * BLOCK, begin = max(first - p0, 0), end = min(len - p0, BLOCK);
    const float s = lost ? NAN : pow2_byte(max((int)u.s[(value ? SCALES : 0) + sub], 1));
    float *to = out + ((size_t)(f.s0 + p0 - first) * nkv + h) * hd;
    if (!value) {
        constexpr int PER = 4 * NB, IT = 2 * NB;
        u32x2 code[IT];
#pragma unroll
        for (int i = 0; i < IT; i++) code[i] = *(const u32x2 *)(u.k + (size_t)sub * BLOCK * HP + 8 * (64 * i + lane));
#pragma unroll
        for (int i = 0; i < IT; i++) {
            const int at = 64 * i + lane, r = at / PER, d = 8 * (at - r * PER);
            if (r < begin || r >= end || d >= hd) continue;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const f32x2 x = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[i][j], false), y = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[i][j], true);
                *(f32x4_a4 *)(to + (size_t)r * nkv * hd + d + 4 * j) = f32x4{x.x * s, x.y * s, y.x * s, y.y * s};
            }
        }
        return;
    }
    const int q = lane & 7, dq = lane >> 3;                          // four positions of four dimensions, as the writer has them
    uint32_t code[NB][4];
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) code[i][j] = *(const uint32_t *)(u.v + (size_t)(32 * i + 4 * dq + j) * PAGE + sub * BLOCK + 4 * q);
#pragma unroll
    for (int i = 0; i < NB; i++) {
        transpose4(code[i]);
        const int d = 32 * i + 4 * dq;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int r = 4 * q + j;
            if (r < begin || r >= end || d >= hd) continue;
            const f32x2 x = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[i][j], false), y = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[i][j], true);
            *(f32x4_a4 *)(to + (size_t)r * nkv * hd + d) = f32x4{x.x * s, x.y * s, y.x * s, y.y * s};
        }
    }
}

// ---------------------------------------------------------------- attention
// Rows: a kv head's (token, query head) pairs of a run, a token's heads side by side (g = nq / nkv), 16 to a product. Per tile, half a page, and wavefront,
// codes converted to bf16 as they are used, exactly, their scale with them (v_cvt_scalef32_pk_bf16_fp8):
//   S = K Q^T        16 positions x 16 rows x 32 dimensions (v_mfma_f32_16x16x32_bf16), q in PARTS of bf16
//   P = 2^(S - m)    m the running maximum
//   O^T += V^T P^T   16 dimensions x 16 rows x 32 positions, P in PARTS of bf16
// A lane of group c reads 16 bytes at once, which are two products' eight columns: the dimensions 64 f + 16 c .. of K and of q, the positions 16 c .. of V.
// K's rows are taken in the order in which a lane then holds the scores of those positions, so no value crosses lanes. All sums in 32 bits; q and P in
// three parts are float32's 24 bits; for bf16 rows q is one part, exactly, and P two, 2^-16 of a weight at the most.
// (v_mfma_scale_f32_16x16x128_f8f6f4 takes the codes as they lie, but aligns a product's 128 terms to the largest one: sums were off by 2^-11 of that.)
//
// Long caches are bound by their bytes: a wavefront has a tile of K and one of V under way, 16 KiB at hd 128, while it uses the last ones; two workgroups
// of four fill LDS. One token over 131071 positions of 8 kv heads of 128 (269 MB), 32 heads: 58.4 us, of which the products' launch is 50 (5.3 TB/s; a copy
// reaches 5.2) and the join 5; float32 queries, three products for one: 59.6. 64 sequences of 2243: 60.4 us; of 100 to 8000: 75 (3.9 TB/s), as the last
// workgroups don't fill the card. Short ones are bound by their instructions one after the other, some 900 a wavefront: 100 positions 6.2 us, 600 8.4.
// Measured and not built: shares by descending size (the listing costs what it saves); a wavefront to a kv head, without the meeting in LDS (512 sequences
// of 281 85 us against 104, but 128 of 100 to 8000 220 against 123); rows' tiles read from memory as operands (64 lines a load: 1346 us for the 131071).
template <bool F32> struct Parts {
    static constexpr int q = F32 ? 3 : 1, p = F32 ? 3 : 2;
};

template <int M> __device__ __forceinline__ float other(float x, float &y) {                // lane ^ 16, lane ^ 32
    const uint32_t a = __float_as_uint(x);
    if constexpr (M == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
        y = __uint_as_float(r[1]);
        return __uint_as_float(r[0]);
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
        y = __uint_as_float(r[1]);
        return __uint_as_float(r[0]);
    }
}
__device__ __forceinline__ float max_groups(float x) {               // over the four lane groups
    float y;
    x = other<16>(x, y); x = fmaxf(x, y);
    x = other<32>(x, y); return fmaxf(x, y);
}
__device__ __forceinline__ float sum_groups(float x) {
    float y;
    x = other<16>(x, y); x += y;
    x = other<32>(x, y); return x + y;
}
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
// Eight codes times `scale`, a power of two.
__device__ __forceinline__ bf16x8 widen(u32x2 w, float scale) {
    u32x4 r;
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, scale, false));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, scale, true));
    r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, scale, false));
    r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, scale, true));
    return __builtin_bit_cast(bf16x8, r);
}
// Eight values as the sum of N bf16 ones each, the weights' nearest ones. TOWARDS_0: three of them are exactly float32's 24 bits, and the largest values stay finite.
template <int N, bool TOWARDS_0 = false> __device__ __forceinline__ void in_parts(const float (&v)[8], bf16x8 (&w)[N]) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = v[i];
#pragma unroll
    for (int p = 0; p < N; p++) {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            r[i] = TOWARDS_0 ? __builtin_amdgcn_perm(__float_as_uint(x[2 * i + 1]), __float_as_uint(x[2 * i]), 0x07060302u) : bf16_pair(x[2 * i], x[2 * i + 1]);
            if (p + 1 < N) {
                x[2 * i] -= __uint_as_float(r[i] << 16);
                x[2 * i + 1] -= __uint_as_float(r[i] & 0xFFFF0000u);
            }
        }
        w[p] = __builtin_bit_cast(bf16x8, r);
    }
}

// Splitting. Per kv head the runs' groups of 16 rows over all their tiles are the work; a group over more than `chunk` tiles is split over as many workgroups as
// have a chunk each, all nearly equal, and their parts are joined by a second launch. The lengths lie in device memory, so each workgroup counts the work and
// finds its share of it by itself (share_of), the same in both launches.
constexpr int SPLIT_ROWS = 1 << 14;
// Workgroups that the work is spread over. One token over 131071: 58.6 us (256: 57.1, 1024: 62.0), over 32768 22.2 (21.9, 28.2); 64 sequences of 100 to 8000 75.8
// (81.5, 72.6), 16 of 8000 57.4 (1024: 60.2). Of heads past 128 one workgroup fills a CU, so half as many where the shares themselves are few: 4 heads of 256,
// one token over 131071 59.4 us by 256 and 68.4 by 512, over 20000 22.8 and 28.5, 16 sequences of 4000 33.9 and 40.5; but 64 of 100 to 8000 82.3 and 77.9.
constexpr int TARGET = 512;
constexpr int WORK = 25;                                             // a batch's work is up to 2^WORK units, of 2^unit tiles each; 64 lanes' are a sum in 32 bits
struct AttendIn {
    l3m_kv8     c;
    Runs        b;
    const void *q;
    void       *out;
    long long   q_stride, out_stride;
    const int32_t *table, *len, *state;
    float      *ml, *parts;                                          // [slot][row] maximum and sum, output; a slot's rows: slot_rows
    int         pages, seqs, width, nq, g, target, least, unit, slot_rows; // target: workgroups of a kv head, 0: nothing is split; least: units of a part
    uint32_t    g_mul, nkv_mul;                                      // of g and of nkv (divide)
    uint8_t    *mem;                                                 // the layer's part of page 0
    size_t      page_bytes;
    float       scale;                                               // of the scores: base 2
};
__device__ __forceinline__ int length_of(const AttendIn &a, int id) { return (unsigned)id < (unsigned)a.seqs ? clamp(a.len[id], 0, a.width * PAGE) : 0; }
__device__ __forceinline__ int groups_of(int rows, int g) { return (int)(((unsigned)rows * (unsigned)g + 15) >> 4); }
__device__ __forceinline__ int tiles_of(int len) { return (len + TILE - 1) / TILE; }

// A workgroup's share: of run `run`, id its sequence, of len positions, rows s0 ..; row group `group`, part `part` of `parts`, whose first one's slot is `slot`.
struct Share {
    int run, id, len, s0, rows, group, part, parts, slot, page;     // page: of the wavefront's first tile, where nothing is split; else to be read
};
// The item-th share of a kv head's work, or (GROUP) the first share of the item-th group of rows. run < 0: none. Up to 64 runs are counted by each wavefront for
// itself, a lane a run; more by the workgroup's W wavefronts, 64 each, which meet in LDS.
template <bool GROUP, int W> __device__ __forceinline__ Share share_of(const AttendIn &a, int item) {
    __shared__ uint32_t work_s[W];
    __shared__ int      sums_s[2][2][W];
    __shared__ Share    found_s;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool alone = a.b.seqs <= 64, once = a.b.seqs <= 64 * W;
    const int mine0 = alone ? 0 : 64 * wave;
    int id, len, s0, rows, page = 0, chunk = 1 << 30;
    const int column = min(wave * TILE / PAGE, a.width - 1);
    const bool early = !GROUP && alone && !a.target;                // the first pages' numbers come with the lengths
    auto read = [&](int r) {
        id = len = s0 = rows = 0;
        if (r < a.b.seqs) {
            id = a.b.id(r);
            s0 = a.b.from(r);
            rows = a.b.to(r, s0) - s0;
            len = length_of(a, id);
            id = (unsigned)id < (unsigned)a.seqs ? id : 0;           // none: no position of any
            if (early) page = a.table[(size_t)id * a.width + column];
        }
    };
    read(mine0 + lane);
    if (a.target) {
        uint32_t work = 0;
        for (int r0 = 0;; r0 += 64 * W) {
            if (r0) read(r0 + mine0 + lane);
            const unsigned units = (unsigned)(tiles_of(len) + (1 << a.unit) - 1) >> a.unit;
            work += (uint32_t)__builtin_amdgcn_readlane(scan_wave((int)min((unsigned long long)groups_of(rows, a.g) * units, (1ull << WORK) + 1)), 63);
            work = min(work, 2u << WORK);
            if (r0 + 64 * W >= a.b.seqs) break;
        }
        if (!alone) {
            if (lane == 0) work_s[wave] = work;
            __syncthreads();
            work = 0;
#pragma unroll
            for (int w = 0; w < W; w++) work = min(work + work_s[w], 2u << WORK);
        }
        // more than that have only runs that overlap: nothing is split, or the parts would be more than the workspace's
        if (work && work <= 1u << WORK) chunk = (int)min((unsigned long long)max((unsigned)a.least, (work - 1) / (unsigned)a.target + 1) << a.unit, 1ull << 30);
    }
    int base = 0, slots = 0;
    for (int r0 = 0, turn = 0; r0 < a.b.seqs; r0 += 64 * W, turn ^= 1) {
        if (!once && (r0 || a.target)) read(r0 + mine0 + lane);
        const int groups = groups_of(rows, a.g), parts = a.target ? max((int)((unsigned)(tiles_of(len) + chunk - 1) / (unsigned)chunk), 1) : 1, split = parts > 1 ? groups * parts : 0;
        const int c = GROUP ? groups : groups * parts;
        int upto = scan_wave(c), slot = scan_wave(split), all = __builtin_amdgcn_readlane(upto, 63), all_slots = __builtin_amdgcn_readlane(slot, 63);
        if (!alone) {
            if (lane == 0) {
                sums_s[turn][0][wave] = min(all, MOST_ITEMS);
                sums_s[turn][1][wave] = all_slots;
            }
            __syncthreads();
            upto += base;
            slot += slots;
            all = base;
            all_slots = slots;
#pragma unroll
            for (int w = 0; w < W; w++) {
                const int x = sums_s[turn][0][w], y = sums_s[turn][1][w];
                upto += w < wave ? x : 0;
                slot += w < wave ? y : 0;
                all += x;
                all_slots += y;
            }
        }
        if (all > item) {
            const uint64_t here = __ballot(upto > item && upto - c <= item);
            Share f = {r0, 0, 0, 0, 0, 0, 0, 1, 0, 0};
            if (here) {
                const int l = __builtin_ctzll(here);
                auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
                const int n = of(parts), at = item - of(upto - c), group = GROUP || n == 1 ? at : (int)((unsigned)at / (unsigned)n);
                f = {r0 + mine0 + l, of(id), of(len), of(s0), of(rows), group, GROUP ? 0 : at - group * n, n, of(slot - split) + group * n, of(page)};
            }
            if (alone) return f;
            if (here && lane == 0) found_s = f;
            __syncthreads();
            auto same = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
            return {same(found_s.run), same(found_s.id), same(found_s.len), same(found_s.s0), same(found_s.rows), same(found_s.group), same(found_s.part), same(found_s.parts), same(found_s.slot), 0};
        }
        base = all;
        slots = all_slots;
    }
    return {-1, 0, 0, 0, 0, 0, 0, 1, 0, 0};
}

// Products' columns over a row's dimensions: step s holds a lane's dimensions dim_of(s, c) .. + 7.
template <int NB> __device__ __forceinline__ int dim_of(int s, int c) { return s / 2 * 2 + 1 < NB ? 64 * (s >> 1) + 16 * c + 8 * (s & 1) : 32 * s + 8 * c; }
template <bool F32, int NB> struct Queries {
    static constexpr int QP = Parts<F32>::q;
    bf16x8 part[NB][QP];
    __device__ __forceinline__ void load(const void *q, long long at, int hd, int lane) {
#pragma unroll
        for (int s = 0; s < NB; s++) {
            const int d = dim_of<NB>(s, lane >> 4);
            const bool in = d < hd;
            if constexpr (F32) {
                Raw8<float> raw;
                raw.load((const float *)q + at + (in ? d : 0));
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = in ? raw.value(i) : 0.f;
                in_parts<QP, true>(x, part[s]);
            } else {
                typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
                u32x4 x = *(const u32x4_a2 *)((const uint16_t *)q + at + (in ? d : 0));
                if (!in) x = u32x4{0, 0, 0, 0};
                part[s][0] = __builtin_bit_cast(bf16x8, x);
            }
        }
    }
    __device__ __forceinline__ void arrived() {
#pragma unroll
        for (int s = 0; s < NB; s++)
#pragma unroll
            for (int p = 0; p < QP; p++) asm volatile("" : "+v"(part[s][p]));
    }
};
// The scores' products of a tile, t of them, element i of lane group c: position 16 c + 4 t + i. So row m of the operand is
__device__ __forceinline__ int position_of(int t, int m) { return 16 * (m >> 2) + 4 * t + (m & 3); }
#define LOCAL __attribute__((address_space(3)))
#define GLOBAL __attribute__((address_space(1)))
#define CONSTANT __attribute__((address_space(4)))
// A wavefront's tile in LDS, 64 rows of K (positions) of 32 NB bytes and 32 NB rows of V (dimensions) of 64, in pieces of 16 bytes, which memory gives in order: 64
// lanes a KiB, where rows read as an operand takes them would be 64 lines. A row's pieces lie in an order of its own, by which a read of 16 rows
// meets no bank more often than it must.
template <int NB> __device__ __forceinline__ int k_turn(int row) {
    return NB % 4 == 0 ? (row & 3) | (row >> 2 & 4) : NB % 2 == 0 ? (row >> 1 & 1) | (row >> 3 & 2) : row >> 2 & 1;
}
__device__ __forceinline__ int v_turn(int row) { return row >> 1 & 3; }
template <int NB> __device__ __forceinline__ void request_k(const uint8_t *k, uint8_t *k_s, int lane) {
#pragma unroll
    for (int i = 0; i < 2 * NB; i++) {
        const int at = 64 * i + lane, row = at / (2 * NB), piece = (at - row * (2 * NB)) ^ k_turn<NB>(row);
        __builtin_amdgcn_global_load_lds((const GLOBAL void *)(k + row * (32 * NB) + 16 * piece), (LOCAL void *)(k_s + 1024 * i), 16, 0, 0);
    }
}
template <int NB> __device__ __forceinline__ void request_v(const uint8_t *v, uint8_t *v_s, int lane) {
#pragma unroll
    for (int i = 0; i < 2 * NB; i++) {
        const int row = 16 * i + (lane >> 2), piece = (lane & 3) ^ v_turn(row);
        __builtin_amdgcn_global_load_lds((const GLOBAL void *)(v + row * PAGE + 16 * piece), (LOCAL void *)(v_s + 1024 * i), 16, 0, 0);
    }
}
// All but the last N requests are done; all reads of LDS are.
template <int N> __device__ __forceinline__ void requests_but() { __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | (N >> 4) << 14); }
__device__ __forceinline__ void reads_done() { __builtin_amdgcn_s_waitcnt(0xC07F); }

// Four values of a result. NaN behind a failed call on the tables; a token before its sequence's first position sees nothing: zeros.
template <bool F32> __device__ __forceinline__ void put_row(const AttendIn &a, long long at, f32x4 x, bool none, bool failed) {
    if (none) x = f32x4{0.f, 0.f, 0.f, 0.f};
    if (failed) x = f32x4{NAN, NAN, NAN, NAN};
    if constexpr (F32) *(f32x4_a4 *)((float *)a.out + at) = x;
    else {
        typedef uint32_t u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));
        *(u32x2_a2 *)((uint16_t *)a.out + at) = u32x2{bf16_pair(x.x, x.y), bf16_pair(x.z, x.w)};
    }
}
// 32-bit words of bytes: those before position `end` of them that begin at `from`.
__device__ __forceinline__ uint32_t bytes_before(int from, int end) {
    const int n = end - from;
    return n >= 4 ? ~0u : n <= 0 ? 0u : ~(~0u << 8 * n);
}

template <bool F32, int NB, int WAVES> __global__ void __launch_bounds__(64 * WAVES) k_kv8_attend(AttendIn a) {
    constexpr int QP = Parts<F32>::q, PP = Parts<F32>::p, HP = 32 * NB, OS = HP + 4, REQUESTS = 2 * NB;
    __shared__ __align__(16) uint8_t tile_s[WAVES][2][TILE * HP];    // K's and V's
    __shared__ float m_s[WAVES][16], l_s[WAVES][16];
    static_assert(sizeof(tile_s) >= WAVES * 16 * OS * 4, "");
    float (*o_s)[16][OS] = (float (*)[16][OS])tile_s;                // behind the tiles
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, c = lane >> 4, hd = a.c.hd, g = a.g;
    // kv heads fastest: consecutive workgroups go to different XCDs, so 8 heads keep to an L2 each
    const int item = (int)divide(blockIdx.x, a.c.nkv, a.nkv_mul), h = (int)blockIdx.x - item * a.c.nkv;
    const bool failed = *(const CONSTANT int32_t *)a.state != 0;
    const Share f = share_of<false, WAVES>(a, item);
    if (f.run < 0) return;
    const int len = f.len, row0 = 16 * f.group, rows = min(f.rows * g - row0, 16);
    // the row of this lane's column: its token, and the positions it sees
    const int r = row0 + min(r16, rows - 1), token = (int)divide(r, g, a.g_mul), head = h * g + r - token * g, seen = max(len - f.rows + token + 1, 0);
    const int last = (int)divide(row0 + rows - 1, g, a.g_mul), end = max(len - f.rows + last + 1, 0);
    const bool several = last != (int)divide(row0, g, a.g_mul);      // tokens: rows that see different numbers of positions
    const int whole = max(len - f.rows + (int)divide(row0, g, a.g_mul) + 1, 0) / TILE;     // tiles that every row sees whole
    // this part's tiles (of all the sequence's; the last ones may lie behind every row)
    int t0 = 0, t1 = tiles_of(end);
    if (f.parts > 1) {
        const int all = tiles_of(len), share = all / f.parts, more = all - share * f.parts;
        t0 = f.part * share + min(f.part, more);
        t1 = min(t0 + share + (f.part < more), t1);
    }
    const CONSTANT int32_t *table = (const CONSTANT int32_t *)(a.table + (size_t)f.id * a.width);
    // the pages' numbers come a turn ahead of their use
    auto page_of = [&](int t) { return table[min(t, max(t1 - 1, 0)) * TILE / PAGE]; };
    struct Tile {                                                    // where a tile's K and V begin, its two blocks' exponents
        const uint8_t *k, *v;
        const CONSTANT uint32_t *s;
        int half;
        bool lost;
    };
    auto tile_at = [&](int t, int page) {
        const int half = min(t, max(t1 - 1, 0)) & 1;
        const bool lost = (unsigned)page >= (unsigned)a.pages;
        const uint8_t *at = a.mem + (lost ? 0 : page) * a.page_bytes, *k = at + h * (2 * PAGE * HP);
        return Tile{k + half * TILE * HP, k + PAGE * HP + half * TILE, (const CONSTANT uint32_t *)(at + a.c.nkv * (2 * PAGE * HP) + 2 * SCALES * h), half, lost};
    };
    int tile = t0 + wave;
    Queries<F32, NB> qs;
    qs.load(a.q, (long long)(f.s0 + token) * a.q_stride + (long long)head * hd, hd, lane);
    Tile u = tile_at(tile, !a.target && a.b.seqs <= 64 && tile < t1 ? f.page : page_of(tile));
    int page = page_of(tile + WAVES);
    uint32_t ks = u.s[0], vs = u.s[1];
    uint8_t *my_k = tile_s[wave][0], *my_v = tile_s[wave][1];
    request_k<NB>(u.k, my_k, lane);
    request_v<NB>(u.v, my_v, lane);
    qs.arrived();                                                    // here, or the loop waits for all requests at its top
    const float scale = a.scale;

    f32x4 acc[2 * NB];
#pragma unroll
    for (int t = 0; t < 2 * NB; t++) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = M0, l = 0.f;
    bool large = false;                                              // some row's m is (LARGE_SCORE)
    for (; tile < t1; tile += WAVES) {
        const bool lost = u.lost, masked = tile >= whole;
        const int left = end - tile * TILE;                          // positions that some row sees
        const float sk = pow2_byte((int)(ks >> (16 * u.half + 8 * (r16 >> 3)) & 255u));
        const float sv = !lost && 32 * (c >> 1) < left ? pow2_byte((int)(vs >> (16 * u.half + 8 * (c >> 1)) & 255u)) : 1.f;   // 1: never written
        requests_but<REQUESTS>();                                    // V's, which came behind K's
        f32x4 s[4];
#pragma unroll
        for (int t = 0; t < 4; t++) s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        // products onto different sums side by side: one waits for the last onto its own
#pragma unroll
        for (int i = 0; i < NB; i += 2) {
            u32x2 w[2][4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const int row = position_of(t, r16);
                const uint8_t *at = my_k + row * HP;
                if (i + 1 < NB) {
                    const u32x4 x = *(const u32x4 *)(at + 16 * ((2 * i + c) ^ k_turn<NB>(row)));
                    w[0][t] = u32x2{x.x, x.y};
                    w[1][t] = u32x2{x.z, x.w};
                } else w[0][t] = *(const u32x2 *)(at + 16 * ((2 * i + (c >> 1)) ^ k_turn<NB>(row)) + 8 * (c & 1));
            }
#pragma unroll
            for (int j = 0; j < 2; j++)
                if (i + j < NB) {
                    bf16x8 x[4];
#pragma unroll
                    for (int t = 0; t < 4; t++) x[t] = widen(w[j][t], sk);
#pragma unroll
                    for (int q = QP - 1; q >= 0; q--)
#pragma unroll
                        for (int t = 0; t < 4; t++) s[t] = mfma(x[t], qs.part[i + j < NB ? i + j : 0][q], s[t]);
                }
        }
        u = tile_at(tile + WAVES, page);
        reads_done();
        request_k<NB>(u.k, my_k, lane);
        __builtin_amdgcn_sched_barrier(0);                           // scalar loads are waited for with LDS's reads: not before them
        ks = u.s[0];
        vs = u.s[1];
        page = page_of(tile + 2 * WAVES);
        float p[16];
        const int p0 = tile * TILE + 16 * c;                         // of p[i]: p0 + i
#pragma unroll
        for (int i = 0; i < 16; i++) p[i] = s[i >> 2][i & 3];
        if (__builtin_expect(masked || lost, 0)) {
            asm volatile("");                                        // no selects for all tiles' sake
#pragma unroll
            for (int i = 0; i < 16; i++) p[i] = p0 + i >= seen ? -INFINITY : lost ? NAN : p[i];
        }
        float top = p[0];
#pragma unroll
        for (int i = 1; i < 16; i++) top = fmaxf(top, p[i]);
        top = fmaxf(max_groups(top) * scale, m);
        if (__ballot(top > m)) {
            const float by = __builtin_amdgcn_exp2f(m - top);
            l *= by;
#pragma unroll
            for (int t = 0; t < 2 * NB; t++) acc[t] *= by;
            m = top;
            large = __ballot(fabsf(m) > LARGE_SCORE && m != M0) != 0;
        }
        float by = scale, less = m;
        if (__builtin_expect(large, 0)) {
            asm volatile("");
#pragma unroll
            for (int i = 0; i < 16; i++) p[i] = scaled_less(p[i], scale, m);
            by = 1.f;
            less = 0.f;
        }
        bf16x8 w[2][PP];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[i] = __builtin_amdgcn_exp2f(fmaf(p[8 * t + i], by, -less));
                l += x[i];
            }
            in_parts<PP>(x, w[t]);
        }
        requests_but<REQUESTS>();                                    // the next K's, which came behind V's
        auto values = [&](int t) { return *(const u32x4 *)(my_v + (16 * t + r16) * TILE + 16 * (c ^ v_turn(16 * t + r16))); };
        // 32 dimensions' sums with their values at the positions before `upto` of the tile
        auto product = [&](int t, f32x4 &to0, f32x4 &to1, auto some, int upto) {
            const u32x4 v[2] = {values(t), values(t + 1)};
#pragma unroll
            for (int j = 0; j < 2; j++) {
                bf16x8 x[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    u32x2 z = {v[i][2 * j], v[i][2 * j + 1]};
                    if constexpr (decltype(some)::value) z = u32x2{z.x & bytes_before(16 * c + 8 * j, upto), z.y & bytes_before(16 * c + 8 * j + 4, upto)};
                    x[i] = widen(z, sv);
                }
#pragma unroll
                for (int q = PP - 1; q >= 0; q--) {
                    to0 = mfma(x[0], w[j][q], to0);
                    to1 = mfma(x[1], w[j][q], to1);
                }
            }
        };
        if (!masked) {
#pragma unroll
            for (int t = 0; t < 2 * NB; t += 2) product(t, acc[t], acc[t + 1], std::false_type{}, 0);
        } else {
            bool apart = false;                                      // a NaN is the rows' that see it: a token's rows at a time, over its own positions
            if (several) {
                // codes of NaN among the values that some row sees, and where the scale is 2^120 or more those from 256 on, which read as infinities
                const uint32_t up = sv >= 0x1p120f ? 0x08080808u : 0x01010101u;
                uint32_t nan = 0;
#pragma unroll
                for (int t = 0; t < 2 * NB; t++) {
                    const u32x4 v = values(t);
#pragma unroll
                    for (int i = 0; i < 4; i++) nan |= ((v[i] & bytes_before(16 * c + 4 * i, left) & 0x7F7F7F7Fu) + up) & 0x80808080u;
                }
                apart = __ballot(nan != 0) != 0;
            }
            for (int to = apart ? min(seen, end) : end, at = __builtin_amdgcn_readfirstlane(to);;) {
#pragma unroll
                for (int t = 0; t < 2 * NB; t += 2) {
                    f32x4 part[2] = {acc[t], acc[t + 1]};
                    product(t, part[0], part[1], std::true_type{}, at - tile * TILE);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        acc[t][i] = to == at ? part[0][i] : acc[t][i];
                        acc[t + 1][i] = to == at ? part[1][i] : acc[t + 1][i];
                    }
                }
                int next = INT_MAX;                                  // the next larger number of positions that a row sees
                for (uint64_t others = __ballot(to > at); others; others &= others - 1) next = min(next, __builtin_amdgcn_readlane(to, __builtin_ctzll(others)));
                if (next == INT_MAX) break;
                at = next;
            }
        }
        reads_done();
        request_v<NB>(u.v, my_v, lane);
    }
    requests_but<0>();

    // the wavefronts' parts meet in LDS
    l = sum_groups(l);
    if (c == 0) {
        m_s[wave][r16] = m;
        l_s[wave][r16] = l;
    }
    __syncthreads();                                                 // the tiles are done with
#pragma unroll
    for (int t = 0; t < 2 * NB; t++) *(f32x4 *)&o_s[wave][r16][16 * t + 4 * c] = acc[t];
    __syncthreads();
    for (int i = threadIdx.x; i < rows * (hd / 4); i += 64 * WAVES) {
        const int row = i / (hd / 4), d = 4 * (i - row * (hd / 4));
        float top = m_s[0][row], sum = 0.f;
#pragma unroll
        for (int w = 1; w < WAVES; w++) top = fmaxf(top, m_s[w][row]);
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const float by = __builtin_amdgcn_exp2f(m_s[w][row] - top);
            sum = fmaf(l_s[w][row], by, sum);
            x += *(const f32x4 *)&o_s[w][row][d] * by;
        }
        if (f.parts > 1) {
            const size_t to = ((size_t)(f.slot + f.part) * a.c.nkv + h) * a.slot_rows + row;
            *(f32x4 *)(a.parts + to * hd + d) = x;
            if (d == 0) *(f32x2 *)(a.ml + 2 * to) = f32x2{top, sum};
            continue;
        }
        const int t = (int)divide(row0 + row, g, a.g_mul), hh = h * g + row0 + row - t * g;
        put_row<F32>(a, (long long)(f.s0 + t) * a.out_stride + (long long)hh * hd + d, x * (1.f / sum), len - f.rows + t < 0, failed);
    }
}

// The parts of a group of rows that was split, of one kv head, to a workgroup: a wavefront a row makes the parts' factors, while the first parts come; threads of one part
// after the other meet in LDS in a fixed order. Bound by latency: 5 us for 66 parts of 4 rows of each of 8 kv heads.
constexpr int PARTS = TARGET + 1;                       // most parts of a group: a chunk each, of at most TARGET, and the last
template <bool F32, int JOIN> __global__ void __launch_bounds__(JOIN) k_kv8_join(AttendIn a) {
    __shared__ f32x4 o_s[JOIN];
    __shared__ float f_s[16][PARTS], sum_s[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hd = a.c.hd, quads = hd >> 2, block = (int)divide(blockIdx.x, a.c.nkv, a.nkv_mul), h = (int)blockIdx.x - block * a.c.nkv;
    const bool failed = *(const CONSTANT int32_t *)a.state != 0;
    const Share f = share_of<true, JOIN / 64>(a, block);
    if (f.run < 0 || f.parts < 2) return;
    const int rows = min(f.rows * a.g - 16 * f.group, 16);
    const size_t slot = ((size_t)f.slot * a.c.nkv + h) * a.slot_rows;                        // of the first part's first row
    const unsigned step = (unsigned)(a.c.nkv * a.slot_rows);                                 // to the next part's
    for (int r = wave; r < rows; r += JOIN / 64) {
        const f32x2 *ml = (const f32x2 *)a.ml + slot + r;
        float top = M0, sum = 0.f;
        for (int i = lane; i < f.parts; i += 64) top = fmaxf(top, ml[i * step].x);
        top = max_wave(top);
        for (int i = lane; i < f.parts; i += 64) {
            const f32x2 x = ml[i * step];
            const float by = __builtin_amdgcn_exp2f(x.x - top);
            f_s[r][i] = by;
            sum = fmaf(x.y, by, sum);
        }
#pragma unroll
        for (int i = 1; i < 64; i <<= 1) sum += __shfl_xor(sum, i);
        if (lane == 0) sum_s[r] = sum;
    }
    // threads by part, row and four dimensions; where the rows are more than the threads, in turns
    const int items = min(rows * quads, JOIN), groups = JOIN / items, mine = tid / items, item = tid - mine * items;
    for (int i0 = 0; i0 < rows * quads; i0 += items) {
        const int all = min(i0 + item, rows * quads - 1), row = all / quads, d = 4 * (all - row * quads);
        const float *from = a.parts + (slot + row) * hd + d;
        const unsigned apart = step * hd;
        f32x4 x[8], o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = *(const f32x4 *)(from + min(mine + i * groups, f.parts - 1) * apart);
        __syncthreads();                                             // the factors; the last turn's sums
        if (mine < groups)
            for (int p = mine; p < f.parts; p += 8 * groups) {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (p + i * groups < f.parts) o += x[i] * f_s[row][p + i * groups];
                if (p + 8 * groups < f.parts)
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] = *(const f32x4 *)(from + min(p + (8 + i) * groups, f.parts - 1) * apart);
            }
        if (groups > 1) {
            o_s[tid] = o;
            __syncthreads();
        }
        if (mine == 0 && i0 + item < rows * quads) {
            for (int i = 1; i < groups; i++) o += o_s[i * items + item];
            const int r = 16 * f.group + row, t = (int)divide(r, a.g, a.g_mul), hh = h * a.g + r - t * a.g;
            put_row<F32>(a, (long long)(f.s0 + t) * a.out_stride + (long long)hh * hd + d, o * (1.f / sum_s[row]), f.len - f.rows + t < 0, failed);
        }
    }
}

// What calls over the cache refuse alike, or NULL.
const char *call_bad(const l3m_kv8 *c, const l3m_pages *p, int layer, const l3m_batch *b) {
    if (const char *why = paged_bad(c, p)) return why;
    if (const char *why = batch_bad(b)) return why;
    if (layer < 0 || layer >= c->layers) return "kv8: no such layer";
    if (on_batch(b, c->mem, l3m_kv8_bytes(c->pages, c->layers, c->nkv, c->hd))) return "kv8: the batch overlaps the cache";
    return nullptr;
}
#define BY_BLOCKS(CALL)                                                                                                                                        \
    switch (padded(c->hd) / 32) {                                                                                                                              \
    case 1: CALL(1); break;                                                                                                                                    \
    case 2: CALL(2); break;                                                                                                                                    \
    case 3: CALL(3); break;                                                                                                                                    \
    case 4: CALL(4); break;                                                                                                                                    \
    case 5: CALL(5); break;                                                                                                                                    \
    case 6: CALL(6); break;                                                                                                                                    \
    case 7: CALL(7); break;                                                                                                                                    \
    default: CALL(8); break;                                                                                                                                   \
    }
// A split group has more than one chunk, so all of them have at most twice the chunks of the work.
int target_of(int nkv, int all) { return nkv < all ? all / nkv : 1; }
size_t slots(int nkv) { return 2 * (size_t)target_of(nkv, TARGET) * nkv; }
int slot_rows(int n, int g) { return (long long)n * g < 16 ? n * g : 16; }
// Blocks of 32 positions that a batch's rows can lie in: a run of r rows in (r + 62) / 32 of them.
long long most_blocks(const l3m_batch *b) { return b->n / BLOCK + 2ll * b->seqs; }

}  // namespace

extern "C" {

size_t l3m_kv8_page_bytes(int layers, int nkv, int hd) {
    if (layers < 1 || layers > 4096 || nkv < 1 || nkv > 4096 || hd < 8 || hd > 256 || hd % 8) return 0;
    return layers * layer_bytes(nkv, hd);
}
size_t l3m_kv8_bytes(int pages, int layers, int nkv, int hd) { return pages < 1 || pages > 1 << 20 ? 0 : pages * l3m_kv8_page_bytes(layers, nkv, hd); }

int l3m_kv8_init(l3m_kv8 *c, int pages, int layers, int nkv, int hd, void *mem) {
    if (!c || !mem || (uintptr_t)mem % 256) return l3m_dev_fail("kv8: memory must be 256-byte aligned");
    if (!l3m_kv8_bytes(pages, layers, nkv, hd)) return l3m_dev_fail("kv8: hd a multiple of 8 up to 256, pages up to 2^20, layers and kv heads up to 4096");
    *c = l3m_kv8{(uint8_t *)mem, pages, layers, nkv, hd};
    return 0;
}

int l3m_k_kv8_append(const l3m_kv8 *c, const l3m_pages *p, int layer, const void *k, const void *v, int stride, int dtype, const l3m_batch *b, void *stream) {
    if (const char *why = call_bad(c, p, layer, b)) return l3m_dev_fail(why);
    const size_t size = value_bytes(dtype);
    if (!size) return l3m_dev_fail("kv8_append: rows are f32 or bf16");
    const long long width = (long long)c->nkv * c->hd;
    if (stride < width) return l3m_dev_fail("kv8_append: a row holds fewer values than its heads");
    if (!b->seqs || !b->n) return 0;
    if (!k || !v || ((uintptr_t)k | (uintptr_t)v) % size) return l3m_dev_fail("kv8_append: no rows, or not aligned to their values");
    const size_t bytes = rows_bytes(b->n, stride, width, size);
    if (on_cache(c, k, bytes) || on_cache(c, v, bytes)) return l3m_dev_fail("kv8_append: the rows overlap the cache");
    const int per = (c->nkv + 1) / 2;
    const long long items = most_blocks(b) * per;
    if (items > 1ll << 28) return l3m_dev_fail("kv8_append: too many rows for one call");
    const RowsIn a = {*c, runs_of(b), k, v, nullptr, nullptr, stride, p->table, p->len, p->state, layer, p->pages, p->seqs, p->width, per, multiplier(per, items)};
    hipStream_t st;
    if (!stream_of(stream, st)) return -1;
    const dim3 grid((unsigned)items);
#define APPEND(NB)                                                                      \
    if (dtype == L3M_HIP_F32) hipLaunchKernelGGL((k_kv8_append<float, NB>), grid, dim3(256), 0, st, a); \
    else hipLaunchKernelGGL((k_kv8_append<uint16_t, NB>), grid, dim3(256), 0, st, a)
    BY_BLOCKS(APPEND)
    return l3m_dev_launched("k_kv8_append");
}

int l3m_k_kv8_rows(const l3m_kv8 *c, const l3m_pages *p, int layer, float *k, float *v, const l3m_batch *b, void *stream) {
    if (const char *why = call_bad(c, p, layer, b)) return l3m_dev_fail(why);
    if ((!k && !v) || ((uintptr_t)k | (uintptr_t)v) % 4) return l3m_dev_fail("kv8_rows: no output, or one that is not 4-byte aligned");
    if (!b->seqs || !b->n) return 0;
    const size_t bytes = 4 * (size_t)b->n * c->nkv * c->hd;
    if (overlap(k, bytes, v, bytes)) return l3m_dev_fail("kv8_rows: k overlaps v");
    if (on_cache(c, k, bytes) || on_cache(c, v, bytes) || on_pages(p, k, bytes) || on_pages(p, v, bytes) || on_batch(b, k, bytes) || on_batch(b, v, bytes))
        return l3m_dev_fail("kv8_rows: k or v overlaps the cache, the tables or the batch");
    const int per = (c->nkv + 1) / 2;
    const long long items = most_blocks(b) * per;
    if (items > 1ll << 28) return l3m_dev_fail("kv8_rows: too many rows for one call");
    const RowsIn a = {*c, runs_of(b), nullptr, nullptr, k, v, 0, p->table, p->len, p->state, layer, p->pages, p->seqs, p->width, per, multiplier(per, items)};
    hipStream_t st;
    if (!stream_of(stream, st)) return -1;
    const dim3 grid((unsigned)items);
#define ROWS(NB) hipLaunchKernelGGL((k_kv8_rows<NB>), grid, dim3(256), 0, st, a)
    BY_BLOCKS(ROWS)
    return l3m_dev_launched("k_kv8_rows");
}

size_t l3m_kv8_work_bytes(const l3m_kv8 *c, int n, int nq) {
    if (kv8_bad(c) || n < 1 || n > 1 << 28 || nq < 1 || nq > 65536 || nq % c->nkv) return 0;
    return 4 * slots(c->nkv) * slot_rows(n, nq / c->nkv) * (c->hd + 2) + 16;
}

int l3m_k_kv8_attend(void *out, int out_stride, const void *q, int q_stride, int dtype, const l3m_kv8 *c, const l3m_pages *p, int layer, const l3m_batch *b, int nq,
                     int longest, void *work, size_t work_bytes, void *stream) {
    if (const char *why = call_bad(c, p, layer, b)) return l3m_dev_fail(why);
    const size_t size = value_bytes(dtype);
    if (!size) return l3m_dev_fail("kv8_attend: queries and outputs are f32 or bf16");
    if (nq < 1 || nq > 65536 || nq % c->nkv) return l3m_dev_fail("kv8_attend: query heads must be a multiple of the kv heads");
    const long long width = (long long)nq * c->hd;
    if (q_stride < width || out_stride < width) return l3m_dev_fail("kv8_attend: a row holds fewer values than its heads");
    if (longest < 0) return l3m_dev_fail("kv8_attend: a negative length");
    if (!b->seqs || !b->n) return 0;
    if (!out || !q || ((uintptr_t)out | (uintptr_t)q) % size) return l3m_dev_fail("kv8_attend: no queries or output, or not aligned to their values");
    const size_t qb = rows_bytes(b->n, q_stride, width, size), ob = rows_bytes(b->n, out_stride, width, size), need = l3m_kv8_work_bytes(c, b->n, nq);
    if (!(out == q && out_stride == q_stride) && overlap(out, ob, q, qb)) return l3m_dev_fail("kv8_attend: q and out must be the same or apart");
    if (!work || (uintptr_t)work % 16 || work_bytes < need) return l3m_dev_fail("kv8_attend: the workspace is too small (l3m_kv8_work_bytes) or not 16-byte aligned");
    if (overlap(work, need, q, qb) || overlap(work, need, out, ob)) return l3m_dev_fail("kv8_attend: the workspace overlaps q or out");
    if (on_cache(c, out, ob) || on_cache(c, work, need) || on_pages(p, out, ob) || on_pages(p, work, need) || on_batch(b, out, ob) || on_batch(b, work, need))
        return l3m_dev_fail("kv8_attend: out or the workspace overlaps the cache, the tables or the batch");
    const int g = nq / c->nkv;
    if ((long long)b->n * g > 1 << 28) return l3m_dev_fail("kv8_attend: too many rows for one call");
    const long long groups = ((long long)b->n * g + 15) / 16 + b->seqs;
    if (groups * c->nkv > 1ll << 28) return l3m_dev_fail("kv8_attend: too many rows for one call");
    const long long most = longest ? longest : (long long)p->width * PAGE, shares = groups * c->nkv;
    // Eight wavefronts where there is work for them and a CU for each workgroup; two of four have the same tiles under way and the shorter meeting. 600 positions
    // of 8 kv heads: 8.4 us against 9.1, 100: 6.8 against 6.2, 32 times 300: 11.4 against 10.6.
    const int nb = padded(c->hd) / 32, waves = nb <= 4 && shares <= 256 && most > 4 * TILE ? 8 : 4;
    // Split where a workgroup's turns, 4 positions a ns, outlast the join, 4 to 5 us. 8 kv heads of 1024 positions: 11.5 us split, 9.8 not; 2048: 11.6 and 13.9;
    // 4001: 12.2 and 22.6. Where there are many shares, the join has more to read, and the turns' loads share the memory: 128 shares of 2000: 21.8 and
    // 18.0, of 4000: 31.9 and 36.0; 1024 of up to 1500: 47.9 and 41.3, 512 of up to 8000: 75.5 and 80.8. Heads past 128 have longer turns and
    // fill a CU by one workgroup: 4 of 256, one token over 500 12.9 and 10.8, over 1000 12.9 and 15.8; 64 shares of 2500 25.8 and 40.5; 256 of up to 2000 44.1 and
    // 36.0. Rows of many tokens fill the card by themselves.
    const bool wide = nb > 4;
    const int few = wide ? 256 : 64;
    const bool split = (long long)b->n * nq <= SPLIT_ROWS && most > (shares >= few ? 2560 : wide ? 768 : 1024);
    const int per = slot_rows(b->n, g), target = split ? target_of(c->nkv, wide && shares < few ? TARGET / 2 : TARGET) : 0;
    int unit = 0;
    while (groups * ((2ll * p->width + (1 << unit) - 1) >> unit) > 1 << WORK) unit++;
    float *ml = (float *)work;
    const AttendIn a = {*c, runs_of(b), q, out, q_stride, out_stride, p->table, p->len, p->state, ml, ml + (2 * slots(c->nkv) * per + 3) / 4 * 4, p->pages, p->seqs, p->width,
                        nq, g, target, 4, unit, per, multiplier(g, (uint64_t)b->n * g), multiplier(c->nkv, (groups + target) * c->nkv), c->mem + layer * layer_bytes(c->nkv, c->hd),
                        c->layers * layer_bytes(c->nkv, c->hd), 1.44269504f / sqrtf((float)c->hd)};
    hipStream_t st;
    if (!stream_of(stream, st)) return -1;
    const dim3 grid((unsigned)((groups + target) * c->nkv));
#define ATTEND(NB)                                                                                                                            \
    if (NB <= 4 && waves == 8 && !split) {                                                                                                    \
        if (dtype == L3M_HIP_F32) hipLaunchKernelGGL((k_kv8_attend<true, NB <= 4 ? NB : 4, 8>), grid, dim3(512), 0, st, a);                    \
        else hipLaunchKernelGGL((k_kv8_attend<false, NB <= 4 ? NB : 4, 8>), grid, dim3(512), 0, st, a);                                        \
    } else if (dtype == L3M_HIP_F32) hipLaunchKernelGGL((k_kv8_attend<true, NB, 4>), grid, dim3(256), 0, st, a);                               \
    else hipLaunchKernelGGL((k_kv8_attend<false, NB, 4>), grid, dim3(256), 0, st, a)
    BY_BLOCKS(ATTEND)
    if (split) {
        const dim3 all((unsigned)(groups * c->nkv));
#define JOINED(N)                                                                       \
    if (dtype == L3M_HIP_F32) hipLaunchKernelGGL((k_kv8_join<true, N>), all, dim3(N), 0, st, a); \
    else hipLaunchKernelGGL((k_kv8_join<false, N>), all, dim3(N), 0, st, a)
        // more threads where few workgroups have many parts: one token over 131071 58.6 us, by 256 threads 60.4; over 4001 12.3 and 11.7; 64 sequences of 100
        // to 8000 78.1 and 75.6
        if (shares < 128 && most > 8192) {
            JOINED(1024);
        } else {
            JOINED(256);
        }
    }
    return l3m_dev_launched("k_kv8_attend");
}

}
