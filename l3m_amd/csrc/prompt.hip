// Causal attention over whole prompts for CDNA4 (gfx950): bf16 rows of many sequences packed one behind the other, grouped heads.
//
// Rows: a kv head's (token, query head) pairs of a run, a token's heads side by side (g = nq / nkv); 32 to a wavefront. Per tile of 64 positions:
//   S = K Q^T        32 positions x 32 rows (v_mfma_f32_32x32x16_bf16), twice. The operand's rows are K's positions with bits 2 and 3 exchanged, so that a
//                    lane holds the scores of its row for eight positions in a row, which is what the next product wants of it: no value crosses lanes
//   P = 2^(S - m)    m moves only where a score passes it by 8: weights up to 2^8, and the sums are seldom scaled. Rounded to bf16, as the
//                    matrix cores take them beside V (a second part of what is left would be half as many products again), and summed as rounded
//   O^T += V^T P^T   32 dimensions x 32 rows x 16 positions, V read from LDS transposed (ds_read_b64_tr_b16)
// K's and V's tiles go from memory to LDS directly, 16 bytes a lane, in an order of pieces within a row by which no read meets a bank twice.
//
// Bound by instruction issue: beside a tile's products of a wavefront (32, hd 128) stand its softmax's some 130 vector instructions and 32 exponentials. Two
// workgroups of four wavefronts a CU fill each other's gaps. 8191 rows of 32/8 heads of 128: 540 to 575 us, 0.96 to 1.02 PFLOP/s, by the card (a bf16 product of 8192^3:
// 1.34); heads of 64 0.83 to 0.90, of 80 0.73 to 0.77 (80 of 96 columns are work), of 256 0.82 to 0.84 (one wavefront a SIMD). 24 prompts of 16 to 2048: 89 to 100 us,
// 0.49 to 0.55: many of their tiles lie on the diagonal, and workgroups are too short to hide their first loads. Five of 1 to 64 rows: 5.6 us, of which a launch is 1.6.
// Measured and not built: one tile in LDS and three workgroups a CU (8191 547 us, 24 prompts 97; hd 256 630 against 671); a tile's scores beside the last
// one's softmax (256 registers: 622 us); eight wavefronts a workgroup; wavefront priorities.
#include <type_traits>
#include "serve.h"

namespace {

constexpr int TILE = 64, ROWS = 32, WAVES = 4, CUS = 256;
constexpr float M0 = -3.40282347e38f;                                // the maximum of no score: float32's lowest
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
#define LOCAL __attribute__((address_space(3)))
#define GLOBAL __attribute__((address_space(1)))

struct PromptIn {
    const uint16_t *q, *k, *v;
    uint16_t       *out;
    Runs            b;
    long long       q_stride, kv_stride, out_stride;
    int             nq, nkv, hd, g;
    uint32_t        g_mul, nkv_mul;                                  // of g and of nkv (divide)
    int             items, cus;                                      // groups of a kv head, at the most; CUs' share of it
    float           scale;                                           // of the scores: base 2
};

// x plus the two bf16 values of a word, in float32: the weights that the product takes are the ones that are summed, so their rounding cancels where a few
// positions have all the weight. A sum waits for the last, so two take turns: 8191 rows of 32/8 heads of 128 544 us, 548 by one, 541 with the weights before their
// rounding (and 561 with the halves made floats, 571 by the matrix cores); of 64 307, 309, 309; 24 prompts 89.1, 89.9, 88.5.
__device__ __forceinline__ float add_pair(uint32_t w, float x) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, 0x3F803F80u), x, false);
}
// Values of a row in LDS, a power of two; pieces of 16 bytes.
__host__ __device__ constexpr int row_values(int nb) { return nb <= 1 ? 32 : nb <= 2 ? 64 : nb <= 4 ? 128 : 256; }
// Where a row's piece lies in it: K by rows read side by side, V by pairs of pieces, of rows r .. r + 3 and r + 8 .. r + 11.
template <int PIECES> __device__ __forceinline__ int k_turn(int row) { return PIECES >= 16 ? row & 15 : PIECES == 8 ? row >> 1 & 7 : row >> 2 & 3; }
template <int PIECES> __device__ __forceinline__ int v_turn(int row) {
    return PIECES >= 16 ? (row & 3) | (row >> 1 & 4) : PIECES == 8 ? (row >> 1 & 1) | (row >> 2 & 2) : 0;
}
__device__ __forceinline__ float other_half(float x, float &y) {     // lane ^ 32
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    y = __uint_as_float(r[1]);
    return __uint_as_float(r[0]);
}

// A workgroup's requests for a tile of K and V, 16 bytes a lane: the i-th round of them is rows i ROUND .. of the tile, in the order of LDS.
// (W 1: a wavefront's requests for a tile of its own.) PAD, for heads that are no multiple of 32: K's pieces past the head, which the products read, are zeros that
// stay; whatever else stood there would meet the queries' zeros, and an infinity times zero is NaN. (V's make dimensions that nobody reads.) Each of a wavefront's
// requests has lanes within the head, so the number under way is the same.
template <int NB, int W, bool PAD> struct Loader {
    static constexpr int RW = row_values(NB), PIECES = RW / 8, TURNS = TILE * PIECES / (64 * W), ROUND = 64 * W / PIECES;
    static constexpr int KINDS = ROUND < 16 ? 16 / ROUND : 1;        // orders of pieces among the rounds
    uint32_t k_off[KINDS], v_off[KINDS];                             // bytes behind a round's first row
    bool k_in[KINDS];                                                // PAD: the lane's piece of K is one of the head's
    const char *k, *v;
    long long row_bytes;
    int len, row, wave;
    __device__ __forceinline__ void init(const PromptIn &a, const uint16_t *k0, const uint16_t *v0, int rows) {
        const int thread = threadIdx.x % (64 * W), slot = thread % PIECES, last = (a.hd >> 3) - 1;
        k = (const char *)k0;
        v = (const char *)v0;
        len = rows;
        row_bytes = 2 * a.kv_stride;
        row = thread / PIECES;
        wave = __builtin_amdgcn_readfirstlane(thread >> 6);
#pragma unroll
        for (int i = 0; i < KINDS; i++) {
            if constexpr (PAD) k_in[i] = (slot ^ k_turn<PIECES>(row + i * ROUND)) <= last;
            k_off[i] = (uint32_t)(row * (int)row_bytes + 16 * min(slot ^ k_turn<PIECES>(row + i * ROUND), last));
            v_off[i] = (uint32_t)(row * (int)row_bytes + 16 * min(slot ^ v_turn<PIECES>(row + i * ROUND) << 1, last));
        }
    }
    // The pieces of K's tile that no request brings. Of a wavefront's own rounds; others read them behind a barrier.
    __device__ __forceinline__ void clear_k(uint16_t *k_s) const {
        if constexpr (PAD)
#pragma unroll
            for (int i = 0; i < TURNS; i++)
                if (!k_in[i % KINDS]) *(u32x4 *)(k_s + 512 * (i * W + wave) + 8 * (threadIdx.x & 63)) = u32x4{0, 0, 0, 0};
    }
    // Positions TILE tile .. of K or V into LDS; positions past the last one are the last one again, pieces past the head its last.
    __device__ __forceinline__ void request_one(int tile, const char *from, const uint32_t (&off)[KINDS], uint16_t *to) const {
        const char *at = from + tile * TILE * row_bytes;
        const int over = tile * TILE + TILE - len;                   // rows past the last
        if (__builtin_expect(over > 0, 0)) {
            asm volatile("");                                        // no selects for all tiles' sake
#pragma unroll
            for (int i = 0; i < TURNS; i++) {
                const int less = max(row + i * ROUND - (TILE - 1 - over), 0);
                __builtin_amdgcn_global_load_lds((const GLOBAL void *)(at + ((i * ROUND - less) * row_bytes + off[i % KINDS])), (LOCAL void *)(to + 512 * (i * W + wave)), 16, 0, 0);
            }
        } else
#pragma unroll
            for (int i = 0; i < TURNS; i++)
                __builtin_amdgcn_global_load_lds((const GLOBAL void *)(at + i * ROUND * row_bytes + off[i % KINDS]), (LOCAL void *)(to + 512 * (i * W + wave)), 16, 0, 0);
    }
    // The same of K's pieces within the head alone; a kind's rounds together, so that lanes are left out once for each.
    __device__ __forceinline__ void request_in_head(int tile, uint16_t *to) const {
        const char *at = k + tile * TILE * row_bytes;
        const int over = tile * TILE + TILE - len;
#pragma unroll
        for (int j = 0; j < KINDS; j++)
            if (k_in[j]) {
                if (__builtin_expect(over > 0, 0)) {
                    asm volatile("");
#pragma unroll
                    for (int i = j; i < TURNS; i += KINDS) {
                        const int less = max(row + i * ROUND - (TILE - 1 - over), 0);
                        __builtin_amdgcn_global_load_lds((const GLOBAL void *)(at + ((i * ROUND - less) * row_bytes + k_off[j])), (LOCAL void *)(to + 512 * (i * W + wave)), 16, 0, 0);
                    }
                } else
#pragma unroll
                    for (int i = j; i < TURNS; i += KINDS)
                        __builtin_amdgcn_global_load_lds((const GLOBAL void *)(at + i * ROUND * row_bytes + k_off[j]), (LOCAL void *)(to + 512 * (i * W + wave)), 16, 0, 0);
            }
    }
    __device__ __forceinline__ void request_k(int tile, uint16_t *k_s) const {
        if constexpr (PAD) request_in_head(tile, k_s);
        else request_one(tile, k, k_off, k_s);
    }
    __device__ __forceinline__ void request_v(int tile, uint16_t *v_s) const { request_one(tile, v, v_off, v_s); }
    __device__ __forceinline__ void request(int tile, uint16_t *k_s, uint16_t *v_s) const {
        request_k(tile, k_s);
        request_v(tile, v_s);
    }
};
// All but the last N requests are done.
template <int N> __device__ __forceinline__ void requests_but() { __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | (N >> 4) << 14); }

__device__ __forceinline__ void loads_done() {                       // and the workgroup's
    __builtin_amdgcn_s_waitcnt(0x0F70);                              // vmcnt(0)
    __syncthreads();
}

// Groups of rows, a workgroup's. Those of the last rows have the most tiles, so they come first, over all runs, or the longest run's would be left at the end:
// the item-th of a kv head's groups by descending number in their run (up to 64 runs; more fill the card without an order). Where all are resident
// at once, two to a CU, the second ones come shortest first, so that a CU's two are about as long together as any other's. 24 prompts: 94.7 us, run by run 103.3;
// 8191 rows: 535, by ascending number 582; 2048: 54.3, without the second half's order 55.8.
template <int GROUP> __device__ __forceinline__ int groups_of(int rows, int g) { return (int)(((unsigned)rows * (unsigned)g + GROUP - 1) / GROUP); }
template <int GROUP> __device__ __forceinline__ Found group_of(const Runs &b, int g, int item, int items, int cus) {
    if (items <= 2 * cus && item >= cus) item = cus + items - 1 - item;
    if (b.seqs > 64) return find_run<WAVES>(b, items - 1 - item, [&](int, int, int rows) { return groups_of<GROUP>(rows, g); });
    const int lane = threadIdx.x & 63;
    int s0 = 0, rows = 0;
    if (lane < b.seqs) {
        s0 = b.from(lane);
        rows = b.to(lane, s0) - s0;
    }
    const int groups = groups_of<GROUP>(rows, g);
    // the highest level at which more than `item` groups lie at it or above
    auto above = [&](int level) { return __builtin_amdgcn_readlane(scan_wave(max(groups - level, 0)), 63); };
    int level = 0, top = (int)max_wave((float)min(groups, 1 << 24));
    if (above(0) <= item) return {-1, 0, 0, 0};
    while (top - level > 1) {
        const int mid = (level + top) >> 1;
        if (above(mid) > item) level = mid;
        else top = mid;
    }
    const int rank = item - above(level + 1);                        // among the runs that have a group there
    const bool has = groups > level;
    const int before = scan_wave(has) - has;
    const uint64_t at = __ballot(has && before == rank);
    const int l = __builtin_ctzll(at);
    return {l, level, __builtin_amdgcn_readlane(s0, l), __builtin_amdgcn_readlane(rows, l)};
}

// One row by the formula, a position at a time: for rows whose products met a value that is not finite behind their token. Exponents as where rows are computed
// together: their rounding cancels for small maxima and is alike for large ones, and a score of -inf has no weight, be it the first.
__device__ void row_alone(const PromptIn &a, const uint16_t *q, const uint16_t *k, const uint16_t *v, int seen, uint16_t *out) {
    const int lane = threadIdx.x & 63;
    float qv[4], o[4] = {0, 0, 0, 0}, m = M0, l = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) qv[i] = lane + 64 * i < a.hd ? bf16_float(q[lane + 64 * i]) : 0.f;
    for (int p = 0; p < seen; p++) {
        float s = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) s += lane + 64 * i < a.hd ? qv[i] * bf16_float(k[(long long)p * a.kv_stride + lane + 64 * i]) : 0.f;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
        const float top = fmaxf(m, s * a.scale), by = __builtin_amdgcn_exp2f(m - top);
        const float e = __builtin_amdgcn_exp2f(fabsf(top) > LARGE_SCORE ? scaled_less(s, a.scale, top) : fmaf(s, a.scale, -top));
        l = l * by + e;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = o[i] * by + (lane + 64 * i < a.hd ? e * bf16_float(v[(long long)p * a.kv_stride + lane + 64 * i]) : 0.f);
        m = top;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (lane + 64 * i < a.hd) out[lane + 64 * i] = (uint16_t)bf16_pair(o[i] / l, 0.f);
}

// Whether a value behind token t, of those before `upto`, may have changed its row: one that is not finite, in a dimension that no value up to the token makes NaN
// anyway. A lane takes a piece of eight dimensions of every few positions, 0x8000 a dimension. 4096 rows of 16/4 heads of 128, a dimension of all values NaN: 0.21 ms
// (none: 0.12), where every such row made anew takes 94; infinities at every position still do.
__device__ bool reached(const PromptIn &a, const uint16_t *v, int t, int upto) {
    const int lane = threadIdx.x & 63, pieces = a.hd >> 3, bits = 32 - __clz(pieces - 1), mine = lane >> bits, at_once = 64 >> bits;   // pieces 1: __clz(0) is 32
    const uint16_t *from = v + 8 * min(lane & ((1 << bits) - 1), pieces - 1);
    auto load = [&](int p) { return *(const u32x4 *)(from + (long long)p * a.kv_stride); };
    auto join = [&](u32x4 &m) {                                      // over the positions
        for (int d = 1 << bits; d < 64; d <<= 1)
#pragma unroll
            for (int i = 0; i < 4; i++) m[i] |= (uint32_t)__shfl_xor((int)m[i], d);
    };
    u32x4 open = {0, 0, 0, 0};
    auto some = [&] { return __ballot((open[0] | open[1] | open[2] | open[3]) != 0) != 0; };
    for (int p = t + 1 + mine; p < upto; p += at_once) open |= ((load(p) & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
    join(open);
    for (int p = t; p >= 0 && some(); p -= 4 * at_once) {
        u32x4 nan = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 4; k++) nan |= ((load(max(p - mine - k * at_once, 0)) & 0x7FFF7FFFu) + 0x007F007Fu) & 0x80008000u;
        join(nan);
        open &= ~nan;
    }
    return some();
}

// SPLIT, for few groups: the four wavefronts take a group of 32 rows together, a tile each in turn, by themselves (the next K comes from a tile's scores on, the next V
// from its values on), and their parts meet in LDS, in a fixed order.
template <int NB, bool SPLIT, bool PAD> __global__ void __launch_bounds__(64 * WAVES) k_attend_packed(PromptIn a) {
    constexpr int RW = row_values(NB), PIECES = RW / 8, GROUP = SPLIT ? ROWS : ROWS * WAVES;
    constexpr int TILES = SPLIT ? WAVES * TILE * RW : TILE * RW, OTHER = SPLIT ? 8 : TILE * RW;
    // two tiles: the next one comes while one is used. Arrays of their own, so that the compiler sees that reads of one do not wait for the other's requests
    __shared__ __align__(16) uint16_t k0_s[TILES], v0_s[TILES], k1_s[OTHER], v1_s[OTHER];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r32 = lane & 31, c = lane >> 5, hd = a.hd, g = a.g;
    // kv heads fastest: consecutive workgroups go to different XCDs, so 8 heads keep to an L2 each
    const int item = (int)divide(blockIdx.x, a.nkv, a.nkv_mul), h = (int)blockIdx.x - item * a.nkv;
    const Found f = group_of<GROUP>(a.b, g, item, a.items, a.cus);
    if (f.run < 0) return;
    const uint16_t *q = a.q + (long long)f.s0 * a.q_stride, *k = a.k + (long long)f.s0 * a.kv_stride + h * hd, *v = a.v + (long long)f.s0 * a.kv_stride + h * hd;
    uint16_t *out = a.out + (long long)f.s0 * a.out_stride;
    const int R = f.rows * g, first = f.at * GROUP, row0 = SPLIT ? first : first + wave * ROWS;
    const int tiles = (int)divide(min(first + GROUP, R) - 1, g, a.g_mul) / TILE + 1;      // of the workgroup
    const int rows = clamp(R - row0, 0, ROWS), row = row0 + min(r32, max(rows, 1) - 1);
    const int token = rows ? (int)divide(row, g, a.g_mul) : 0, head = rows ? h * g + row - token * g : 0;
    const int low = rows ? (int)divide(row0, g, a.g_mul) : 0, high = rows ? (int)divide(row0 + rows - 1, g, a.g_mul) : -1;   // the wavefront's tokens
    const uint16_t *my_q = q + (long long)token * a.q_stride + (long long)head * hd;
    bf16x8 qs[2 * NB];
#pragma unroll
    for (int i = 0; i < 2 * NB; i++) {
        const int d = 16 * i + 8 * c;
        u32x4 x = *(const u32x4 *)(my_q + (d < hd ? d : 0));
        if (d >= hd) x = u32x4{0, 0, 0, 0};
        qs[i] = __builtin_bit_cast(bf16x8, x);
    }
    Loader<NB, SPLIT ? 1 : WAVES, PAD> loads;
    loads.init(a, k, v, f.rows);
    uint16_t *my_k = SPLIT ? k0_s + wave * TILE * RW : k0_s, *my_v = SPLIT ? v0_s + wave * TILE * RW : v0_s;
    loads.clear_k(my_k);
    if constexpr (!SPLIT) loads.clear_k(k1_s);
    loads.request(SPLIT ? min(wave, tiles - 1) : 0, my_k, my_v);
#pragma unroll
    for (int i = 0; i < 2 * NB; i++) asm volatile("" : "+v"(qs[i]));   // here, or the loop waits for requests at its top
    const float scale = a.scale;
    f32x16 acc[NB];
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
        for (int j = 0; j < 16; j++) acc[i][j] = 0.f;
    float m = M0, l = 0.f, sums[2] = {};                             // of the weights, in turn (add_pair)
    bool large = false;                                              // some row's m is (LARGE_SCORE)

    auto step = [&](int tile, const uint16_t *k_s, const uint16_t *v_s) {
        constexpr int REQUESTS = decltype(loads)::TURNS;
        const int next = min(tile + WAVES, tiles - 1);
        if constexpr (SPLIT) requests_but<REQUESTS>();               // V's, which came behind K's
        f32x16 s[2];
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int j = 0; j < 16; j++) s[b][j] = 0.f;
        const int key = (r32 & 19) + (r32 & 4) * 2 + (r32 & 8) / 2;    // bits 2 and 3 exchanged
        auto keys = [&](int i, int b) { return *(const bf16x8 *)(k_s + (32 * b + key) * RW + 8 * ((2 * i + c) ^ k_turn<PIECES>(key))); };
        bf16x8 kx[2][2];
        kx[0][0] = keys(0, 0);
        kx[0][1] = keys(0, 1);
#pragma unroll
        for (int i = 0; i < 2 * NB; i++) {
            if (i + 1 < 2 * NB) {
                kx[(i + 1) & 1][0] = keys(i + 1, 0);
                kx[(i + 1) & 1][1] = keys(i + 1, 1);
            }
#pragma unroll
            for (int b = 0; b < 2; b++) s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kx[i & 1][b], qs[i], s[b], 0, 0, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);           // LDS reads two products ahead
#pragma unroll
        for (int i = 0; i < 2 * NB; i++) {
            __builtin_amdgcn_sched_group_barrier(0x8, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        if constexpr (SPLIT) {
            __builtin_amdgcn_s_waitcnt(0xC07F);                      // LDS is read
            loads.request_k(next, my_k);
        }
        // s[b][8 j + e]: position 32 b + 16 j + 8 c + e
        if (__builtin_expect(tile * TILE + TILE - 1 > low, 0)) {
            asm volatile("");                                        // no selects for all tiles' sake
            const int seen = token - tile * TILE - 8 * c;
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int j = 0; j < 16; j++) s[b][j] = 32 * b + 16 * (j >> 3) + (j & 7) <= seen ? s[b][j] : -INFINITY;
        }
        float top = s[0][0];
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int j = 0; j < 16; j++) top = fmaxf(top, s[b][j]);
        float y;
        top = other_half(top, y);
        top = fmaxf(top, y) * scale;
        if (__ballot(top > m + 8.f)) {
            const float to = top > m + 8.f ? top : m, by = m == to ? 1.f : __builtin_amdgcn_exp2f(m - to);
#pragma unroll
            for (int i = 0; i < 2; i++) sums[i] *= by;
#pragma unroll
            for (int i = 0; i < NB; i++) acc[i] *= by;
            m = to;
            large = __ballot(fabsf(m) > LARGE_SCORE && m != M0) != 0;
        }
        float by = scale, less = m;
        if (__builtin_expect(large, 0)) {
            asm volatile("");
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int j = 0; j < 16; j++) s[b][j] = scaled_less(s[b][j], scale, m);
            by = 1.f;
            less = 0.f;
        }
        // lane (c, d): positions 8 c .. + 7 of dimension d, four at a time of 16 dimensions by 16 lanes
        auto values = [&](int n) {
            const int i = n % NB, b = n / NB >> 1, j = n / NB & 1;
            s16x4 x[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int at = 32 * b + 16 * j + 8 * c + 4 * u + (lane >> 2 & 3), pair = 2 * i + (lane >> 4 & 1);
                x[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LOCAL s16x4 *)(v_s + at * RW + 16 * (pair ^ v_turn<PIECES>(8 * c + (lane >> 2 & 3))) + 4 * (lane & 3)));
            }
            typedef short s16x8 __attribute__((ext_vector_type(8)));
            return __builtin_bit_cast(bf16x8, s16x8{x[0][0], x[0][1], x[0][2], x[0][3], x[1][0], x[1][1], x[1][2], x[1][3]});
        };
        bf16x8 p[2][2], vx[2];
        if constexpr (SPLIT) requests_but<REQUESTS>();               // the next K's, which came behind V's
        vx[0] = values(0);
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                u32x4 w;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x0 = __builtin_amdgcn_exp2f(fmaf(s[b][8 * j + 2 * e], by, -less)), x1 = __builtin_amdgcn_exp2f(fmaf(s[b][8 * j + 2 * e + 1], by, -less));
                    w[e] = bf16_pair(x0, x1);
                    sums[e & 1] = add_pair(w[e], sums[e & 1]);
                }
                p[b][j] = __builtin_bit_cast(bf16x8, w);
            }
#pragma unroll
        for (int n = 0; n < 4 * NB; n++) {
            if (n + 1 < 4 * NB) vx[(n + 1) & 1] = values(n + 1);
            acc[n % NB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vx[n & 1], p[n / NB >> 1][n / NB & 1], acc[n % NB], 0, 0, 0);
        }
        if constexpr (SPLIT) {
            __builtin_amdgcn_s_waitcnt(0xC07F);
            loads.request_v(next, my_v);
        }
    };
    auto turn = [&](int tile, const uint16_t *k_s, const uint16_t *v_s, uint16_t *next_k, uint16_t *next_v) {
        loads_done();                                                // this tile is here, and nobody reads the last one any more
        if (tile + 1 < tiles) loads.request(tile + 1, next_k, next_v);
        if (tile * TILE <= high) step(tile, k_s, v_s);
    };
    if constexpr (SPLIT) {
        for (int tile = wave; tile < tiles; tile += WAVES) step(tile, my_k, my_v);
        requests_but<0>();
    } else
        for (int tile = 0; tile < tiles; tile += 2) {
            turn(tile, k0_s, v0_s, k1_s, v1_s);
            if (tile + 1 < tiles) turn(tile + 1, k1_s, v1_s, k0_s, v0_s);
        }
    __syncthreads();                                                 // the tiles are done with
    if (!rows) return;                                               // (a group has rows, so not where all meet)
    float y;
#pragma unroll
    for (int i = 0; i < 2; i++) l += sums[i];
    l = other_half(l, y);
    l += y;
    float bad = 0.f;                                                 // NaN where a value is not finite
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
        for (int j = 0; j < 16; j++) bad = fmaf(acc[i][j], 0.f, bad);
    const uint64_t lanes = __ballot(bad != bad);
    uint32_t wrong = 0;                                              // rows that a value behind their token may have reached
    if (__builtin_expect(lanes != 0, 0))                             // (else the loop over tiles is laid out worse, 1%)
        for (uint32_t of = (uint32_t)lanes | (uint32_t)(lanes >> 32); of; of &= of - 1) {
            const int r = __builtin_ctz(of), t = __builtin_amdgcn_readlane(token, r), upto = min((high / TILE + 1) * TILE, f.rows);
            if (r >= rows) break;
            if (reached(a, v, t, upto)) wrong |= 1u << r;
        }
    constexpr int HP = 32 * NB;
    if constexpr (SPLIT) {
        constexpr int OS = HP + 4;
        static_assert(2 * ROWS * OS * 4 <= (int)sizeof(k0_s), "");
        __shared__ float m_s[WAVES][ROWS], l_s[WAVES][ROWS];
        __shared__ uint32_t wrong_s[WAVES];
        float (*o_s)[ROWS][OS] = (float (*)[ROWS][OS])k0_s, (*p_s)[ROWS][OS] = (float (*)[ROWS][OS])v0_s;   // of two wavefronts each
        float (*mine)[OS] = wave < 2 ? o_s[wave] : p_s[wave - 2];
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) mine[r32][32 * i + 8 * j + 4 * c + e] = acc[i][4 * j + e];
        if (c == 0) {
            m_s[wave][r32] = m;
            l_s[wave][r32] = l;
        }
        if (lane == 0) wrong_s[wave] = wrong;
        __syncthreads();
        wrong = wrong_s[0] | wrong_s[1] | wrong_s[2] | wrong_s[3];
        static_assert(WAVES == 4, "");
        for (int at = threadIdx.x; at < rows * (hd >> 3); at += 64 * WAVES) {
            const int r = at / (hd >> 3), d = 8 * (at - r * (hd >> 3));
            if (wrong >> r & 1u) continue;
            const float top = fmaxf(fmaxf(m_s[0][r], m_s[1][r]), fmaxf(m_s[2][r], m_s[3][r]));
            float x[8] = {0, 0, 0, 0, 0, 0, 0, 0}, sum = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                const float part = __builtin_amdgcn_exp2f(m_s[w][r] - top), *from = w < 2 ? &o_s[w][r][d] : &p_s[w - 2][r][d];
                sum = fmaf(l_s[w][r], part, sum);
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = fmaf(from[e], part, x[e]);
            }
            const float one = 1.f / sum;
            const int rr = row0 + r, t = (int)divide(rr, g, a.g_mul), hh = h * g + rr - t * g;
            *(u32x4 *)(out + (long long)t * a.out_stride + (long long)hh * hd + d) =
                u32x4{bf16_pair(x[0] * one, x[1] * one), bf16_pair(x[2] * one, x[3] * one), bf16_pair(x[4] * one, x[5] * one), bf16_pair(x[6] * one, x[7] * one)};
        }
        for (uint32_t of = wrong; of; of &= of - 1) {
            const int r = __builtin_ctz(of), t = __builtin_amdgcn_readlane(token, r), hh = __builtin_amdgcn_readlane(head, r);
            if (r % WAVES == wave) row_alone(a, q + (long long)t * a.q_stride + (long long)hh * hd, k, v, t + 1, out + (long long)t * a.out_stride + (long long)hh * hd);
        }
        return;
    }
    for (uint32_t of = wrong; of; of &= of - 1) {
        const int r = __builtin_ctz(of), t = __builtin_amdgcn_readlane(token, r), hh = __builtin_amdgcn_readlane(head, r);
        row_alone(a, q + (long long)t * a.q_stride + (long long)hh * hd, k, v, t + 1, out + (long long)t * a.out_stride + (long long)hh * hd);
    }
    // through LDS, 32 rows a wavefront, so that rows leave in whole lines; a row's pieces of 16 bytes in the order that K's have
    uint16_t *o_s = wave < 2 ? k0_s + wave * ROWS * HP : v0_s + (wave - 2) * ROWS * HP;
    static_assert(WAVES == 4 && 2 * ROWS * HP <= TILE * RW, "");
    const float by = 1.f / l;
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
        for (int j = 0; j < 4; j++)
            *(u32x2 *)(o_s + r32 * HP + 8 * ((4 * i + j) ^ (r32 & 3)) + 4 * c) = u32x2{bf16_pair(acc[i][4 * j] * by, acc[i][4 * j + 1] * by), bf16_pair(acc[i][4 * j + 2] * by, acc[i][4 * j + 3] * by)};
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int i = 0; i < 2 * NB; i++) {
        const int at = 64 * i + lane, r = at / (4 * NB), piece = at - r * (4 * NB);
        const u32x4 x = *(const u32x4 *)(o_s + r * HP + 8 * (piece ^ (r & 3)));
        if (r >= rows || 8 * piece >= hd || wrong >> r & 1u) continue;
        const int rr = row0 + r, t = (int)divide(rr, g, a.g_mul), hh = h * g + rr - t * g;
        *(u32x4 *)(out + (long long)t * a.out_stride + (long long)hh * hd + 8 * piece) = x;
    }
}

}  // namespace

extern "C" {

int l3m_k_attend_packed(uint16_t *out, int out_stride, const uint16_t *q, int q_stride, const uint16_t *k, const uint16_t *v, int kv_stride, const l3m_batch *b,
                        int nq, int nkv, int hd, void *stream) {
    if (const char *why = batch_bad(b)) return l3m_dev_fail(why);
    if (hd < 8 || hd > 256 || hd % 8) return l3m_dev_fail("attend_packed: hd must be a multiple of 8 up to 256");
    if (nkv < 1 || nkv > 4096 || nq < 1 || nq > 65536 || nq % nkv) return l3m_dev_fail("attend_packed: query heads must be a multiple of the kv heads");
    const long long qw = (long long)nq * hd, kw = (long long)nkv * hd;
    if (q_stride < qw || out_stride < qw || kv_stride < kw) return l3m_dev_fail("attend_packed: a row holds fewer values than its heads");
    if (!b->seqs || !b->n) return 0;
    if (!out || !q || !k || !v) return l3m_dev_fail("attend_packed: no rows, or no output");
    if (((uintptr_t)out | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % 16 || q_stride % 8 || kv_stride % 8 || out_stride % 8)
        return l3m_dev_fail("attend_packed: rows must be 16-byte aligned, strides multiples of 8 values");
    const size_t ob = rows_bytes(b->n, out_stride, qw, 2), kb = rows_bytes(b->n, kv_stride, kw, 2);
    if (!(out == q && out_stride == q_stride) && overlap(out, ob, q, rows_bytes(b->n, q_stride, qw, 2))) return l3m_dev_fail("attend_packed: q and out must be the same or apart");
    // in a fused row k and v lie behind q, so out == q lies between them
    auto apart = [&](const uint16_t *x) {
        if (!overlap(out, ob, x, kb)) return true;
        const long long gap = x - out;
        return out_stride == kv_stride && (gap >= 0 ? gap >= qw && gap + kw <= kv_stride : -gap >= kw && qw - gap <= kv_stride);
    };
    if (!apart(k) || !apart(v)) return l3m_dev_fail("attend_packed: out overlaps k or v");
    if (on_batch(b, out, ob)) return l3m_dev_fail("attend_packed: out overlaps the batch");
    if (kv_stride > 1 << 23) return l3m_dev_fail("attend_packed: rows of K and V may be up to 2^23 values apart");   // a tile's offsets in 32 bits
    const int g = nq / nkv;
    if ((long long)b->n * g > 1 << 28) return l3m_dev_fail("attend_packed: too many rows for one call");
    long long items = (long long)b->n * g / (ROWS * WAVES) + b->seqs;
    if (items * nkv > 1ll << 28) return l3m_dev_fail("attend_packed: too many rows for one call");
    // Wavefronts share groups of 32 rows where groups of 128 are too few for the card, in one tile's time for four, and not where a run has a tile or so: 2000
    // rows of 9/3 heads of 64 (141 groups of 128) 19.3 us against 34.5, 3000 (213) 31 and 48, 1500 of 32/4 (376) 31.4 and 28.1; of 64 rows 6.1 and 5.6. Past 64
    // a CU holds one such workgroup: 1705 of 3/1 heads of 80 (40) 18.2 and 33.8, 700 of 16/2 of 128 (88) 17.6 and 19.2, 400 of 32/8 (104) 17.2 and 14.5. Past 128 none.
    const bool split = hd <= 128 && items * nkv < (hd <= 64 ? 256 : 96) && b->n > TILE * b->seqs;
    if (split) items = (long long)b->n * g / ROWS + b->seqs;
    const PromptIn a = {q, k, v, out, runs_of(b), q_stride, kv_stride, out_stride, nq, nkv, hd, g, multiplier(g, (uint64_t)b->n * g), multiplier(nkv, items * nkv),
                        (int)items, CUS / nkv, 1.44269504f / sqrtf((float)hd)};
    hipStream_t st;
    if (!stream_of(stream, st)) return -1;
    const dim3 grid((unsigned)(items * nkv)), wg(64 * WAVES);
#define KERNEL(NB, SPLIT)                                                                                       \
    if (hd % 32) hipLaunchKernelGGL((k_attend_packed<NB, SPLIT, true>), grid, wg, 0, st, a);                      \
    else hipLaunchKernelGGL((k_attend_packed<NB, SPLIT, false>), grid, wg, 0, st, a)
#define ATTEND(NB)                                                                                              \
    if (split) {                                                                                                \
        KERNEL((NB <= 4 ? NB : 4), (NB <= 4));                                                                  \
    } else {                                                                                                    \
        KERNEL(NB, false);                                                                                      \
    }
    switch ((hd + 31) / 32) {
    case 1: ATTEND(1); break;
    case 2: ATTEND(2); break;
    case 3: ATTEND(3); break;
    case 4: ATTEND(4); break;
    case 5: ATTEND(5); break;
    case 6: ATTEND(6); break;
    case 7: ATTEND(7); break;
    default: ATTEND(8); break;
    }
#undef ATTEND
#undef KERNEL
    return l3m_dev_launched("k_attend_packed");
}

}
