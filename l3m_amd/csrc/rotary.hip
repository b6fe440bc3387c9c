// Rotary positions of query and key heads for CDNA4 (gfx950): a position for each row, pairs (2i, 2i + 1) or halves, the whole head or its first
// part, frequencies scaled for long contexts.
#include "serve.h"

namespace {

constexpr int THREADS = 256;

struct RotaryIn {
    l3m_rotary     r;
    const void    *x;
    void          *q, *k;
    const int32_t *pos;
    long long      stride, q_stride, k_stride;
    int            n, nq, nkv, pos0, tokens;                         // tokens: of a workgroup
    int            turned, per_head, per_token, rest_gap;            // items: of the turned part of a head, of a head, of a token; rest_gap: below
    uint32_t       token_mul, head_mul, pair_mul;                    // of per_token, per_head and rd / 2 (divide)
};

// Sine and cosine of `turns` 2^-64 of a turn: the angle is a whole number, so its quarter and what is left of it are exact for any position;
// then the power series in 64 bits on [-pi / 4, pi / 4], off by less than 1e-13.
__device__ __forceinline__ void sincos_turns(uint64_t turns, double &s, double &c) {
    const uint64_t quarter = (turns + (1ull << 61)) >> 62;
    const double   x = (double)(int64_t)(turns - (quarter << 62)) * 3.4061215800304124e-19, y = x * x;   // 2 pi 2^-64
    const double   sn = x * (1 + y * (-1.0 / 6 + y * (1.0 / 120 + y * (-1.0 / 5040 + y * (1.0 / 362880 + y * (-1.0 / 39916800 + y * (1.0 / 6227020800.0)))))));
    const double   cs = 1 + y * (-0.5 + y * (1.0 / 24 + y * (-1.0 / 720 + y * (1.0 / 40320 + y * (-1.0 / 3628800 + y * (1.0 / 479001600.0 + y * (-1.0 / 87178291200.0)))))));
    s = quarter & 1 ? cs : sn;
    c = quarter & 1 ? sn : cs;
    if (quarter & 2) s = -s;
    if ((quarter + 1) & 2) c = -c;
}

// V values of type T as they lie in memory, and as float32.
template <class T, int V> struct Raw {
    static constexpr int words = V * (int)sizeof(T) < 4 ? 1 : V * (int)sizeof(T) / 4;
    uint32_t w[words];
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (V == 1) w[0] = sizeof(T) == 4 ? *(const uint32_t *)p : *(const uint16_t *)p;
        else
#pragma unroll
            for (int i = 0; i < words; i += 4) {
                const u32x4 x = *(const u32x4 *)(p + i * V / words);
#pragma unroll
                for (int j = 0; j < 4; j++) w[i + j] = x[j];
            }
    }
    __device__ __forceinline__ float value(int i) const { return sizeof(T) == 4 ? __uint_as_float(w[i]) : __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16); }
};
template <class T, int V> __device__ __forceinline__ void store_values(T *p, const float (&x)[V]) {
    if constexpr (V == 1) {
        if constexpr (sizeof(T) == 4) *(float *)p = x[0];
        else *(uint16_t *)p = (uint16_t)bf16_pair(x[0], 0.f);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V; i += 4) *(f32x4 *)(p + i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
    } else *(u32x4 *)p = u32x4{bf16_pair(x[0], x[1]), bf16_pair(x[2], x[3]), bf16_pair(x[4], x[5]), bf16_pair(x[6], x[7])};
}

// y = mag (u c - w s, u s + w c) of each pair (u, w), c and s of position times frequency; what lies behind the turned part goes as it is. A workgroup makes
// its tokens' sines once, in LDS, while the first rows come, and then turns every head by them. A thread's items, UNROLL at once: V pairs (halves: V values of
// either half; else V values, pairs side by side; V 1: a pair), or of what lies behind the turned part V values, and V more rest_gap behind them where that is not 0.
// Bound by the bytes: 8192 rows of 32 + 8 heads of 128 out of wider ones, half of each turned, bf16: 168 MB in 39.8 us, 4.2 TB/s (a copy of 1 GiB: 5.2); 16384: 4.75.
// One row: 3.4 us, of which a launch is 1.6.
// (Of one item at a time: 1000 rows 6.8 us against 6.6, 8192 the same.)
template <class TI, int V> constexpr int unroll() { return V == 1 || sizeof(TI) == 4 ? 2 : 4; }
template <class TI, class TO, int V> __global__ void __launch_bounds__(THREADS) k_rotary(RotaryIn a) {
    constexpr int UNROLL = unroll<TI, V>();
    extern __shared__ float cs_s[];                                  // [tokens][rd / 2] (cos, sin)
    const int pairs = a.r.rd >> 1, t0 = (int)blockIdx.x * a.tokens, tokens = min(a.tokens, a.n - t0), halves = a.r.halves, hd = a.r.hd, rd = a.r.rd;
    const unsigned items = (unsigned)(tokens * a.per_token);
    struct Item {
        const TI *x;
        TO       *y;
        const float *cs;
        int       d, gap;                                            // first value; how far second ones lie behind, 0: beside them, or there are none
        bool      turn;
    };
    auto item_at = [&](unsigned i) {
        const unsigned t = divide(i, a.per_token, a.token_mul), j = i - t * a.per_token, h = divide(j, a.per_head, a.head_mul);
        const int e = (int)(j - h * a.per_head);
        const size_t row = (size_t)t0 + t;
        Item m;
        m.turn = e < a.turned;
        m.gap = !m.turn ? a.rest_gap : halves ? pairs : V == 1 ? 1 : 0;
        m.d = !m.turn ? rd + (e - a.turned) * V : V == 1 && !halves ? 2 * e : e * V;
        m.x = (const TI *)a.x + row * a.stride + (size_t)h * hd + m.d;
        m.y = ((int)h >= a.nq ? (TO *)a.k + row * a.k_stride + (size_t)((int)h - a.nq) * hd : (TO *)a.q + row * a.q_stride + (size_t)h * hd) + m.d;
        m.cs = cs_s + 2 * (t * pairs) + (halves ? 2 * m.d : m.d);
        return m;
    };
    Item         m[UNROLL];
    Raw<TI, V>   u[UNROLL], w[UNROLL];
    auto request = [&](unsigned i0) {
#pragma unroll
        for (int k = 0; k < UNROLL; k++) {
            const unsigned i = i0 + k * THREADS;
            if (i >= items) continue;
            m[k] = item_at(i);
            u[k].load(m[k].x);
            if (m[k].gap > 0) w[k].load(m[k].x + m[k].gap);
        }
    };
    request(threadIdx.x);
    for (int i = threadIdx.x; i < tokens * pairs; i += THREADS) {
        const int t = (int)divide(i, pairs, a.pair_mul), p = i - t * pairs;
        const long long pos = a.pos ? a.pos[t0 + t] : (long long)a.pos0 + t0 + t;
        double s, c;
        sincos_turns((uint64_t)pos * a.r.turn[p], s, c);
        cs_s[2 * i] = (float)(c * (double)a.r.mag);
        cs_s[2 * i + 1] = (float)(s * (double)a.r.mag);
    }
    __syncthreads();
    for (unsigned i0 = threadIdx.x; i0 < items; i0 += UNROLL * THREADS) {
        if (i0 != threadIdx.x) request(i0);
#pragma unroll
        for (int k = 0; k < UNROLL; k++) {
            if (i0 + k * THREADS >= items) continue;
            float x[V], z[V];
            const float *cs = m[k].cs;
            if (!m[k].turn) {
#pragma unroll
                for (int r = 0; r < V; r++) {
                    x[r] = u[k].value(r);
                    z[r] = w[k].value(r);
                }
            } else if (m[k].gap > 0) {
#pragma unroll
                for (int r = 0; r < V; r++) {
                    const float c = cs[2 * r], s = cs[2 * r + 1], p = u[k].value(r), o = w[k].value(r);
                    x[r] = p * c - o * s;
                    z[r] = p * s + o * c;
                }
            } else if constexpr (V > 1) {
#pragma unroll
                for (int r = 0; r < V; r += 2) {
                    const float c = cs[r], s = cs[r + 1], p = u[k].value(r), o = u[k].value(r + 1);
                    x[r] = p * c - o * s;
                    x[r + 1] = p * s + o * c;
                }
            }
            if (m[k].gap > 0) store_values<TO, V>(m[k].y + m[k].gap, z);
            store_values<TO, V>(m[k].y, x);
        }
    }
}

template <class TI, class TO, int V> int launch(RotaryIn a, hipStream_t st) {
    const int pairs = a.r.rd / 2, heads = a.nq + a.nkv;
    // what does not turn stays where it is where both outputs are the rows' own heads
    const bool in_place = (!a.q || a.q == a.x) && (!a.k || a.k == (const TI *)a.x + (size_t)a.nq * a.r.hd), rest = !in_place;
    const int  behind = rest ? a.r.hd - a.r.rd : 0;
    a.rest_gap = V > 1 && a.r.halves && behind % (2 * V) == 0 ? behind / 2 : 0;    // as many bytes an item as the halves' items
    a.turned = V == 1 ? pairs : a.r.halves ? pairs / V : a.r.rd / V;
    a.per_head = a.turned + (a.rest_gap ? behind / 2 : behind) / V;
    a.per_token = a.per_head * heads;
    if (!a.per_token) return 0;
    // a workgroup's tokens: one while there are few; then as many up to 8 as give its threads whole turns, with a sine a thread at the most. 32 + 8 heads of 128,
    // half of each turned: 8192 rows 39.8 us against 40.8 by one token, 4096 18.7 and 19.2, 2048 11.2 and 10.8, 1024 9.4 and 6.6
    constexpr int TURN = THREADS * unroll<TI, V>();
    a.tokens = 1;
    auto used = [&](int t) { return (double)t * a.per_token / ((t * a.per_token + TURN - 1) / TURN * TURN); };
    if (a.n >= 4096)
        for (int t = 2; t <= 8 && t * pairs <= THREADS; t++)
            if (used(t) >= used(a.tokens)) a.tokens = t;
    a.token_mul = multiplier(a.per_token, (uint64_t)a.tokens * a.per_token);
    a.head_mul = multiplier(a.per_head, a.per_token);
    a.pair_mul = multiplier(pairs, (uint64_t)a.tokens * pairs);
    hipLaunchKernelGGL((k_rotary<TI, TO, V>), dim3((a.n + a.tokens - 1) / a.tokens), dim3(THREADS), (size_t)a.tokens * pairs * 8, st, a);
    return l3m_dev_launched("k_rotary");
}
template <class TI, class TO> int launch_wide(const RotaryIn &a, bool wide, hipStream_t st) { return wide ? launch<TI, TO, 8>(a, st) : launch<TI, TO, 1>(a, st); }

}  // namespace

extern "C" {

int l3m_rotary_init(l3m_rotary *r, int hd, int rd, int halves, double theta, int scaling, double factor, double low, double high, int trained) {
    if (!r) return l3m_dev_fail("rotary: no plan");
    if (hd < 1 || hd > L3M_ROTARY_HD || rd < 0 || rd > hd || rd % 2) return l3m_dev_fail("rotary: a head of 1 to 256 values, of which an even number turn");
    if (!(theta > 0 && theta < INFINITY)) return l3m_dev_fail("rotary: the base must be positive");
    if (scaling < L3M_ROTARY_PLAIN || scaling > L3M_ROTARY_TURNS) return l3m_dev_fail("rotary: unknown scaling");
    if (scaling != L3M_ROTARY_PLAIN && !(factor >= 1 && factor < INFINITY)) return l3m_dev_fail("rotary: the factor must be 1 or more");
    if (scaling >= L3M_ROTARY_INDEX && !(low > 0 && high > low && high < INFINITY && trained >= 1))
        return l3m_dev_fail("rotary: turns 0 < low < high over a trained context of 1 or more positions");
    if (scaling == L3M_ROTARY_INDEX && !(theta > 1)) return l3m_dev_fail("rotary: scaling by index needs a base above 1");
    if (scaling == L3M_ROTARY_BASE && rd == 2) return l3m_dev_fail("rotary: scaling of the base needs more than one pair");
    const long double two_pi = 6.283185307179586476925286766559L;
    const long double base = scaling == L3M_ROTARY_BASE ? (long double)theta * powl(factor, (long double)rd / (rd - 2)) : (long double)theta;
    r->hd = hd;
    r->rd = rd;
    r->halves = halves != 0;
    r->mag = scaling == L3M_ROTARY_INDEX ? (float)(0.1 * log(factor) + 1) : 1.f;
    long double a = 0, b = 0;
    if (scaling == L3M_ROTARY_INDEX && rd) {
        a = floorl(rd * logl(trained / (high * two_pi)) / (2 * logl(base)));
        b = ceill(rd * logl(trained / (low * two_pi)) / (2 * logl(base)));
        a = a > 0 ? a : 0;
        b = b < rd - 1 ? b : rd - 1;
        b = b - a > 0.001L ? b : a + 0.001L;
    }
    for (int i = 0; i < L3M_ROTARY_HD / 2; i++) {
        long double f = i < rd / 2 ? powl(base, -2.0L * i / rd) : 0;
        if (scaling == L3M_ROTARY_LINEAR) f /= factor;
        else if (scaling == L3M_ROTARY_INDEX) {
            long double slow = (i - a) / (b - a);
            slow = slow < 0 ? 0 : slow > 1 ? 1 : slow;
            f = f * (1 - slow) + f / factor * slow;
        } else if (scaling == L3M_ROTARY_TURNS) {
            long double keep = (trained * f / two_pi - low) / (high - low);
            keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
            f = f * keep + f / factor * (1 - keep);
        }
        long double turns = f / two_pi;
        turns -= floorl(turns);
        r->turn[i] = (uint64_t)(turns * 18446744073709551616.0L + 0.5L);
    }
    return 0;
}

int l3m_k_rotary(const l3m_rotary *r, void *q, int q_stride, void *k, int k_stride, int out_dtype, const void *rows, int stride, int dtype, int n, int nq, int nkv,
                 const int32_t *pos, int pos0, void *stream) {
    if (!r || r->hd < 1 || r->hd > L3M_ROTARY_HD || r->rd < 0 || r->rd > r->hd || r->rd % 2) return l3m_dev_fail("rotary: not a plan (l3m_rotary_init)");
    const size_t in = value_bytes(dtype), out = value_bytes(out_dtype);
    if (!in || !out) return l3m_dev_fail("rotary: rows and outputs are f32 or bf16");
    if (n < 0 || n > 1 << 28 || nq < 0 || nkv < 0 || nq > 65536 || nkv > 65536 || nq + nkv < 1) return l3m_dev_fail("rotary: counts out of range");
    const long long qw = (long long)nq * r->hd, kw = (long long)nkv * r->hd;
    if (stride < qw + kw || (nq && q_stride < qw) || (nkv && k_stride < kw)) return l3m_dev_fail("rotary: a row holds fewer values than its heads");
    if (!n) return 0;
    if (!rows || (nq && !q) || (nkv && !k)) return l3m_dev_fail("rotary: no rows, or no output");
    if (!nq) q = nullptr;
    if (!nkv) k = nullptr;
    if ((uintptr_t)rows % in || ((uintptr_t)q | (uintptr_t)k) % out || (uintptr_t)pos % 4) return l3m_dev_fail("rotary: rows, outputs and positions must be aligned to their values");
    if (!pos && (pos0 < 0 || pos0 > INT_MAX - n)) return l3m_dev_fail("rotary: positions out of range");
    const char *x = (const char *)rows;
    const size_t xb = rows_bytes(n, stride, qw + kw, in), qb = rows_bytes(n, q_stride, qw, out), kb = rows_bytes(n, k_stride, kw, out);
    // an output lies apart from the rows or is the rows' own heads
    const bool q_in = in == out && q == rows && (q_stride == stride || n == 1), k_in = in == out && k == x + qw * in && (k_stride == stride || n == 1);
    if ((!q_in && overlap(q, qb, x, xb)) || (!k_in && overlap(k, kb, x, xb))) return l3m_dev_fail("rotary: an output overlaps the rows and is not the rows' own heads");
    // q and k apart, or columns of the same rows
    const long long gap = ((const char *)k - (const char *)q) / (long long)out;
    const bool columns = q_stride == k_stride && (gap >= 0 ? gap >= qw && gap + kw <= q_stride : -gap >= kw && qw - gap <= q_stride);
    if (!columns && overlap(q, qb, k, kb)) return l3m_dev_fail("rotary: q overlaps k");
    if (overlap(q, qb, pos, 4 * (size_t)n) || overlap(k, kb, pos, 4 * (size_t)n)) return l3m_dev_fail("rotary: an output overlaps the positions");
    const RotaryIn a = {*r, rows, q, k, pos, stride, q_stride, k_stride, n, nq, nkv, pos0, 0, 0, 0, 0, 0, 0, 0, 0};
    hipStream_t st;
    if (!stream_of(stream, st)) return -1;
    const bool wide = r->hd % 8 == 0 && r->rd % (r->halves ? 16 : 8) == 0 && stride % 8 == 0 && (!q || q_stride % 8 == 0) && (!k || k_stride % 8 == 0) &&
                      ((uintptr_t)rows | (uintptr_t)q | (uintptr_t)k) % 16 == 0;
    if (dtype == L3M_HIP_F32) return out_dtype == L3M_HIP_F32 ? launch_wide<float, float>(a, wide, st) : launch_wide<float, uint16_t>(a, wide, st);
    return out_dtype == L3M_HIP_F32 ? launch_wide<uint16_t, float>(a, wide, st) : launch_wide<uint16_t, uint16_t>(a, wide, st);
}

}
