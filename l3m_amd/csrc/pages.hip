// Who holds which page of a paged K/V cache, for CDNA4 (gfx950): sequences given room, forked, cut and freed, the pool compacted; shared pages are
// copied when a sequence writes behind them.
//
// The tables are small and their steps depend on each other, so one workgroup plans a call; the copies that the plan lists are a second launch over the
// whole card. Every result is the same whatever the order of the threads: pages are taken by ascending index in the list's order, and counts are
// sums of whole numbers. A call that cannot be done as a whole changes nothing and sets state[0], and until that is cleared every call that changes
// something does nothing.
//
// Measured: 8 sequences forked by 4 and all grown by a row, shared pages of 4 layers of 8 heads of 64 copied (34 MB), 20.5 us: three launches, the plans of 2 and
// 5 us (a chain of loads, scans and barriers), the copies 6.2. 700 pages half in use compacted (163 MB): 43 us, of which the plan 4 and the copies 33
// (4.9 TB/s).
#include "serve.h"

namespace {

constexpr int PLAN = 1024;                                           // threads of the planning workgroup, at the most
constexpr int MOST_SEQS = 65536;
enum { STATE_FAILED, STATE_USED, STATE_COPIES };

struct Tables {
    int32_t *refs, *table, *len, *state, *scratch;
    int      pages, seqs, width;
};
Tables tables_of(const l3m_pages *p) { return {p->refs, p->table, p->len, p->state, p->scratch, p->pages, p->seqs, p->width}; }
// The scratch: pages' ints [4][pages] (copies' sources, their destinations; two more that the calls name), then runs' [2][seqs].
__device__ __forceinline__ int32_t *scratch(const Tables &t, int plane) { return t.scratch + (size_t)plane * t.pages; }

__device__ __forceinline__ int pages_for(int n) { return (int)(((unsigned)n + PAGE - 1) / PAGE); }

// The sums of x over the threads before this one; total: over all. Every thread of the planning workgroup, T of them, calls it.
struct Scan {
    int sums[PLAN / 64];
};
template <int T = PLAN> __device__ int scan_all(Scan &s, int x, int &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, upto = scan_wave(x);
    __syncthreads();
    if (lane == 63) s.sums[wave] = upto;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < T / 64; w++) {
        before += w < wave ? s.sums[w] : 0;
        total += s.sums[w];
    }
    return before + upto - x;
}
// Numbers of sequences that were listed, a bit each; and the gravest reason against a call, 0: none.
struct Listed {
    uint32_t bits[MOST_SEQS / 32];
    int      why;
    template <int T = PLAN> __device__ void clear() {
        if (threadIdx.x == 0) why = 0;
        for (int i = threadIdx.x; i < MOST_SEQS / 32; i += T) bits[i] = 0;
        __syncthreads();
    }
    __device__ bool add(int id) { return !(atomicOr(&bits[id >> 5], 1u << (id & 31)) >> (id & 31) & 1u); }    // false: it was there
    __device__ bool has(int id) const { return bits[id >> 5] >> (id & 31) & 1u; }
    __device__ int worst(int mine) {
        if (mine) atomicMax(&why, mine);
        __syncthreads();
        return why;
    }
};
// f(v, 0 .. count - 1) of each thread's own count and values, over all threads of the workgroup alike.
template <int N> struct Spread {
    int first[PLAN], v[N][PLAN];
};
template <int N, int T = PLAN, class F> __device__ __forceinline__ void spread(Scan &scan, Spread<N> &s, int count, const int (&v)[N], F f) {
    int total;
    const int before = scan_all<T>(scan, count, total);
    s.first[threadIdx.x] = before;
#pragma unroll
    for (int i = 0; i < N; i++) s.v[i][threadIdx.x] = v[i];
    __syncthreads();
    for (int e = threadIdx.x; e < total; e += T) {
        int of = 0;                                                  // the last one that begins at e or before it
#pragma unroll
        for (int step = T / 2; step; step >>= 1) of += s.first[of + step] <= e ? step : 0;
        int u[N];
#pragma unroll
        for (int i = 0; i < N; i++) u[i] = s.v[i][of];
        f(u, e - s.first[of]);
    }
}
__device__ __forceinline__ bool in_pool(const Tables &t, int page) { return (unsigned)page < (unsigned)t.pages; }
// One workgroup's stores and atomics to memory are done, and every thread is here: they meet in one L2, so no fence beyond the workgroup is needed (an
// agent's writes that L2 back).
__device__ __forceinline__ void memory_done() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0x0F70);                              // vmcnt(0)
    __syncthreads();
}
// Values that this launch's atomics changed, past the CU's cache.
__device__ __forceinline__ int32_t now(const int32_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

__global__ void __launch_bounds__(256) k_pages_reset(Tables t) {
    const size_t entries = (size_t)t.seqs * t.width, step = (size_t)gridDim.x * 256;
    for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < entries; i += step) {
        t.table[i] = -1;
        if (i < (size_t)t.seqs) t.len[i] = 0;
        if (i < STATE_INTS) t.state[i] = 0;
    }
    for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < (size_t)t.pages; i += step) t.refs[i] = 0;
    if (blockIdx.x == 0 && threadIdx.x < STATE_INTS) t.state[threadIdx.x] = 0;
}
__global__ void k_pages_clear(Tables t) { t.state[STATE_FAILED] = 0; }

// A run of `add` rows makes its sequence that much longer. The pages that it begins are new; one that it goes on in and that others hold too is replaced by
// a new one and listed to be copied, but where all of its holders are in the list the first of them keeps it.
// Bound by latency: each step's loads hang on the last one's. Up to T runs are read once and kept in registers. Steps of few rows meet sooner with
// fewer threads: 40 sequences a row each, forks and copies among them, 20.5 us by 256 threads, 22.5 by 1024; 80 of 200 rows each 45.5 and 32.9.
struct Grown {
    int id, s0, add, old, page, held;                                // page: that it goes on in, -1: none; held: by so many
    int more, copy, at;                                              // new pages, one of them a copy; where they begin among all
};
template <int T> __global__ void __launch_bounds__(T) k_pages_grow(Tables t, Runs b, int32_t *pos) {
    __shared__ Listed listed;
    __shared__ Scan   scan;
    __shared__ Spread<5> spread_s;
    __shared__ int    copies_s;
    const int tid = threadIdx.x, first_free = tid < t.pages ? t.refs[tid] : 1;
    int32_t *growers = scratch(t, 2), *eldest = scratch(t, 3), *fresh = eldest, *plan = scratch(t, 4);   // of a page: how many grow into it, and the first
    const int failed = t.state[STATE_FAILED];
    auto read = [&](int i) {
        Grown r = {b.id(i), b.from(i), 0, 0, -1, 0, 0, 0, 0};
        r.add = b.to(i, r.s0) - r.s0;
        if ((unsigned)r.id >= (unsigned)t.seqs) return r;
        r.old = t.len[r.id];
        if (r.add && r.old % PAGE && r.old > 0 && r.old <= (long long)t.width * PAGE) {
            r.page = t.table[(size_t)r.id * t.width + r.old / PAGE];
            r.held = in_pool(t, r.page) ? t.refs[r.page] : 0;
        }
        return r;
    };
    const bool one = b.seqs <= T;
    Grown mine = {};
    if (tid < b.seqs) mine = read(tid);
    if (failed) {
        if (tid == 0) t.state[STATE_COPIES] = 0;
        return;
    }
    listed.clear<T>();
    if (tid == 0) copies_s = 0;
    int why = 0, shared = 0;
    for (int i = tid; i < b.seqs; i += T) {
        const Grown r = one ? mine : read(i);
        if ((unsigned)r.id >= (unsigned)t.seqs || !listed.add(r.id) || r.old < 0 || r.old > (long long)t.width * PAGE) why = max(why, (int)L3M_PAGES_BAD);
        else if ((long long)r.old + r.add > (long long)t.width * PAGE) why = max(why, (int)L3M_PAGES_LONG);
        else if (r.add && r.old % PAGE && !in_pool(t, r.page)) why = max(why, (int)L3M_PAGES_BAD);
        else if (r.held > 1) {
            shared = 1;
            growers[r.page] = 0;
            eldest[r.page] = INT_MAX;
        }
    }
    why = listed.worst(why);
    if (!why && __syncthreads_or(shared)) {
        memory_done();
        for (int i = tid; i < b.seqs; i += T) {
            const Grown r = one ? mine : read(i);
            if (r.held > 1) {
                atomicAdd(&growers[r.page], 1);
                atomicMin(&eldest[r.page], i);
            }
        }
        memory_done();
    }
    int total = 0;
    if (!why)
        for (int i0 = 0; i0 < b.seqs; i0 += T) {
            const int i = i0 + tid;
            Grown r = {};
            if (i < b.seqs) {
                r = one ? mine : read(i);
                r.copy = r.held > 1 && !(now(&growers[r.page]) == r.held && now(&eldest[r.page]) == i);
                r.more = pages_for(r.old + r.add) - pages_for(r.old) + r.copy;
            }
            int sum;
            r.at = scan_all<T>(scan, r.more, sum) + total;
            if (one) mine = r;
            else if (i < b.seqs) {
                plan[i] = r.at;
                plan[t.seqs + i] = 2 * r.more + r.copy;
            }
            total += sum;
            if (total > t.pages) break;                              // uniform; no pool has so many
        }
    // the free pages that are needed, in order
    if (!why && total) {
        __syncthreads();
        int got = 0;
        for (int p0 = 0; p0 < t.pages && got < total; p0 += T) {
            const int p = p0 + tid, free = p < t.pages && (p0 ? t.refs[p] : first_free) == 0;
            int sum;
            const int at = scan_all<T>(scan, free, sum);
            if (free && got + at < total) fresh[got + at] = p;       // who grows where is in the plan by now
            got += sum;
        }
        if (got < total) why = L3M_PAGES_FULL;
    }
    if (why) {
        if (tid == 0) {
            t.state[STATE_FAILED] = why;
            t.state[STATE_COPIES] = 0;
        }
        return;
    }
    __syncthreads();
    for (int i0 = 0; i0 < b.seqs; i0 += T) {
        const int i = i0 + tid;
        Grown r = {};
        int v[5] = {0, 0, 0, 0, 0};                                  // its first new page's place among them, sequence, place in the table, first row, length
        if (i < b.seqs) {
            r = one ? mine : read(i);
            if (!one) {
                r.at = plan[i];
                r.copy = plan[t.seqs + i] & 1;
                r.more = plan[t.seqs + i] >> 1;
            }
            v[0] = r.at;
            v[1] = r.id;
            v[2] = r.copy ? r.old / PAGE : pages_for(r.old);
            v[3] = r.s0;
            v[4] = r.old;
            if (r.copy) {
                const int k = atomicAdd(&copies_s, 1);
                atomicSub(&t.refs[r.page], 1);
                scratch(t, 0)[k] = r.page;
                scratch(t, 1)[k] = fresh[r.at];
            }
            t.len[r.id] = r.old + r.add;
        }
        spread<5, T>(scan, spread_s, r.more, v, [&](const int (&u)[5], int j) {
            const int page = fresh[u[0] + j];
            t.refs[page] = 1;
            t.table[(size_t)u[1] * t.width + u[2] + j] = page;
        });
        if (pos) spread<5, T>(scan, spread_s, r.add, v, [&](const int (&u)[5], int j) { pos[u[3] + j] = u[4] + j; });
    }
    __syncthreads();
    if (tid == 0) {
        t.state[STATE_USED] += total;
        t.state[STATE_COPIES] = copies_s;
    }
}

// to[i] becomes a sequence of from[i]'s pages.
__global__ void __launch_bounds__(PLAN) k_pages_fork(Tables t, const int32_t *from, const int32_t *to, int n) {
    __shared__ Listed listed;
    __shared__ Scan   scan;
    __shared__ Spread<2> spread_s;
    const int tid = threadIdx.x;
    // the first PLAN pairs are read once: number, number, lengths
    auto read = [&](int i, int (&v)[4]) {
        v[0] = from[i];
        v[1] = to[i];
        v[2] = (unsigned)v[0] < (unsigned)t.seqs ? t.len[v[0]] : -1;
        v[3] = (unsigned)v[1] < (unsigned)t.seqs ? t.len[v[1]] : -1;
    };
    int mine[4] = {0, 0, 0, 0};
    if (tid < n) read(tid, mine);
    if (t.state[STATE_FAILED]) return;
    listed.clear();
    int why = 0;
    for (int i = tid; i < n; i += PLAN) {
        int v[4] = {mine[0], mine[1], mine[2], mine[3]};
        if (i >= PLAN) read(i, v);
        if (v[2] < 0 || v[2] > (long long)t.width * PAGE || v[3] != 0 || !listed.add(v[1])) why = L3M_PAGES_BAD;
    }
    __syncthreads();
    for (int i = tid; i < n; i += PLAN) {
        const int id = i < PLAN ? mine[0] : from[i];
        if ((unsigned)id < (unsigned)t.seqs && listed.has(id)) why = L3M_PAGES_BAD;
    }
    if ((why = listed.worst(why))) {
        if (tid == 0) t.state[STATE_FAILED] = why;
        return;
    }
    for (int i0 = 0; i0 < n; i0 += PLAN) {
        const int i = i0 + tid;
        int v[4] = {mine[0], mine[1], mine[2], mine[3]};
        if (i0 && i < n) read(i, v);
        if (i < n) t.len[v[1]] = v[2];
        spread<2>(scan, spread_s, i < n ? pages_for(v[2]) : 0, {v[0], v[1]}, [&](const int (&u)[2], int j) {
            const int page = t.table[(size_t)u[0] * t.width + j];
            t.table[(size_t)u[1] * t.width + j] = page;
            if (in_pool(t, page)) atomicAdd(&t.refs[page], 1);
        });
    }
}

// Sequence ids[i] is cut to its first keep[i] positions (keep NULL: none).
__global__ void __launch_bounds__(PLAN) k_pages_cut(Tables t, const int32_t *ids, const int32_t *keep, int n) {
    __shared__ Listed listed;
    __shared__ Scan   scan;
    __shared__ Spread<2> spread_s;
    __shared__ int    freed_s;
    const int tid = threadIdx.x;
    if (t.state[STATE_FAILED]) return;
    listed.clear();
    if (tid == 0) freed_s = 0;
    int why = 0;
    for (int i = tid; i < n; i += PLAN) {
        const int id = ids[i], to = keep ? keep[i] : 0;
        if ((unsigned)id >= (unsigned)t.seqs || !listed.add(id) || to < 0 || to > t.len[id] || t.len[id] > (long long)t.width * PAGE) why = L3M_PAGES_BAD;
    }
    if ((why = listed.worst(why))) {
        if (tid == 0) t.state[STATE_FAILED] = why;
        return;
    }
    for (int i0 = 0; i0 < n; i0 += PLAN) {
        const int i = i0 + tid;
        int count = 0, v[2] = {0, 0};
        if (i < n) {
            v[0] = ids[i];
            const int to = keep ? keep[i] : 0;
            v[1] = pages_for(to);
            count = pages_for(t.len[v[0]]) - v[1];
            t.len[v[0]] = to;
        }
        spread<2>(scan, spread_s, count, v, [&](const int (&u)[2], int j) {
            int32_t &entry = t.table[(size_t)u[0] * t.width + u[1] + j];
            if (in_pool(t, entry) && atomicSub(&t.refs[entry], 1) == 1) atomicAdd(&freed_s, 1);
            entry = -1;
        });
    }
    __syncthreads();
    if (tid == 0) t.state[STATE_USED] -= freed_s;
}

// The pages in use behind the first `live` ones, by ascending index, into the free ones among those.
__global__ void __launch_bounds__(PLAN) k_pages_compact(Tables t) {
    __shared__ Scan scan;
    const int tid = threadIdx.x;
    int32_t *src = scratch(t, 0), *dst = scratch(t, 1), *map = scratch(t, 2);
    if (t.state[STATE_FAILED]) {
        if (tid == 0) t.state[STATE_COPIES] = 0;
        return;
    }
    int mine = 0, live;
    for (int p = tid; p < t.pages; p += PLAN) mine += t.refs[p] > 0;
    scan_all(scan, mine, live);
    int movers = 0, holes = 0;
    for (int p0 = 0; p0 < t.pages; p0 += PLAN) {
        const int p = p0 + tid, held = p < t.pages && t.refs[p] > 0, mover = held && p >= live, hole = p < live && !held;
        int sum;
        if (p0 < live) {
            const int at = scan_all(scan, hole, sum);
            if (hole) dst[holes + at] = p;
            holes += sum;
        }
        if (p0 + PLAN > live) {
            const int at = scan_all(scan, mover, sum);
            if (mover) src[movers + at] = p;
            movers += sum;
        }
        if (p < t.pages) map[p] = p;
    }
    __syncthreads();
    for (int k = tid; k < movers; k += PLAN) {
        map[src[k]] = dst[k];
        t.refs[dst[k]] = t.refs[src[k]];
        t.refs[src[k]] = 0;
    }
    if (tid == 0) t.state[STATE_COPIES] = movers;
}

// The copies that a plan listed, CHUNK bytes a workgroup at a time; and, where pages moved, the tables' entries. Bound by the bytes.
constexpr int CHUNK = 256 * 16 * 4;
__global__ void __launch_bounds__(256) k_pages_copy(Tables t, uint8_t *mem, size_t bytes, int moved) {
    const int copies = t.state[STATE_COPIES];
    const unsigned per = (unsigned)((bytes + CHUNK - 1) / CHUNK);
    const size_t items = (size_t)copies * per;
    for (size_t i = blockIdx.x; i < items; i += gridDim.x) {
        const unsigned k = (unsigned)(i / per), chunk = (unsigned)(i - (size_t)k * per);
        const uint8_t *from = mem + (size_t)scratch(t, 0)[k] * bytes;
        uint8_t *to = mem + (size_t)scratch(t, 1)[k] * bytes;
        const size_t at = (size_t)chunk * CHUNK + 16 * threadIdx.x;
        u32x4 x[4];
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (at + 4096 * j < bytes) x[j] = *(const u32x4 *)(from + at + 4096 * j);
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (at + 4096 * j < bytes) *(u32x4 *)(to + at + 4096 * j) = x[j];
    }
    if (moved && copies)
        for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < (size_t)t.seqs * t.width; i += (size_t)gridDim.x * 256) {
            const int page = t.table[i];
            if (in_pool(t, page)) {
                const int to = scratch(t, 2)[page];
                if (to != page) t.table[i] = to;
            }
        }
}

const char *list_bad(const l3m_pages *p, const int32_t *a, const int32_t *b, int n, bool need_b) {
    if (const char *why = pages_bad(p)) return why;
    if (n < 0 || n > p->seqs) return "pages: more sequences listed than there are";
    if (n && (!a || (need_b && !b))) return "pages: no list";
    if (((uintptr_t)a | (uintptr_t)b) % 4) return "pages: lists must be 4-byte aligned";
    if (on_pages(p, a, 4 * (size_t)n) || on_pages(p, b, 4 * (size_t)n)) return "pages: a list overlaps the tables";
    return nullptr;
}
// The copies are listed on the device: enough workgroups for the card, which end at once where there are none.
constexpr int COPY_WGS = 2048;
void launch_copy(const Tables &t, const l3m_kv8 *c, int moved, hipStream_t st) {
    hipLaunchKernelGGL(k_pages_copy, dim3(COPY_WGS), dim3(256), 0, st, t, c->mem, c->layers * layer_bytes(c->nkv, c->hd), moved);
}

}  // namespace

extern "C" {

size_t l3m_pages_bytes(int pages, int seqs, int width) {
    if (pages < 1 || pages > 1 << 20 || seqs < 1 || seqs > MOST_SEQS || width < 1 || width > 1 << 20 || (long long)seqs * width > 1 << 28) return 0;
    auto up = [](size_t ints) { return (4 * ints + 255) & ~(size_t)255; };
    return up(pages) + up((size_t)seqs * width) + up(seqs) + up(STATE_INTS) + up(scratch_ints(pages, seqs));
}

int l3m_pages_init(l3m_pages *p, int pages, int seqs, int width, void *mem) {
    if (!p || !mem || (uintptr_t)mem % 16) return l3m_dev_fail("pages: memory must be 16-byte aligned");
    if (!l3m_pages_bytes(pages, seqs, width)) return l3m_dev_fail("pages: pages up to 2^20, sequences up to 65536, pages of a sequence up to 2^20, 2^28 entries in all");
    auto up = [](size_t ints) { return (4 * ints + 255) & ~(size_t)255; };
    char *m = (char *)mem;
    p->refs = (int32_t *)m;
    p->table = (int32_t *)(m += up(pages));
    p->len = (int32_t *)(m += up((size_t)seqs * width));
    p->state = (int32_t *)(m += up(seqs));
    p->scratch = (int32_t *)(m + up(STATE_INTS));
    p->pages = pages;
    p->seqs = seqs;
    p->width = width;
    return 0;
}

int l3m_k_pages_reset(const l3m_pages *p, void *stream) {
    if (const char *why = pages_bad(p)) return l3m_dev_fail(why);
    hipStream_t st;
    if (!stream_of(stream, st)) return -1;
    const size_t entries = (size_t)p->seqs * p->width;
    hipLaunchKernelGGL(k_pages_reset, dim3((unsigned)(entries < 1 << 18 ? (entries + 255) / 256 : 1024)), dim3(256), 0, st, tables_of(p));
    return l3m_dev_launched("k_pages_reset");
}

int l3m_k_pages_clear(const l3m_pages *p, void *stream) {
    if (const char *why = pages_bad(p)) return l3m_dev_fail(why);
    hipStream_t st;
    if (!stream_of(stream, st)) return -1;
    hipLaunchKernelGGL(k_pages_clear, dim3(1), dim3(1), 0, st, tables_of(p));
    return l3m_dev_launched("k_pages_clear");
}

int l3m_k_pages_grow(const l3m_pages *p, const l3m_kv8 *c, const l3m_batch *b, int32_t *pos, void *stream) {
    if (const char *why = paged_bad(c, p)) return l3m_dev_fail(why);
    if (const char *why = batch_bad(b)) return l3m_dev_fail(why);
    if (b->seqs > p->seqs) return l3m_dev_fail("pages_grow: more runs than sequences");
    if (!b->seqs) return 0;
    const size_t mem = l3m_kv8_bytes(c->pages, c->layers, c->nkv, c->hd), pb = 4 * (size_t)b->n;
    if ((uintptr_t)pos % 4) return l3m_dev_fail("pages_grow: positions must be 4-byte aligned");
    if (on_pages(p, pos, pb) || on_cache(c, pos, pb) || on_batch(b, pos, pb)) return l3m_dev_fail("pages_grow: the positions overlap the tables, the cache or the batch");
    if (on_pages(p, b->starts, 4 * ((size_t)b->seqs + 1)) || on_pages(p, b->ids, 4 * (size_t)b->seqs) || on_batch(b, c->mem, mem))
        return l3m_dev_fail("pages_grow: the batch overlaps the tables or the cache");
    hipStream_t st;
    if (!stream_of(stream, st)) return -1;
    const Tables t = tables_of(p);
    if (b->seqs <= 256 && b->n <= 1024 && p->pages <= 4096) hipLaunchKernelGGL((k_pages_grow<256>), dim3(1), dim3(256), 0, st, t, runs_of(b), pos);
    else hipLaunchKernelGGL((k_pages_grow<PLAN>), dim3(1), dim3(PLAN), 0, st, t, runs_of(b), pos);
    launch_copy(t, c, 0, st);
    return l3m_dev_launched("k_pages_grow");
}

int l3m_k_pages_fork(const l3m_pages *p, const int32_t *from, const int32_t *to, int n, void *stream) {
    if (const char *why = list_bad(p, from, to, n, true)) return l3m_dev_fail(why);
    if (!n) return 0;
    hipStream_t st;
    if (!stream_of(stream, st)) return -1;
    hipLaunchKernelGGL(k_pages_fork, dim3(1), dim3(PLAN), 0, st, tables_of(p), from, to, n);
    return l3m_dev_launched("k_pages_fork");
}

int l3m_k_pages_cut(const l3m_pages *p, const int32_t *ids, const int32_t *keep, int n, void *stream) {
    if (const char *why = list_bad(p, ids, keep, n, false)) return l3m_dev_fail(why);
    if (!n) return 0;
    hipStream_t st;
    if (!stream_of(stream, st)) return -1;
    hipLaunchKernelGGL(k_pages_cut, dim3(1), dim3(PLAN), 0, st, tables_of(p), ids, keep, n);
    return l3m_dev_launched("k_pages_cut");
}

int l3m_k_pages_compact(const l3m_pages *p, const l3m_kv8 *c, void *stream) {
    if (const char *why = paged_bad(c, p)) return l3m_dev_fail(why);
    hipStream_t st;
    if (!stream_of(stream, st)) return -1;
    const Tables t = tables_of(p);
    hipLaunchKernelGGL(k_pages_compact, dim3(1), dim3(PLAN), 0, st, t);
    launch_copy(t, c, 1, st);
    return l3m_dev_launched("k_pages_compact");
}

}
