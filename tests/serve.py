"""What the tests of the kernels that serve many sequences share: bf16 and e4m3 in numpy, the formulas in 64 bits, and the tables as lists."""
import numpy as np

PAGE, BLOCK = 128, 32
E4M3 = np.array([np.nan if c == 127 else (1 + c % 8 / 8) * 2.0 ** (c // 8 - 7) if c >= 8 else c / 8 * 2.0 ** -6 for c in range(128)])


def bf16(x):
    """float32 to the nearest bf16, ties to even, as uint16; NaN stays NaN."""
    x = np.ascontiguousarray(x, np.float32)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + (u >> 16 & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bf16(u):
    return (np.asarray(u, np.uint16).astype(np.uint32) << 16).view(np.float32)


def typed(x, dtype):
    """float32 x as a call takes it (float32 or bf16 as uint16), and the values that stands for."""
    if dtype == "f32":
        return np.float32(x), np.float32(x)
    u = bf16(x)
    return u, from_bf16(u)


def values(x):
    return x if x.dtype == np.float32 else from_bf16(x)


def nearest_e4m3(x):
    """The e4m3 value nearest to each of x (64 bits, at most 448 in size), of two the one with an even code; NaN for what is not finite."""
    a = np.abs(np.where(np.isfinite(x), x, 0))
    hi = np.minimum(np.searchsorted(E4M3[:127], a), 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - E4M3[lo], E4M3[hi] - a
    y = E4M3[np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)]
    return np.where(np.isfinite(x), np.where(x < 0, -y, y), np.nan)


def unit(x):
    """The scale of a block that holds x: the smallest power of two, 2^-126 at least, by which its largest finite magnitude is at most 448."""
    m = np.abs(x[np.isfinite(x)]).max(initial=0)
    e = -126
    while m > 448 * 2.0 ** e:
        e += 1
    return 2.0 ** e


class Blocks:
    """One sequence's K or V of a kv head, block by block: rows added call by call."""

    def __init__(self, hd):
        self.x, self.u = np.zeros((0, hd)), []

    def add(self, rows):
        while len(rows):
            at = len(self.x) % BLOCK
            new, rows = rows[:BLOCK - at].astype(np.float64), rows[BLOCK - at:]
            if at == 0:
                self.u.append(unit(new))
            else:
                u = max(self.u[-1], unit(new))
                self.x[-at:] = nearest_e4m3(self.x[-at:] / u) * u
                self.u[-1] = u
            self.x = np.concatenate([self.x, nearest_e4m3(new / self.u[-1]) * self.u[-1]])

    def cut(self, n):
        self.x, self.u = self.x[:n], self.u[:-(-n // BLOCK)]


class Lists:
    """The tables as lists: what the calls do, one after the other."""

    def __init__(self, pages, seqs, width):
        self.refs, self.held, self.len, self.width, self.state = [0] * pages, [[] for _ in range(seqs)], [0] * seqs, width, "ok"

    def grow(self, ids, counts):
        """The rows' positions and the copies (from, to), or None."""
        if self.state != "ok":
            return None
        if len(set(ids)) < len(ids) or any(not 0 <= i < len(self.len) for i in ids):
            self.state = "bad"
            return None
        if any(self.len[i] + c > self.width * PAGE for i, c in zip(ids, counts)):
            self.state = "long"
            return None
        inside = [self.held[i][-1] if c and self.len[i] % PAGE else None for i, c in zip(ids, counts)]
        copy = [p is not None and self.refs[p] > 1 and not (inside.count(p) == self.refs[p] and inside.index(p) == n) for n, p in enumerate(inside)]
        need = [-(-(self.len[i] + c) // PAGE) - -(-self.len[i] // PAGE) + x for i, c, x in zip(ids, counts, copy)]
        free = [p for p, r in enumerate(self.refs) if r == 0]
        if sum(need) > len(free):
            self.state = "full"
            return None
        pos, copies = [], []
        for i, c, x, n in zip(ids, counts, copy, need):
            new, free = free[:n], free[n:]
            if x:
                copies.append((self.held[i][-1], new[0]))
                self.refs[self.held[i].pop()] -= 1
            self.held[i] += new
            for p in new:
                self.refs[p] = 1
            pos += range(self.len[i], self.len[i] + c)
            self.len[i] += c
        return pos, copies

    def fork(self, sources, to):
        if self.state != "ok":
            return
        if any(not 0 <= i < len(self.len) for i in [*sources, *to]) or len(set(to)) < len(to) or set(to) & set(sources) or any(self.len[i] for i in to):
            self.state = "bad"
            return
        for a, b in zip(sources, to):
            self.held[b], self.len[b] = list(self.held[a]), self.len[a]
            for p in self.held[a]:
                self.refs[p] += 1

    def cut(self, ids, keep=None):
        if self.state != "ok":
            return
        keep = keep if keep is not None else [0] * len(ids)
        if any(not 0 <= i < len(self.len) for i in ids) or len(set(ids)) < len(ids) or any(not 0 <= k <= self.len[i] for i, k in zip(ids, keep)):
            self.state = "bad"
            return
        for i, k in zip(ids, keep):
            for p in self.held[i][-(-k // PAGE):]:
                self.refs[p] -= 1
            self.held[i], self.len[i] = self.held[i][:-(-k // PAGE)], k

    def compact(self):
        if self.state != "ok":
            return []
        live = sum(r > 0 for r in self.refs)
        moves = list(zip([p for p in range(live, len(self.refs)) if self.refs[p]], [p for p in range(live) if not self.refs[p]]))
        to = dict(moves)
        self.held = [[to.get(p, p) for p in h] for h in self.held]
        for a, b in moves:
            self.refs[b], self.refs[a] = self.refs[a], 0
        return moves

    def check(self, got):
        """Against Device.pages_state."""
        assert got["state"] == self.state
        assert list(got["refs"]) == self.refs and list(got["len"]) == self.len
        assert got["used"] == sum(r > 0 for r in self.refs)
        assert [list(r) for r in got["table"]] == [h + [-1] * (self.width - len(h)) for h in self.held]


def attended(q, k, v, seen, rel, least, q_off=0.0, steps=None):
    """Attention of q [n][nq][hd] over k, v [positions][nkv][hd], row t over its first seen[t] positions, in 64 bits, and the bound of a float32 kernel's error.

    A score is a sum of hd products in float32, each step off by 2^-24 of the sum of the terms' magnitudes, and q is off by q_off of its row's largest; a
    weight by as much, the sum's again, and the exponential's 2^-21. rel: what a weight's rounding to fewer bits is off by, least: at the least, of the largest
    weight. And a float32 rounding of its terms for each step of the sums."""
    n, nq, hd = q.shape
    g = nq // k.shape[1]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for t in range(n):
        s = seen[t]
        if s <= 0:
            continue
        for h in range(nq):
            kh, vh, qh = (x.astype(np.float64) for x in (k[:s, h // g], v[:s, h // g], q[t, h]))
            z = kh @ qh / np.sqrt(hd)
            off = (((hd + 8) * 2.0 ** -24) * (np.abs(kh) @ np.abs(qh)) + q_off * np.abs(qh).max() * np.abs(kh).sum(1)).max() / np.sqrt(hd)
            p = np.exp(z - z.max())
            p /= p.sum()
            out[t, h] = p @ vh
            size = p @ np.abs(vh)
            tol[t, h] = (2 * off + 2.0 ** -21 + rel + (s if steps is None else steps) * 2.0 ** -24) * size + least * p.max() * np.abs(vh).sum(0) + 1e-42
    return out, tol
