"""The paged 8-bit K/V cache: the writer and the read-back against the formats' definition, the attention against its formula in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import l3m_amd as A
from serve import BLOCK, PAGE, Blocks, attended, bf16, from_bf16, typed, values

pytestmark = pytest.mark.gpu
DTYPES = pytest.mark.parametrize("dtype", ["f32", "bf16"])


@pytest.fixture(autouse=True)
def clean(dev):
    yield
    dev.free_all()


class Cache:
    """A cache of a few layers with its tables, and what its sequences hold by the definition."""

    def __init__(self, dev, seqs, nkv, hd, pages=40, width=12, layers=2, seed=0):
        self.dev, self.c, self.p = dev, dev.kv8(pages, layers, nkv, hd), dev.pages(pages, seqs, width)
        self.nkv, self.hd, self.rng, self.layer = nkv, hd, np.random.default_rng(seed), layers - 1
        # what memory holds before it is written: NaN codes and scales
        size = dev.lib.l3m_kv8_bytes(pages, layers, nkv, hd)
        before = np.full(size, 255, np.uint8)
        assert dev.lib.l3m_dev_upload(self.c.mem, C.c_void_p(before.ctypes.data), size) == 0
        self.held = {(s, kv, h): Blocks(hd) for s in range(seqs) for kv in (0, 1) for h in range(nkv)}

    def rows(self, n, dtype, size=1.0):
        x = self.rng.standard_normal((2, n, self.nkv, self.hd)) * size * np.exp(self.rng.standard_normal((2, 1, self.nkv, self.hd)))
        return [typed(y, dtype) for y in x]

    def add(self, ids, counts, dtype="f32", size=1.0, rows=None):
        (k, kx), (v, vx) = rows or self.rows(sum(counts), dtype, size)
        starts = np.cumsum([0] + list(counts))
        b = self.dev.batch(starts, ids)
        self.dev.pages_grow(self.p, self.c, b)
        self.dev.kv8_append(self.c, self.p, self.layer, k, v, b)
        for i, s in enumerate(ids):
            for h in range(self.nkv):
                for kv, x in ((0, kx), (1, vx)):
                    self.held[s, kv, h].add(x[starts[i]:starts[i + 1], h])
        return b

    def want(self, s, kv):
        return np.stack([self.held[s, kv, h].x for h in range(self.nkv)], 1)

    def check(self, ids):
        counts = [len(self.held[s, 0, 0].x) for s in ids]
        k, v = self.dev.kv8_rows(self.c, self.p, self.layer, self.dev.batch(np.cumsum([0] + counts), ids))
        for got, kv in ((k, 0), (v, 1)):
            with np.errstate(over="ignore"):                          # 256 2^120, which 3.4e38 is rounded to, is no float32: infinity
                want = np.float32(np.concatenate([self.want(s, kv) for s in ids]))
            bad = (got != want) & ~(np.isnan(got) & np.isnan(want))
            assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5])


# ---------------------------------------------------------------- writer and read-back

@DTYPES
@pytest.mark.parametrize("hd", [8, 32, 40, 64, 80, 96, 128, 160, 200, 256])
def test_append_rows(dev, dtype, hd):
    """Prompts and single rows at all places of a block; values that grow, so that scales rise and old codes are rounded again."""
    o = Cache(dev, 3, 2, hd, seed=hd)
    o.add([2, 0], [70, 1], dtype)
    o.add([0, 1, 2], [1, 33, 5], dtype, 3.0)
    for size in (0.1, 10.0, 1.0, 300.0, 1e-3):
        o.add([1, 0], [1, 2], dtype, size)
    o.add([2, 1], [150, 91], dtype, 0.5)
    o.add([0], [129], dtype)
    o.check([0, 1, 2])
    o.check([2])


def test_append_extremes(dev):
    """Zeros; the smallest and largest values; scales at their ends; NaN and infinities, which are their own positions' alone; values on borders."""
    o = Cache(dev, 1, 2, 16)
    f = np.float32
    x = np.zeros((2, 8, 2, 16), f)
    x[0, 0] = 0
    x[0, 1, 0] = 1e-45
    x[0, 2, 0] = 2.0 ** -133
    x[0, 3, 1] = 3.4e38
    x[0, 4, 1] = -3.4e38
    x[1, 0, 0] = np.linspace(-448, 448, 16)
    x[1, 1, 0] = 448 * 2.0 ** -np.arange(16)
    x[1, 2, 1, :4] = [np.nan, np.inf, -np.inf, 1]
    x[1, 3, 1] = 2.0 ** -10 * np.arange(16)
    for i in range(8):
        o.add([0], [1], rows=[(y[i:i + 1], y[i:i + 1]) for y in x])
    o.check([0])
    steps = np.concatenate([[(2 * i + 1) * 2.0 ** e for i in range(8, 16)] for e in range(-14, 4)] + [[448.0, 2.0 ** -10, 3 * 2.0 ** -10]])    # ties between codes
    y = np.zeros((2, BLOCK - 8, 2, 16), f)
    y.reshape(2, -1)[:, :len(steps)] = steps
    o.add([0], [BLOCK - 8], rows=[(z, z) for z in y])
    o.add([0], [3], rows=[(z, z) for z in np.float32(np.random.default_rng(0).standard_normal((2, 3, 2, 16)))])
    o.check([0])


def test_append_strides_layers_and_bounds(dev):
    """Rows inside wider ones; another layer and other pages keep their bytes, and so does all memory behind a sequence's last block."""
    nkv, hd = 3, 24
    c, p = dev.kv8(8, 3, nkv, hd), dev.pages(8, 3, 4)
    size = dev.lib.l3m_kv8_bytes(8, 3, nkv, hd)
    marks = np.random.default_rng(5).integers(0, 256, size, dtype=np.uint8)
    assert dev.lib.l3m_dev_upload(c.mem, C.c_void_p(marks.ctypes.data), size) == 0
    b = dev.batch([0, 40, 41], [2, 0])
    dev.pages_grow(p, c, b)
    x = np.random.default_rng(6).standard_normal((41, 200)).astype(np.float32)
    d = dev.put(x)
    assert dev.lib.l3m_k_kv8_append(C.byref(c), C.byref(p), 1, d + 4, d + 4 * 100, 200, A.F32, C.byref(b), None) == 0
    k, v = dev.kv8_rows(c, p, 1, b)
    for got, at in ((k, 1), (v, 100)):
        for lo, hi in ((0, 32), (32, 40), (40, 41)):
            for h in range(nkv):
                want = Blocks(hd)
                want.add(x[lo:hi, at + h * hd:at + (h + 1) * hd])
                assert np.array_equal(got[lo:hi, h], want.x)
    page = dev.lib.l3m_kv8_page_bytes(3, nkv, hd)
    got, was = (m.reshape(8, 3, page // 3) for m in (dev.get(c.mem, size, np.uint8), marks))
    assert np.array_equal(got[2:], was[2:]) and np.array_equal(got[:, 0], was[:, 0]) and np.array_equal(got[:, 2], was[:, 2])
    for n, pg in ((40, 0), (1, 1)):
        g, w = (m[pg, 1, :nkv * 256 * 32].reshape(nkv, 2, 4096) for m in (got, was))
        keys, vals = ([m[:, i].reshape(nkv, *shape) for m in (g, w)] for i, shape in ((0, (128, 32)), (1, (32, 128))))
        assert np.array_equal(keys[0][:, n:], keys[1][:, n:]) and np.array_equal(vals[0][:, :, -(-n // 4) * 4:], vals[1][:, :, -(-n // 4) * 4:])


def test_bad_pages_and_sequences(dev):
    """Table entries that are no page: reads are NaN, writes do nothing. Numbers that are no sequence and lengths past the table: nothing is out of bounds."""
    o = Cache(dev, 2, 1, 32, pages=6, width=3)
    o.add([0, 1], [200, 100])
    table = dev.get(o.p.table, (2, 3), np.int32)
    before = dev.get(o.c.mem, dev.lib.l3m_kv8_bytes(6, 2, 1, 32), np.uint8)
    for bad in (-1, 6, 2 ** 31 - 1, -2 ** 31):
        t = table.copy()
        t[0, 1] = bad
        assert dev.lib.l3m_dev_upload(o.p.table, C.c_void_p(t.ctypes.data), t.nbytes) == 0
        b = dev.batch([0, 200, 300], [0, 1])
        k, v = dev.kv8_rows(o.c, o.p, 1, b)
        assert np.isnan(k[128:200]).all() and np.isnan(v[128:200]).all() and np.array_equal(k[:128, 0], o.held[0, 0, 0].x[:128]) and np.isfinite(v[200:]).all()
        q = np.ones((2, 2, 32), np.float32)
        out = dev.kv8_attend(o.c, o.p, 1, q, dev.batch([0, 1, 2], [0, 1]))
        assert np.isnan(out[0]).all() and np.isfinite(out[1]).all()
        dev.kv8_append(o.c, o.p, 1, *(np.ones((72, 1, 32), np.float32) for _ in range(2)), dev.batch([0, 72], [0]))
        assert np.array_equal(dev.get(o.c.mem, before.shape, np.uint8), before)
    assert dev.lib.l3m_dev_upload(o.p.table, C.c_void_p(table.ctypes.data), table.nbytes) == 0
    out = dev.kv8_attend(o.c, o.p, 1, np.ones((3, 1, 32), np.float32), dev.batch([0, 1, 2, 3], [5, -1, 1]))
    assert np.all(out[:2] == 0) and np.isfinite(out[2]).all()
    lens = np.int32([1 << 30, -5])
    assert dev.lib.l3m_dev_upload(o.p.len, C.c_void_p(lens.ctypes.data), 8) == 0
    out = dev.kv8_attend(o.c, o.p, 1, np.ones((2, 1, 32), np.float32), dev.batch([0, 1, 2], [0, 1]))
    assert np.isnan(out[0]).all() and np.all(out[1] == 0)


# ---------------------------------------------------------------- attention

def attend(o, ids, counts, nq, dtype, longest=0, size=1.0, q=None, held=lambda x: x):
    """The cache's attention and its error's bound."""
    n = sum(counts)
    q, qx = q or typed(o.rng.standard_normal((n, nq, o.hd)) * size, dtype)
    starts = np.cumsum([0] + list(counts))
    got = values(o.dev.kv8_attend(o.c, o.p, o.layer, q, o.dev.batch(starts, ids), longest))
    f32 = dtype == "f32"
    for i, s in enumerate(ids):
        k, v = (held(o.want(s, kv)) for kv in (0, 1))
        rows = slice(starts[i], starts[i + 1])
        seen = [len(k) - counts[i] + t + 1 for t in range(counts[i])]
        # weights in three parts of bf16 are off by 2^-24 of themselves, in two by 2^-16; one below 2^-126 of the largest may be zero
        want, tol = attended(qx[rows], k, v, seen, 2.0 ** -24 if f32 else 2.0 ** -16, 2.0 ** -126, 2.0 ** -24 if f32 else 0.0)
        if not f32:
            tol = tol + 2.0 ** -8 * (np.abs(want) + tol)
        off = np.abs(got[rows] - want) - tol
        assert np.all(off <= 0), (s, off.max(), np.abs(want).max())
    return got


@DTYPES
@pytest.mark.parametrize("hd", [8, 32, 40, 64, 80, 96, 128, 160, 192, 224, 256])
def test_attend_heads(dev, dtype, hd):
    """Head sizes, one or several query heads a kv head, lengths from one to several pages, ragged."""
    for nkv, g in ((1, 1), (2, 3), (1, 8), (1, 17)):
        o = Cache(dev, 6, nkv, hd, seed=hd + g)
        o.add([0, 1, 2, 3, 4, 5], [1, 31, 128, 129, 300, 700], dtype)
        attend(o, [4, 0, 3, 1, 2, 5], [1] * 6, nkv * g, dtype)
        attend(o, [5, 2, 4], [9, 5, 2], nkv * g, dtype, longest=700)
        dev.free_all()


@DTYPES
def test_attend_long(dev, dtype):
    """Long sequences beside short ones, in one batch, so that the work of one is split over workgroups and that of another is not."""
    o = Cache(dev, 8, 2, 64, pages=260, width=200, seed=1)
    o.add([0, 1, 2, 3, 4], [20011, 5, 3001, 128, 900], dtype)
    for longest in (0, 20011):
        attend(o, [1, 0, 2, 3, 4], [1, 1, 1, 1, 1], 8, dtype, longest)
    attend(o, [0], [1], 8, dtype)
    attend(o, [2, 0, 1], [40, 3, 2], 8, dtype)
    attend(o, [3, 4, 3], [1, 0, 1], 8, dtype)                        # the same sequence twice, one without rows


@DTYPES
def test_attend_sizes(dev, dtype):
    """Queries and keys so large that one position takes all the weight, and so small that all take the same; values of very different sizes."""
    o = Cache(dev, 2, 1, 64, seed=2)
    o.add([0], [200], dtype, 1e-3)
    o.add([0], [100], dtype, 30.0)
    for size in (1e-30, 1e-3, 1.0, 100.0):
        attend(o, [0], [4], 2, dtype, size=size)
    q = np.zeros((2, 2, 64), np.float32)
    q[1, 0, 5], q[1, 1] = 1e4, 2.0 ** -np.arange(64)
    attend(o, [0], [2], 2, dtype, q=typed(q, dtype))


def test_attend_parts(dev):
    """float32: a relative error that two parts of the queries or the weights, 2^-16 of each value, do not reach."""
    o = Cache(dev, 1, 1, 128, seed=3)
    o.add([0], [500])
    q = o.rng.standard_normal((1, 16, 128)).astype(np.float32)
    got = o.dev.kv8_attend(o.c, o.p, 1, q, dev.batch([0, 1], [0]))
    want, _ = attended(q, o.want(0, 0), o.want(0, 1), [500], 0, 0)
    assert np.linalg.norm(got - want) < 2.0 ** -20 * np.linalg.norm(want)


@DTYPES
def test_attend_not_finite(dev, dtype):
    """NaN and infinities of keys, values and queries reach the rows that see them and change no bit of the others."""
    nkv, hd, n = 2, 48, 270
    rng = np.random.default_rng(4)
    x = [rng.standard_normal((n, nkv, hd)).astype(np.float32) for _ in range(2)]
    q = typed(rng.standard_normal((12, 4, hd)), dtype)[0]
    outs = []
    for what in ("none", "k", "v", "both"):
        y = [z.copy() for z in x]
        if what in ("k", "both"):
            y[0][263, 0, 7] = np.nan
        if what in ("v", "both"):
            y[1][266, 1, 3] = np.inf
            y[1][268, 1, 9] = np.nan
        o = Cache(dev, 1, nkv, hd)
        o.add([0], [n], rows=[(z, z) for z in y])
        outs.append(values(dev.kv8_attend(o.c, o.p, 1, q, dev.batch([0, 12], [0]))))
    # a value that is not finite is left out of its block's scale: here the others' scales stay, for none of them was the largest
    none, k, v, both = outs
    assert np.array_equal(k[:5], none[:5]) and np.array_equal(k[:, 2:], none[:, 2:]) and np.isnan(k[5:, :2]).all()
    assert np.array_equal(v[:8], none[:8]) and np.array_equal(v[:, :2], none[:, :2]) and np.isnan(v[8:, 2:, 3]).all() and np.isnan(v[10:, 2:, 9]).all()
    keep = np.ones(hd, bool)
    keep[[3, 9]] = False
    assert np.array_equal(v[:, 2:][..., keep], none[:, 2:][..., keep]) and np.array_equal(v[:10, 2:, 9], none[:10, 2:, 9])
    assert np.isnan(both[5:, :2]).all() and np.array_equal(both[:5], none[:5])
    bad = values(q).copy()
    bad[3, 1, 5], bad[4, 2, 0] = np.nan, np.inf
    o = Cache(dev, 1, nkv, hd)
    o.add([0], [n], rows=[(z, z) for z in x])
    got = values(dev.kv8_attend(o.c, o.p, 1, typed(bad, dtype)[0], dev.batch([0, 12], [0])))
    assert np.isnan(got[3, 1]).all() and np.isnan(got[4, 2]).all()
    got[3, 1], got[4, 2] = none[3, 1], none[4, 2]
    assert np.array_equal(got, none)


@DTYPES
def test_attend_rows(dev, dtype):
    """Strided queries and outputs, out in q's place, rows of no run and what lies between rows left as they were; rows before the first position are zeros."""
    o = Cache(dev, 3, 2, 40, seed=5)
    o.add([0, 1, 2], [2, 150, 33], dtype)
    n, nq, hd, gap = 12, 4, 40, 24
    q, qx = typed(o.rng.standard_normal((n, nq * hd + gap)), dtype)
    b = dev.batch([1, 5, 7, 9], [0, 1, 2], n=n)                      # four rows of a sequence of two positions
    dense = np.ascontiguousarray(q[:, :nq * hd]).reshape(n, nq, hd)
    size = dev.lib.l3m_kv8_work_bytes(C.byref(o.c), n, nq)
    code, work = A.F32 if dtype == "f32" else A.BF16, dev.alloc(size)
    p = dev.put(q)
    assert dev.lib.l3m_k_kv8_attend(p, nq * hd + gap, p, nq * hd + gap, code, C.byref(o.c), C.byref(o.p), 1, C.byref(b), nq, 0, work, size, None) == 0
    got = dev.get(p, q.shape, q.dtype)
    assert np.array_equal(got[:, nq * hd:], q[:, nq * hd:]) and np.array_equal(got[[0, 9, 10, 11]], q[[0, 9, 10, 11]])
    want = dev.kv8_attend(o.c, o.p, 1, dense, b)
    assert np.array_equal(got[1:9, :nq * hd], want[1:9].reshape(8, -1)) and np.all(values(want)[1:3] == 0) and np.all(values(want)[3:9] != 0)


def test_attend_behind_a_failed_call(dev):
    """A batch that found no room is not attended: NaN, and its append writes nothing."""
    o = Cache(dev, 2, 1, 32, pages=2, width=8)
    o.add([0], [200])
    before = dev.get(o.c.mem, dev.lib.l3m_kv8_bytes(2, 2, 1, 32), np.uint8)
    b = dev.batch([0, 100], [1])
    dev.pages_grow(o.p, o.c, b)
    dev.kv8_append(o.c, o.p, 1, *(np.ones((100, 1, 32), np.float32) for _ in range(2)), b)
    assert np.array_equal(dev.get(o.c.mem, before.shape, np.uint8), before)
    assert np.isnan(dev.kv8_attend(o.c, o.p, 1, np.ones((100, 1, 32), np.float32), b)).all()
    dev.pages_clear(o.p)
    attend(o, [0], [1], 1, "f32")


def test_far_page(dev):
    """A page that lies past 4 GiB of the pool: rows written, copied and attended there."""
    nkv, hd, layers = 8, 128, 8
    pages = (5 << 30) // dev.lib.l3m_kv8_page_bytes(layers, nkv, hd)
    c, p = dev.kv8(pages, layers, nkv, hd), dev.pages(pages, 2, pages)
    t = np.full((2, pages), -1, np.int32)
    t[0, :2] = pages - 1, pages - 3
    lens, refs = np.int32([130, 0]), np.ones(pages, np.int32)
    refs[pages - 2] = 0
    for at, x in ((p.table, t), (p.len, lens), (p.refs, refs)):
        assert dev.lib.l3m_dev_upload(at, C.c_void_p(x.ctypes.data), x.nbytes) == 0
    rng = np.random.default_rng(7)
    x = [rng.standard_normal((130, nkv, hd)).astype(np.float32) for _ in range(2)]
    b = dev.batch([0, 130], [0])
    dev.kv8_append(c, p, layers - 1, *x, b)
    dev.pages_fork(p, [0], [1])
    dev.pages_grow(p, c, dev.batch([0, 1], [1]))                     # its second page to the one that is free
    assert list(dev.get(p.table, (2, pages), np.int32)[1, :2]) == [pages - 1, pages - 2]
    dev.pages_cut(p, [1], [130])
    got = [dev.kv8_rows(c, p, layers - 1, dev.batch([0, 130], [s])) for s in (0, 1)]
    for kv in (0, 1):
        assert np.array_equal(got[0][kv], got[1][kv])
        for h in range(nkv):
            want = Blocks(hd)
            want.add(x[kv][:, h])
            assert np.array_equal(got[0][kv][:, h], want.x)
    q = rng.standard_normal((1, nkv, hd)).astype(np.float32)
    out = dev.kv8_attend(c, p, layers - 1, q, dev.batch([0, 1], [1]))
    want, tol = attended(q, got[1][0], got[1][1], [130], 2.0 ** -24, 2.0 ** -126, 2.0 ** -24)
    assert np.all(np.abs(out - want) <= tol)


def test_attend_much_work(dev):
    """Groups of rows times tiles past 2^25: a table that names the same page 2^19 times. Nothing is written behind the workspace."""
    nkv, hd, g, n, width = 1, 8, 16, 128, 1 << 19
    c, p = dev.kv8(2, 1, nkv, hd), dev.pages(2, 2, width)
    rng = np.random.default_rng(8)
    x = [rng.standard_normal((PAGE, nkv, hd)).astype(np.float32) for _ in range(2)]
    b = dev.batch([0, PAGE], [0])
    dev.pages_grow(p, c, b)
    dev.kv8_append(c, p, 0, *x, b)
    k, v = dev.kv8_rows(c, p, 0, b)
    table, lens = np.zeros((2, width), np.int32), np.int32([PAGE, PAGE * width])
    for at, y in ((p.table, table), (p.len, lens)):
        assert dev.lib.l3m_dev_upload(at, C.c_void_p(y.ctypes.data), y.nbytes) == 0
    q = rng.standard_normal((n, g, hd)).astype(np.float32)
    size = dev.lib.l3m_kv8_work_bytes(C.byref(c), n, g)
    marks = np.full(size // 4 + 4096, 7.0, np.float32)
    work, out, b = dev.put(marks), dev.alloc(q.nbytes), dev.batch([0, n], [1])
    assert dev.lib.l3m_k_kv8_attend(out, g * hd, dev.put(q), g * hd, A.F32, C.byref(c), C.byref(p), 0, C.byref(b), g, 0, work, size, None) == 0
    assert np.all(dev.get(work, marks.shape, np.float32)[size // 4:] == 7)
    # position i of the page counts `width` times, those behind the token once less. Four parts a group, four wavefronts a part, 16 positions a lane and tile:
    # sums of 2^20 terms, of the weights and of the values
    got, want, size = dev.get(out, q.shape, np.float32), np.zeros(q.shape), np.zeros(q.shape)
    z = np.einsum("tgd,id->tgi", q.astype(np.float64), k[:, 0].astype(np.float64)) / np.sqrt(hd)
    for t in range(n):
        w = np.exp(z[t] - z[t].max(1, keepdims=True)) * (width - (np.arange(PAGE) > t))
        w /= w.sum(1, keepdims=True)
        want[t], size[t] = w @ v[:, 0].astype(np.float64), w @ np.abs(v[:, 0].astype(np.float64))
    assert np.all(np.abs(got - want) <= 2.0 ** -3 * size)


def test_attend_runs_that_overlap(dev):
    """Starts that go up and down give runs over the same rows, more of them than rows: nothing is written behind the workspace or the rows."""
    o = Cache(dev, 70, 1, 32, pages=300, width=64, seed=9)
    o.add([0, 1], [8000, 3000])
    n, seqs, g = 64, 70, 4
    q = o.rng.standard_normal((n, g, 32)).astype(np.float32)
    b = dev.batch([0, n] * (seqs // 2) + [0], [i % 2 for i in range(seqs)], n=n)
    size = dev.lib.l3m_kv8_work_bytes(C.byref(o.c), n, g)
    work, out = dev.put(np.full(size // 4 + 4096, 7.0, np.float32)), dev.put(np.full(q.size + 4096, 7.0, np.float32))
    assert dev.lib.l3m_k_kv8_attend(out, g * 32, dev.put(q), g * 32, A.F32, C.byref(o.c), C.byref(o.p), 1, C.byref(b), g, 0, work, size, None) == 0
    assert np.all(dev.get(work, (size // 4 + 4096,), np.float32)[size // 4:] == 7) and np.all(dev.get(out, (q.size + 4096,), np.float32)[q.size:] == 7)


@DTYPES
def test_attend_split_of_many_runs(dev, dtype):
    """More runs than a wavefront has lanes, some of them split, some without rows; heads of 128 and 256; a length that is said to be less than it is."""
    o = Cache(dev, 150, 1, 128, pages=400, width=100, seed=10)
    counts = [int(x) for x in o.rng.choice([0, 1, 2, 40], 150)]
    counts[3], counts[77], counts[149] = 9001, 4000, 12000
    o.add(list(range(150)), counts, dtype)
    ids = [int(i) for i in o.rng.permutation(150)]
    rows = [min(counts[i], int(o.rng.choice([0, 1, 3]))) for i in ids]
    got = attend(o, ids, rows, 4, dtype, longest=12000)
    dev.free_all()
    o = Cache(dev, 2, 2, 256, pages=60, width=50, seed=11)
    o.add([0, 1], [6000, 70], dtype)
    q = typed(o.rng.standard_normal((2, 6, 256)), dtype)
    far = attend(o, [0, 1], [1, 1], 6, dtype, q=q)
    near = attend(o, [0, 1], [1, 1], 6, dtype, longest=1, q=q)
    assert got.size and far.shape == near.shape


@DTYPES
def test_attend_very_large_scores(dev, dtype):
    """Scores of 10^4 to 10^34, positive and negative, the largest ones apart by far or the same: one position takes all the weight, or several take equal parts."""
    hd, n = 64, 700
    rng = np.random.default_rng(12)
    for sign in (1, -1):
        o = Cache(dev, 1, 1, hd, seed=13)
        k = np.zeros((n, 1, hd), np.float32)
        k[:, 0, 5] = 2.0 ** -rng.integers(0, 8, n)                    # exactly held
        k[:, 0, 5][k[:, 0, 5] == (1 if sign > 0 else 2.0 ** -7)] = 2.0 ** -3
        best = [7, 133, 300, 690]
        k[best, 0, 5] = 1 if sign > 0 else 2.0 ** -7
        v = rng.standard_normal((n, 1, hd)).astype(np.float32)
        o.add([0], [n], rows=[(k, k), (v, v)])
        held = o.want(0, 1)[:, 0]
        for e in (20, 40, 70, 100, 113):
            q = np.zeros((20, 3, hd), np.float32)
            q[..., 5] = sign * 2.0 ** e * (1 + np.arange(3) / 4)
            got = values(o.dev.kv8_attend(o.c, o.p, o.layer, typed(q, dtype)[0], dev.batch([0, 20], [0])))
            for t in range(20):
                rows = held[[b for b in best if b <= n - 20 + t]]
                # weights are 1 or 0; sums of four, a quotient, and the rounding to bf16
                tol = 6 * 2.0 ** -24 * np.abs(rows).mean(0) + (2.0 ** -8 if dtype == "bf16" else 0) * (np.abs(rows.mean(0)) + 1e-6)
                assert np.all(np.abs(got[t] - rows.mean(0)) <= tol), (sign, e, t)
        dev.free_all()


def test_attend_largest_queries(dev):
    """float32's largest values as queries of keys so small that the scores are ordinary: bf16 has no value that near them."""
    o = Cache(dev, 1, 1, 32, seed=14)
    o.add([0], [90], size=2.0 ** -126)
    q = np.float32(o.rng.choice([-1, 1], (2, 4, 32)) * 3.4028e38)
    # what is held of them is taken as bf16, which is the same from 2^-126 up and in steps of 2^-133 below
    attend(o, [0], [2], 4, "f32", q=(q, q), held=lambda x: from_bf16(bf16(x)))


@DTYPES
def test_attend_lost_pages_are_their_rows(dev, dtype):
    """A page that is none takes the rows that see it and no others, whatever the cache's unwritten pages hold."""
    o = Cache(dev, 2, 1, 32, pages=6, width=3, seed=15)
    dev.pages_grow(o.p, o.c, dev.batch([0, 1], [1]))                 # page 0: never written
    o.add([0], [130], dtype)
    q, qx = typed(o.rng.standard_normal((4, 2, 32)), dtype)
    b = dev.batch([0, 4], [0])
    whole = values(dev.kv8_attend(o.c, o.p, 1, q, b))
    table = dev.get(o.p.table, (2, 3), np.int32)
    table[0, 1] = -1
    assert dev.lib.l3m_dev_upload(o.p.table, C.c_void_p(table.ctypes.data), table.nbytes) == 0
    got = values(dev.kv8_attend(o.c, o.p, 1, q, b))
    assert np.array_equal(got[:2], whole[:2]) and np.isnan(got[2:]).all()


@DTYPES
@pytest.mark.parametrize("nkv", [1, 3, 4])
def test_append_many_runs(dev, dtype, nkv):
    """More runs than lanes, some without rows, heads that are no multiple of a workgroup's wavefronts; then read back, some of K or V alone."""
    o = Cache(dev, 300, nkv, 24, pages=700, width=4, seed=16)
    counts = [int(x) for x in o.rng.choice([0, 1, 5, 33, 130], 300)]
    o.add([int(i) for i in o.rng.permutation(300)], counts, dtype)
    ids = [int(i) for i in o.rng.permutation(300)]
    o.add(ids, [1] * 300, dtype, 2.0)
    o.check(ids)
    n = len(o.held[ids[0], 0, 0].x)
    b = dev.batch([0, n], [ids[0]])
    for kv in (0, 1):
        out = dev.alloc(4 * n * nkv * 24)
        assert dev.lib.l3m_k_kv8_rows(C.byref(o.c), C.byref(o.p), 1, None if kv else out, out if kv else None, C.byref(b), None) == 0
        assert np.array_equal(dev.get(out, (n, nkv, 24), np.float32), np.float32(o.want(ids[0], kv)))


@DTYPES
def test_append_not_finite_beside_finite(dev, dtype):
    """A block of which one row holds NaN and infinities: the others' codes are what they are without it."""
    o = Cache(dev, 1, 2, 40, seed=17)
    (k, kx), (v, vx) = o.rows(70, dtype)
    bad = [x.copy() for x in (kx, vx)]
    bad[0][5, 0, 3], bad[0][40, 1, 39], bad[1][33, 1, 0], bad[1][69, 0, 8] = np.nan, -np.inf, np.inf, np.nan
    o.add([0], [70], rows=[(typed(x, dtype)[0], x) for x in bad])
    o.check([0])
