"""The paged 8-bit K/V cache (l3m_k_kv8_attend) where it can go wrong: values that read as infinities, and the forms of a call by its runs, rows and heads."""
import ctypes as C

import numpy as np
import pytest

import l3m_amd as A
from serve import PAGE, attended
from test_gpu_kv8 import DTYPES, Cache, attend, typed, values

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean(dev):
    yield
    dev.free_all()


@DTYPES
@pytest.mark.parametrize("longest", [0, 300, 100])
def test_attend_values_read_as_infinities(dev, dtype, longest):
    """Values next to float32's (or bf16's) largest, which are held as 256 2^120 and read as infinities: they reach the rows that see them and no others, be the ones
    before them their block's or an earlier block's."""
    nkv, hd, nq = 2, 48, 4
    for first in (32, 33, 64):                                        # a block's first position, its second, a tile's first
        n, rng = first + 3, np.random.default_rng(first)
        k, v = (rng.standard_normal((n, nkv, hd)).astype(np.float32) for _ in range(2))
        v[first, 0, 5], v[first + 1, 1, 7] = 3.38e38, -3.38e38
        o = Cache(dev, 1, nkv, hd)
        (k, kx), (v, vx) = typed(k, dtype), typed(v, dtype)
        o.add([0], [n], rows=[(k, kx), (v, vx)])
        q, qx = typed(rng.standard_normal((6, nq, hd)), dtype)
        got = values(dev.kv8_attend(o.c, o.p, o.layer, q, dev.batch([0, 6], [0]), longest))
        seen = list(range(n - 5, n + 1))
        held = o.want(0, 1)
        for t, s in enumerate(seen):
            bad = [(h, d) for at, h, d in ((first, 0, 5), (first + 1, 1, 7)) if s > at]
            vt = held.copy()
            for h, d in bad:
                vt[:, h, d] = 0
            want, tol = attended(qx[t:t + 1], o.want(0, 0), vt, [s], 2.0 ** -24 if dtype == "f32" else 2.0 ** -16, 2.0 ** -126, 2.0 ** -24 if dtype == "f32" else 0.0)
            if dtype == "bf16":
                tol = tol + 2.0 ** -8 * (np.abs(want) + tol)
            keep = np.ones((nq, hd), bool)
            for h, d in bad:
                keep[2 * h:2 * h + 2, d] = False
            assert np.all((np.abs(got[t] - want[0]) <= tol[0])[keep]) and not np.isfinite(got[t][~keep]).any(), (first, t)


@DTYPES
@pytest.mark.parametrize("runs, nkv, g, hd, longest", [(65, 1, 4, 64, 1000), (100, 1, 4, 128, 600), (300, 1, 3, 64, 1000), (90, 4, 2, 128, 1000), (130, 4, 1, 64, 250), (70, 2, 3, 160, 700)])
def test_attend_many_short_runs(dev, dtype, runs, nkv, g, hd, longest):
    """More runs than a wavefront has lanes, none of them split: few enough heads that eight wavefronts take a group together, and so many that four do; tokens of
    several, one or none a run, rows that no run names between them."""
    o = Cache(dev, runs, nkv, hd, pages=1200, width=9, seed=runs + hd)
    counts = [int(x) for x in o.rng.choice([1, 5, 31, 64, 65, 200], runs)]
    counts[0], counts[runs - 1] = longest, longest - 1
    o.add(list(range(runs)), counts, dtype)
    ids = [int(i) for i in o.rng.permutation(runs)]
    rows = [min(counts[i], int(o.rng.choice([0, 1, 1, 1, 2, 7]))) for i in ids]
    attend(o, ids, rows, nkv * g, dtype, longest=longest)


@DTYPES
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_attend_short(dev, dtype, hd):
    """Sequences of up to four tiles, which four wavefronts take; one group of rows and several."""
    o = Cache(dev, 4, 2, hd, seed=hd + 50)
    o.add([0, 1, 2, 3], [256, 1, 130, 64], dtype)
    attend(o, [1, 0, 3, 2], [1, 1, 1, 1], 8, dtype, longest=256)
    attend(o, [0, 2, 3], [40, 9, 3], 6, dtype, longest=256)


@DTYPES
def test_attend_many_rows(dev, dtype):
    """A run of so many rows that nothing is split, over positions before them; the length is not said."""
    o = Cache(dev, 1, 8, 64, seed=60)
    o.add([0], [300], dtype)
    o.add([0], [520], dtype)
    attend(o, [0], [520], 32, dtype)


@pytest.mark.parametrize("order", ["parts", "wavefronts"])
def test_attend_much_work_of_two_pages(dev, order):
    """Groups of rows times tiles past 2^25, of a page of values around 1 and one of values around -1: the first quarter of a sequence is one page and the rest the
    other, or they take turns. A part of a group, a quarter of its tiles, or a wavefront, every fourth tile, that is lost or counted twice moves the result by a
    sixth or more."""
    nkv, hd, g, n, width = 1, 8, 16, 128, 1 << 19
    c, p = dev.kv8(2, 1, nkv, hd), dev.pages(2, 2, width)
    rng = np.random.default_rng(61)
    k = rng.standard_normal((2 * PAGE, nkv, hd)).astype(np.float32) / 8
    v = rng.standard_normal((2 * PAGE, nkv, hd)).astype(np.float32) / 64 + np.float32(np.repeat([1, -1], PAGE))[:, None, None]
    b = dev.batch([0, 2 * PAGE], [0])
    dev.pages_grow(p, c, b)
    dev.kv8_append(c, p, 0, k, v, b)
    k, v = (x[:, 0].astype(np.float64) for x in dev.kv8_rows(c, p, 0, b))
    table, lens = np.zeros((2, width), np.int32), np.int32([2 * PAGE, PAGE * width])
    table[:, 1] = 1
    table[1] = np.arange(width) >= width // 4 if order == "parts" else np.arange(width) % 2
    for at, y in ((p.table, table), (p.len, lens)):
        assert dev.lib.l3m_dev_upload(at, C.c_void_p(y.ctypes.data), y.nbytes) == 0
    q = rng.standard_normal((n, g, hd)).astype(np.float32)
    size = dev.lib.l3m_kv8_work_bytes(C.byref(c), n, g)
    out, b = dev.alloc(q.nbytes), dev.batch([0, n], [1])
    assert dev.lib.l3m_k_kv8_attend(out, g * hd, dev.put(q), g * hd, A.F32, C.byref(c), C.byref(p), 0, C.byref(b), g, 0, dev.alloc(size), size, None) == 0
    got = dev.get(out, q.shape, np.float32)
    # the pages' positions count as often as the table names them, those behind the token in the last page once less; sums of 2^20 terms for a lane, of the weights
    # (which all have one sign) and of the values, 2^-24 of the sum of their magnitudes each
    times = np.repeat([np.sum(table[1] == 0), np.sum(table[1] == 1)], PAGE).astype(np.float64)
    z = q.reshape(-1, hd).astype(np.float64) @ k.T / np.sqrt(hd)
    for t in range(n):
        w = np.exp(z[t * g:(t + 1) * g]) * (times - ((np.arange(2 * PAGE) % PAGE > t) & (np.arange(2 * PAGE) // PAGE == table[1, -1])))
        w /= w.sum(1, keepdims=True)
        assert np.all(np.abs(got[t] - w @ v) <= 2.0 ** -3 * (w @ np.abs(v)))


def test_python_rows_of_no_run(dev, monkeypatch):
    """Results of the Python calls for rows that no run names, or that a sequence doesn't have, are zeros, whatever their memory held before."""
    alloc = dev.alloc

    def used(nbytes):
        p, marks = alloc(nbytes), np.full(nbytes, 0x41, np.uint8)
        assert dev.lib.l3m_dev_upload(p, C.c_void_p(marks.ctypes.data), nbytes) == 0
        return p

    monkeypatch.setattr(dev, "alloc", used)
    o = Cache(dev, 2, 1, 32, seed=62)
    o.add([0], [9])
    q, k = np.ones((8, 2, 32), np.uint16), np.ones((8, 1, 32), np.uint16)
    b = dev.batch([2, 5], [0], n=8)
    for got in (dev.attend_packed(q, k, k, b), dev.kv8_attend(o.c, o.p, o.layer, q, b), *dev.kv8_rows(o.c, o.p, o.layer, b), dev.pages_grow(o.p, o.c, b)):
        assert not got[:2].any() and not got[5:].any() and got[2:5].any()
    k, v = dev.kv8_rows(o.c, o.p, o.layer, dev.batch([0, 20], [0]))
    assert not k.any() and not v.any()


@DTYPES
@pytest.mark.parametrize("hd", [8, 40, 128])
def test_rows_aligned_to_their_values(dev, dtype, hd):
    """Rows of odd strides that begin one value behind a round address, in and out: the same bits as dense ones, and nothing beside them."""
    nkv, nq, n = 3, 6, 75
    x, y = Cache(dev, 1, nkv, hd, seed=63), Cache(dev, 1, nkv, hd, seed=63)
    (k, kx), (v, vx) = x.rows(n, dtype)
    x.add([0], [n], rows=[(k, kx), (v, vx)])
    kind, size = (A.F32, 4) if dtype == "f32" else (A.BF16, 2)
    b, width = dev.batch([0, n], [0]), 2 * nkv * hd + 5
    fused = np.zeros((n, width), k.dtype)
    fused[:, 1:1 + nkv * hd], fused[:, 2 + nkv * hd:2 + 2 * nkv * hd] = k.reshape(n, -1), v.reshape(n, -1)
    p = dev.put(fused)
    dev.pages_grow(y.p, y.c, b)
    assert dev.lib.l3m_k_kv8_append(C.byref(y.c), C.byref(y.p), y.layer, p + size, p + size * (2 + nkv * hd), width, kind, C.byref(b), None) == 0
    for one, two in zip(dev.kv8_rows(x.c, x.p, x.layer, b), dev.kv8_rows(y.c, y.p, y.layer, b)):
        assert np.array_equal(one, two) and one.any()
    q = typed(x.rng.standard_normal((n, nq, hd)), dtype)[0]
    wide, marks = np.zeros((n, nq * hd + 3), q.dtype), np.full((n, nq * hd + 7), 3, q.dtype)
    wide[:, 1:1 + nq * hd] = q.reshape(n, -1)
    need = dev.lib.l3m_kv8_work_bytes(C.byref(y.c), n, nq)
    out = dev.put(marks)
    assert dev.lib.l3m_k_kv8_attend(out + size, nq * hd + 7, dev.put(wide) + size, nq * hd + 3, kind, C.byref(y.c), C.byref(y.p), y.layer, C.byref(b), nq, 0, dev.alloc(need), need, None) == 0
    got = dev.get(out, marks.shape, q.dtype)
    assert np.array_equal(got[:, 1:1 + nq * hd], dev.kv8_attend(x.c, x.p, x.layer, q, b).reshape(n, -1))
    marks[:, 1:1 + nq * hd] = got[:, 1:1 + nq * hd]
    assert np.array_equal(got, marks)
