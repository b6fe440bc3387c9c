"""Calls of the kernels that serve many sequences whose arguments mean nothing: refused on the host, before a launch, with the reason."""
import ctypes as C

import numpy as np
import pytest

import l3m_amd as A
from serve import BLOCK, PAGE, Blocks, Lists, bf16, from_bf16, nearest_e4m3

lib = A.lib()
MB = 1 << 20
F32, BF16 = A.F32, A.BF16
ROWS, Q, K, V, POS, IDS, STARTS, WORK, OUT = (x * 16 * MB for x in range(4, 13))
MEM, TABLES = 300 * MB, 400 * MB
NQ, NKV, HD, LAYERS, N, SEQS, NPAGES, WIDTH = 4, 2, 64, 3, 10, 5, 12, 6


@pytest.fixture(autouse=True)
def clear():
    lib.l3m_dev_clear_error()
    yield
    lib.l3m_dev_clear_error()


def refused(rc, word):
    err = (lib.l3m_dev_error() or b"").decode()
    lib.l3m_dev_clear_error()
    assert rc == -1 and word in err, (rc, err)


def plan(hd=HD, rd=HD, halves=0, theta=1e4, scaling=0, factor=1.0, low=1.0, high=4.0, trained=100):
    r = A.Rotary()
    return lib.l3m_rotary_init(C.byref(r), hd, rd, halves, theta, scaling, factor, low, high, trained), r


def rotary(q=Q, qs=NQ * HD, k=K, ks=NKV * HD, out=F32, rows=ROWS, stride=1000, dtype=F32, n=N, nq=NQ, nkv=NKV, pos=POS, pos0=0, r=None):
    r = r or plan()[1]
    return lib.l3m_k_rotary(C.byref(r), q, qs, k, ks, out, rows, stride, dtype, n, nq, nkv, pos, pos0, None)


def batch(ids=IDS, starts=STARTS, seqs=SEQS, n=N):
    return A.Batch(ids, starts, seqs, n)


def cache(**change):
    return A.KV8(**{"mem": MEM, "pages": NPAGES, "layers": LAYERS, "nkv": NKV, "hd": HD, **change})


def tables(mem=TABLES, pages=NPAGES, seqs=SEQS, width=WIDTH, **change):
    p = A.Pages()
    assert lib.l3m_pages_init(C.byref(p), pages, seqs, width, mem) == 0
    for name, x in change.items():
        setattr(p, name, x)
    return p


def prompt(out=OUT, os=NQ * HD, q=Q, qs=NQ * HD, k=K, v=V, kvs=NKV * HD, b=None, nq=NQ, nkv=NKV, hd=HD):
    return lib.l3m_k_attend_packed(out, os, q, qs, k, v, kvs, C.byref(b or batch()), nq, nkv, hd, None)


def append(c=None, p=None, layer=0, k=K, v=V, stride=NKV * HD, dtype=F32, b=None):
    return lib.l3m_k_kv8_append(C.byref(c or cache()), C.byref(p or tables()), layer, k, v, stride, dtype, C.byref(b or batch()), None)


def rows(c=None, p=None, layer=0, k=K, v=V, b=None):
    return lib.l3m_k_kv8_rows(C.byref(c or cache()), C.byref(p or tables()), layer, k, v, C.byref(b or batch()), None)


def attend(out=OUT, os=NQ * HD, q=Q, qs=NQ * HD, dtype=F32, c=None, p=None, layer=0, b=None, nq=NQ, longest=0, work=WORK, size=16 * MB):
    return lib.l3m_k_kv8_attend(out, os, q, qs, dtype, C.byref(c or cache()), C.byref(p or tables()), layer, C.byref(b or batch()), nq, longest, work, size, None)


def grow(c=None, p=None, b=None, pos=POS):
    return lib.l3m_k_pages_grow(C.byref(p or tables()), C.byref(c or cache()), C.byref(b or batch()), pos, None)


def fork(p=None, a=IDS, b=STARTS, n=3):
    return lib.l3m_k_pages_fork(C.byref(p or tables()), a, b, n, None)


def cut(p=None, a=IDS, b=STARTS, n=3):
    return lib.l3m_k_pages_cut(C.byref(p or tables()), a, b, n, None)


@pytest.mark.parametrize("change, word", [({"hd": 0}, "head"), ({"hd": 257, "rd": 2}, "head"), ({"rd": 65}, "head"), ({"rd": 3}, "head"), ({"rd": -2}, "head"), ({"theta": 0.0}, "base"),
                                          ({"theta": float("nan")}, "base"), ({"theta": float("inf")}, "base"), ({"scaling": 5}, "scaling"), ({"scaling": -1}, "scaling"),
                                          ({"scaling": 1, "factor": 0.5}, "factor"), ({"scaling": 1, "factor": float("nan")}, "factor"), ({"scaling": 3, "low": 0.0}, "turns"),
                                          ({"scaling": 4, "high": 1.0}, "turns"), ({"scaling": 4, "trained": 0}, "turns"), ({"scaling": 3, "theta": 1.0}, "base"),
                                          ({"scaling": 2, "rd": 2, "factor": 2.0}, "pair")], ids=str)
def test_plans(change, word):
    refused(plan(**change)[0], word)


@pytest.mark.parametrize("change, word", [({"dtype": 2}, "f32 or bf16"), ({"out": 9}, "f32 or bf16"), ({"n": -1}, "counts"), ({"nq": -1}, "counts"), ({"nq": 0, "nkv": 0}, "counts"),
                                          ({"stride": 6 * HD - 1}, "fewer"), ({"qs": NQ * HD - 1}, "fewer"), ({"ks": 1}, "fewer"), ({"rows": None}, "no rows"), ({"q": None}, "no rows"),
                                          ({"k": None}, "no rows"), ({"rows": ROWS + 2}, "aligned"), ({"q": Q + 1, "out": BF16}, "aligned"), ({"pos": POS + 2}, "aligned"),
                                          ({"pos": None, "pos0": -1}, "positions"), ({"pos": None, "pos0": 2 ** 31 - 5}, "positions"), ({"q": ROWS + 4}, "overlaps"),
                                          ({"q": ROWS}, "overlaps"), ({"q": ROWS, "qs": 1000, "out": BF16}, "overlaps"), ({"k": ROWS + 4 * NQ * HD}, "overlaps"),
                                          ({"k": Q + 4}, "overlaps"), ({"q": POS}, "overlaps"), ({"k": POS - 4}, "overlaps"), ({"q": Q, "k": Q + 4 * (NQ * HD - 1), "qs": 600, "ks": 600}, "overlaps")],
                         ids=str)
def test_rotary(change, word):
    refused(rotary(**change), word)


SHAPES = [({"hd": 0}, "hd"), ({"hd": 12}, "hd"), ({"hd": 264}, "hd"), ({"nq": 3}, "multiple"), ({"nq": 0}, "multiple")]


@pytest.mark.parametrize("change, word", SHAPES + [({"nkv": 0}, "multiple"), ({"os": NQ * HD - 8}, "fewer"), ({"qs": 8}, "fewer"), ({"kvs": HD}, "fewer"), ({"out": None}, "no rows"),
                                                   ({"v": None}, "no rows"), ({"q": Q + 2}, "aligned"), ({"kvs": NKV * HD + 4}, "aligned"), ({"out": Q + 16}, "the same or apart"),
                                                   ({"out": Q, "os": NQ * HD + 8}, "the same or apart"), ({"out": K}, "k or v"), ({"out": V + 16}, "k or v"), ({"out": IDS - 16}, "batch"),
                                                   ({"b": batch(seqs=-1)}, "counts"), ({"b": batch(n=-1)}, "counts"), ({"b": batch(starts=None)}, "starts"),
                                                   ({"b": batch(ids=IDS + 1)}, "aligned"), ({"b": batch(seqs=65537)}, "counts")], ids=str)
def test_attend_packed(change, word):
    refused(prompt(**change), word)


CACHES = [({"c": cache(mem=None)}, "memory"), ({"c": cache(mem=MEM + 16)}, "aligned"), ({"c": cache(hd=20)}, "cache"), ({"c": cache(pages=0)}, "cache"), ({"c": cache(layers=0)}, "cache"),
          ({"c": cache(nkv=0)}, "cache"), ({"p": tables(table=None)}, "memory"), ({"p": tables(len=TABLES + 8)}, "aligned"), ({"p": tables(seqs=SEQS, **{"scratch": None})}, "memory"),
          ({"p": tables(pages=NPAGES + 1)}, "more pages"), ({"p": tables(mem=MEM + MB // 4)}, "overlap"), ({"b": batch(starts=None)}, "starts"), ({"b": batch(n=-4)}, "counts")]
LAYER = [({"layer": -1}, "layer"), ({"layer": LAYERS}, "layer"), ({"b": batch(ids=MEM)}, "overlaps")]


@pytest.mark.parametrize("change, word", CACHES + LAYER + [({"dtype": 2}, "f32 or bf16"), ({"stride": NKV * HD - 1}, "fewer"), ({"k": None}, "no rows"), ({"v": None}, "no rows"),
                                                           ({"k": K + 2}, "aligned"), ({"v": MEM + 4}, "overlap")], ids=str)
def test_append(change, word):
    refused(append(**change), word)


@pytest.mark.parametrize("change, word", CACHES + LAYER + [({"k": None, "v": None}, "no output"), ({"k": K + 1}, "aligned"), ({"v": K + 4}, "overlaps"), ({"k": MEM}, "overlaps"),
                                                           ({"v": TABLES}, "overlaps"), ({"v": STARTS}, "overlaps")], ids=str)
def test_rows(change, word):
    refused(rows(**change), word)


@pytest.mark.parametrize("change, word", CACHES + LAYER + [({"dtype": 3}, "f32 or bf16"), ({"nq": 3}, "multiple"), ({"nq": 0}, "multiple"), ({"os": 8}, "fewer"), ({"qs": 8}, "fewer"),
                                                           ({"longest": -1}, "negative"), ({"out": None}, "no queries"), ({"q": Q + 2}, "aligned"), ({"out": Q + 4}, "the same or apart"),
                                                           ({"work": None}, "workspace"), ({"work": WORK + 8}, "workspace"), ({"size": 8}, "workspace"), ({"work": Q}, "overlaps"),
                                                           ({"work": OUT}, "overlaps"), ({"out": MEM}, "overlaps"), ({"work": MEM}, "overlaps"), ({"out": TABLES}, "overlaps"),
                                                           ({"out": STARTS}, "overlaps"), ({"work": IDS}, "overlaps")], ids=str)
def test_attend(change, word):
    refused(attend(**change), word)


@pytest.mark.parametrize("change, word", CACHES + [({"b": batch(seqs=SEQS + 1)}, "more runs"), ({"pos": POS + 2}, "aligned"), ({"pos": MEM}, "overlap"), ({"pos": TABLES}, "overlap"),
                                                   ({"pos": STARTS + 4}, "overlap"), ({"b": batch(ids=TABLES)}, "overlaps"), ({"b": batch(starts=MEM)}, "overlaps")], ids=str)
def test_grow(change, word):
    refused(grow(**change), word)


@pytest.mark.parametrize("call", [fork, cut])
@pytest.mark.parametrize("change, word", [({"p": tables(refs=None)}, "memory"), ({"n": -1}, "more sequences"), ({"n": SEQS + 1}, "more sequences"), ({"a": None}, "no list"), ({"a": IDS + 2}, "aligned"),
                                          ({"a": TABLES}, "overlaps"), ({"b": TABLES + 256}, "overlaps")], ids=str)
def test_lists(call, change, word):
    refused(call(**change), word)


def test_shapes():
    """Sizes that are refused are 0; a page's bytes are as documented; memory that is not aligned."""
    assert lib.l3m_kv8_page_bytes(3, 2, 80) == 3 * -(-(2 * (256 * 96 + 8)) // 256) * 256 and lib.l3m_kv8_bytes(7, 3, 2, 80) == 7 * lib.l3m_kv8_page_bytes(3, 2, 80)
    for bad in ((0, 1, 1, 64), (1, 0, 1, 64), (1, 1, 0, 64), (1, 1, 1, 4), (1, 1, 1, 68), (1, 1, 1, 264), ((1 << 20) + 1, 1, 1, 64)):
        assert lib.l3m_kv8_bytes(*bad) == 0
        refused(lib.l3m_kv8_init(C.byref(A.KV8()), *bad, MEM), "kv8")
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 65537, 1), (1, 65536, 1 << 13), (1 << 21, 1, 1)):
        assert lib.l3m_pages_bytes(*bad) == 0
        refused(lib.l3m_pages_init(C.byref(A.Pages()), *bad, TABLES), "pages")
    refused(lib.l3m_kv8_init(C.byref(A.KV8()), 1, 1, 1, 64, MEM + 128), "aligned")
    refused(lib.l3m_pages_init(C.byref(A.Pages()), 1, 1, 1, TABLES + 8), "aligned")
    refused(lib.l3m_k_pages_reset(C.byref(tables(refs=None)), None), "memory")
    refused(lib.l3m_k_pages_clear(C.byref(tables(state=None)), None), "memory")
    refused(lib.l3m_k_pages_compact(C.byref(tables()), C.byref(cache(mem=None)), None), "memory")
    c = cache()
    assert lib.l3m_kv8_work_bytes(C.byref(c), 1, 4) > 0 and lib.l3m_kv8_work_bytes(C.byref(c), 1, 3) == 0 and lib.l3m_kv8_work_bytes(C.byref(c), 0, 4) == 0
    assert lib.l3m_kv8_work_bytes(C.byref(c), 100, 4) >= lib.l3m_kv8_work_bytes(C.byref(c), 1, 4)


def test_nothing_to_do():
    """No rows, no runs or an empty list are no error, with no device and no memory either."""
    none = batch(None, STARTS, 0, 0)
    assert rotary(n=0, rows=None, q=None, k=None) == 0 and prompt(b=none, out=None, q=None, k=None, v=None) == 0
    assert append(b=none, k=None, v=None) == 0 and rows(b=none) == 0 and attend(b=none, out=None, q=None, work=None, size=0) == 0 and grow(b=none, pos=None) == 0
    assert fork(a=None, b=None, n=0) == 0 and cut(a=None, b=None, n=0) == 0


def test_allowed_neighbours():
    """What is allowed gets past the checks: what stops these calls here is the missing device (nothing is run where there is one)."""
    if lib.l3m_dev_init() == 0:
        pytest.skip("the addresses stand for no memory")
    lib.l3m_dev_clear_error()
    width = (NQ + 2 * NKV) * HD
    for call in (lambda: rotary(q=ROWS, qs=1000, k=ROWS + 4 * NQ * HD, ks=1000), lambda: rotary(q=Q, qs=600, k=Q + 4 * NQ * HD, ks=600), lambda: rotary(k=None, nkv=0, ks=0),
                 lambda: rotary(q=None, nq=0, qs=0, pos=None), lambda: prompt(out=Q), lambda: prompt(q=Q, out=Q, qs=width, os=width, kvs=width, k=Q + 2 * NQ * HD, v=Q + 2 * (NQ + NKV) * HD),
                 lambda: append(k=K, v=K + 4 * NKV * HD, stride=500), lambda: rows(v=None), lambda: rows(k=None), lambda: attend(out=Q), lambda: attend(b=batch(ids=None)), lambda: grow(pos=None),
                 lambda: cut(b=None), lambda: append(c=cache(pages=NPAGES + 4)), lambda: attend(size=lib.l3m_kv8_work_bytes(C.byref(cache()), N, NQ))):
        rc, err = call(), lib.l3m_dev_error()
        assert rc == -1 and b"no " in err and b"device" in err, err
        lib.l3m_dev_clear_error()


def test_python_lengths(dev_free):
    """Lengths that do not go together are refused before anything is uploaded."""
    r, p, c = dev_free.rotary_plan(HD), tables(), cache()
    x = np.zeros((4, 6 * HD), np.float32)
    kv, b = np.zeros((4, NKV, HD), np.float32), batch(n=4)
    for call in (lambda: dev_free.rotary(r, x, 4, 2, pos=[1, 2, 3]), lambda: dev_free.batch([0, 1], [1, 2]), lambda: dev_free.pages_fork(p, [0], [1, 2]), lambda: dev_free.pages_cut(p, [0, 1], [3]),
                 lambda: dev_free.kv8_append(c, p, 0, kv, kv[:3], b), lambda: dev_free.kv8_append(c, p, 0, kv, kv, batch(n=5)), lambda: dev_free.kv8_append(c, p, 0, kv, bf16(kv), b),
                 lambda: dev_free.kv8_attend(c, p, 0, np.zeros((4, 4, 32), np.float32), b), lambda: dev_free.kv8_attend(c, p, 0, np.zeros((3, 4, HD), np.float32), b),
                 lambda: dev_free.attend_packed(bf16(x.reshape(4, 6, HD)), bf16(kv), bf16(kv[:3]), b), lambda: dev_free.kv8(0, 1, 1, 64), lambda: dev_free.pages(1, 0, 1)):
        with pytest.raises(ValueError):
            call()


# ---------------------------------------------------------------- the tests' own oracles

def test_oracle_of_codes():
    """nearest_e4m3 by a second way: the last place a value of its exponent has."""
    x = np.concatenate([np.linspace(-448, 448, 4001), 2.0 ** np.linspace(-12, 8, 999), [0, 2.0 ** -10, 3 * 2.0 ** -10, 17, 19, 2.0 ** -9]])
    e = np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 1e-30))), -6) - 3
    want = np.round(x / 2.0 ** e) * 2.0 ** e                         # to even
    assert np.array_equal(nearest_e4m3(x), want)
    assert np.array_equal(from_bf16(bf16(np.float32([1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, -3.0]))), np.float32([1, 1 + 2.0 ** -6, -3]))


def test_oracle_of_blocks():
    """Rows of one block in one call or two: the same while the first sets the scale, rounded twice where the second raises it."""
    x = np.float64([[448.0, 100.1], [1.03, 2.0 ** -9], [3000.0, 0.4]])
    one, two, low = Blocks(2), Blocks(2), Blocks(2)
    one.add(x[:2])
    two.add(x[:1])
    two.add(x[1:2])
    assert np.array_equal(one.x, two.x) and np.array_equal(one.x[1], [1.0, 2.0 ** -9])
    two.add(x[2:])
    assert two.u == [8.0] and np.array_equal(two.x, [[448, 104], [1, 0], [3 * 2.0 ** 10, 0.40625]])
    low.add(x[1:2] * 0)
    assert low.u == [2.0 ** -126]
    low.cut(0)
    assert BLOCK * 4 == PAGE and low.u == []


def test_oracle_of_lists():
    """A wrong page, count or length in the oracle's place is found."""
    o = Lists(4, 2, 3)
    o.grow([0], [130])
    good = {"state": "ok", "used": 2, "refs": np.int32(o.refs), "len": np.int32(o.len), "table": np.int32([[0, 1, -1], [-1, -1, -1]])}
    o.check(good)
    for name, wrong in (("state", "bad"), ("used", 3), ("refs", np.int32([1, 1, 1, 0])), ("len", np.int32([131, 0])), ("table", np.int32([[1, 0, -1], [-1, -1, -1]]))):
        with pytest.raises(AssertionError):
            o.check({**good, name: wrong})


def test_attend_packed_far_rows():
    """Rows of K and V so far apart that a tile's offsets pass 32 bits."""
    refused(prompt(kvs=(1 << 23) + 8, b=batch(n=1)), "2^23")
