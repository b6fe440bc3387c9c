"""Calls around the 4-bit K/V cache whose outputs lie on what the call reads or on the cache: refused on the host, before a launch, with the reason. And
the Python calls' weights and tables, which have to be as long as the call reads them."""
import ctypes as C

import numpy as np
import pytest

import l3m_amd as A
from weights import MXFP4, Q4_0

lib = A.lib()
MB = 1 << 20
NKV, HD, CAP = 2, 64, 100
CODES, SCALES = 2 * 4 * 512 * 2, {Q4_0: 2 * 4 * 32 * 2 * 2, MXFP4: 2 * 4 * 32 * 2}    # a plane's bytes
PLANES = {"kq": 16 * MB, "ks": 17 * MB, "vq": 18 * MB, "vs": 19 * MB}
ROWS, Q, K, WQ, WK, TABLE, WORK = (x * MB for x in (32, 40, 48, 56, 57, 58, 60))


@pytest.fixture(autouse=True)
def clear():
    lib.l3m_dev_clear_error()
    yield
    lib.l3m_dev_clear_error()


def cache(dtype=Q4_0, **change):
    return C.byref(A.KV4(**{**PLANES, "nkv": NKV, "hd": HD, "cap": CAP, "dtype": dtype, **change}))


def overlaps(rc):
    return rc == -1 and b"overlap" in (lib.l3m_dev_error() or b"")


def rope(q=Q, k=K, n=4, wq=WQ, wk=WK, table=TABLE, pos=10, nq=4):
    return lib.l3m_k_qk_norm_rope(q, k, ROWS, 640, n, nq, NKV, HD, wq, wk, 1e-5, 0, pos, table, None)


def append(c, q=Q, rows=ROWS, n=4, wq=WQ, wk=WK, table=TABLE, pos=10, nq=4):
    return lib.l3m_k_kv4_append(c, q, rows, 640, n, nq, wq, wk, 1e-5, 1, pos, table, None)


def attend(c, out=Q, q=ROWS, work=WORK, n=4, size=4 * MB):
    return lib.l3m_k_kv4_attend(out, q, c, n, 4, 3, work, size, None)


LAST_Q = 4 * 4 * 4 * HD - 4                       # the queries' last float, in bytes
ROW = 4 * HD                                      # a table row's bytes


@pytest.mark.parametrize("call", [rope, lambda **kw: append(cache(), **kw)], ids=["rope", "append"])
@pytest.mark.parametrize("change", [{"q": WQ}, {"q": WQ + 4 * HD - 4}, {"q": WQ - LAST_Q}, {"q": WK}, {"q": TABLE + 10 * ROW}, {"q": TABLE + 14 * ROW - 4},
                                    {"q": TABLE + 10 * ROW - LAST_Q}], ids=str)
def test_queries_on_weights(call, change):
    assert overlaps(call(**change))


@pytest.mark.parametrize("change", [{"k": WQ}, {"k": WK + 4 * HD - 4}, {"k": TABLE + 13 * ROW}], ids=str)
def test_keys_on_weights(change):
    assert overlaps(rope(**change))


@pytest.mark.parametrize("dtype", [Q4_0, MXFP4])
@pytest.mark.parametrize("plane, last", [("kq", None), ("ks", None), ("vq", None), ("vs", None), ("kq", CODES), ("vq", CODES), ("ks", 0), ("vs", 0)])
def test_on_the_planes(dtype, plane, last):
    at = PLANES[plane] + (0 if last is None else (last or SCALES[dtype]) - 16)
    c = cache(dtype)
    assert overlaps(append(c, q=at))
    lib.l3m_dev_clear_error()
    assert overlaps(append(c, rows=at))
    lib.l3m_dev_clear_error()
    for w in ("wq", "wk"):
        assert overlaps(append(c, **{w: at}))
        lib.l3m_dev_clear_error()
    assert overlaps(append(c, table=at - 10 * ROW))
    lib.l3m_dev_clear_error()
    assert overlaps(attend(c, out=at))
    lib.l3m_dev_clear_error()
    assert overlaps(attend(c, out=at, q=at))
    lib.l3m_dev_clear_error()
    assert overlaps(attend(c, work=at))
    lib.l3m_dev_clear_error()
    assert overlaps(lib.l3m_k_kv4_rows(c, at, None, 3, 2, None))
    lib.l3m_dev_clear_error()
    assert overlaps(lib.l3m_k_kv4_rows(c, Q, at, 3, 2, None))


@pytest.mark.parametrize("dtype", [Q4_0, MXFP4])
@pytest.mark.parametrize("change", [{"ks": PLANES["kq"] + CODES - 16}, {"vq": PLANES["kq"]}, {"vs": PLANES["ks"]}, {"vs": PLANES["vq"] + 16}, {"kq": PLANES["ks"] - 16}], ids=str)
def test_planes_on_each_other(dtype, change):
    c = cache(dtype, **change)
    for call in (append, attend, lambda c: lib.l3m_k_kv4_rows(c, Q, K, 0, 1, None)):
        assert overlaps(call(c))
        lib.l3m_dev_clear_error()


def test_neighbours_are_not_overlaps():
    """Next to each other is apart: what stops these calls here is the missing device, or nothing where there is one (nothing is run there)."""
    if lib.l3m_dev_init() == 0:
        pytest.skip("the addresses stand for no memory")
    lib.l3m_dev_clear_error()
    c = cache()
    for call in (lambda: rope(q=WQ + 4 * HD), lambda: rope(q=WQ - LAST_Q - 4), lambda: rope(q=TABLE + 14 * ROW), lambda: rope(q=TABLE + 10 * ROW - LAST_Q - 4),
                 lambda: append(c, q=PLANES["kq"] + CODES), lambda: attend(c, out=PLANES["vq"] - 4 * 4 * 4 * HD), lambda: append(c, q=WK, nq=0),
                 lambda: append(c, q=WK, wk=None, wq=None), lambda: attend(c, q=PLANES["kq"])):
        assert call() == -1 and b"overlap" not in lib.l3m_dev_error()
        lib.l3m_dev_clear_error()


@pytest.mark.parametrize("wq, wk, rows", [(HD - 1, None, 14), (None, HD // 2, 14), (HD + 1, HD, 14), (HD, HD, 13), (None, None, 0), ((1, HD), None, 14)], ids=str)
def test_python_lengths(dev_free, wq, wk, rows):
    """Weights of another length than a head's, a table that ends before the last token's row: refused before anything is uploaded."""
    dev_free._live = {TABLE: 4 * HD * rows}
    x = np.zeros((4, 8 * HD), np.float32)
    wq, wk = (None if n is None else np.ones(n, np.float32) for n in (wq, wk))
    with pytest.raises(ValueError):
        dev_free.qk_norm_rope(x, 4, 2, HD, wq, wk, pos=10, table=TABLE)
    with pytest.raises(ValueError):
        dev_free.kv4_append(A.KV4(**PLANES, nkv=NKV, hd=HD, cap=CAP, dtype=Q4_0), x, 4, 10, wq, wk, table=TABLE)
