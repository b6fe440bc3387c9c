"""What the calls around the 4-bit K/V cache refuse, on the host alone (no launch, no device), and the cache's size."""
import ctypes as C

import pytest

import l3m_amd as A
from weights import BF16, MXFP4, Q4_0, Q8_0

lib = A.lib()
P = 1 << 24                                       # stands for device memory: nothing reads it
BIG = 1 << 30


@pytest.fixture(autouse=True)
def clear():
    yield
    lib.l3m_dev_clear_error()


def cache(dtype=Q4_0, nkv=2, hd=64, cap=100, **change):
    c = A.KV4(P, 2 * P, 3 * P, 4 * P, nkv, hd, cap, dtype)
    for k, v in change.items():
        setattr(c, k, v)
    return c


def refused(rc):
    return rc == -1 and lib.l3m_dev_error() is not None


@pytest.mark.parametrize("dtype, scale", [(Q4_0, 2), (MXFP4, 1)])
@pytest.mark.parametrize("nkv, hd, cap", [(1, 8, 1), (3, 64, 32), (8, 128, 33), (2, 80, 1000), (1, 256, 1 << 22), (8, 256, 1 << 24)])
def test_size(dtype, scale, nkv, hd, cap):
    blocks = nkv * -(-cap // 32) * 32 * -(-hd // 32)
    plane = [-(-blocks * b // 256) * 256 for b in (16, scale)]
    assert lib.l3m_kv4_bytes(dtype, nkv, hd, cap) == 2 * sum(plane)
    c = A.KV4()
    assert lib.l3m_kv4_init(C.byref(c), dtype, nkv, hd, cap, P) == 0
    assert (c.kq, c.ks, c.vq, c.vs) == (P, P + plane[0], P + sum(plane), P + sum(plane) + plane[0])
    assert (c.nkv, c.hd, c.cap, c.dtype) == (nkv, hd, cap, dtype)


@pytest.mark.parametrize("dtype, nkv, hd, cap", [(Q8_0, 1, 64, 8), (BF16, 1, 64, 8), (-1, 1, 64, 8), (Q4_0, 0, 64, 8), (Q4_0, 1, 0, 8), (Q4_0, 1, 4, 8),
                                                 (Q4_0, 1, 68, 8), (MXFP4, 1, 264, 8), (MXFP4, 1, 64, 0), (MXFP4, 1, 64, -5), (MXFP4, 1, 64, BIG + 1)])
def test_shapes_refused(dtype, nkv, hd, cap):
    c = A.KV4()
    assert lib.l3m_kv4_bytes(dtype, nkv, hd, cap) == 0
    assert refused(lib.l3m_kv4_init(C.byref(c), dtype, nkv, hd, cap, P))
    bad = cache(dtype, nkv, hd, cap)
    assert refused(lib.l3m_k_kv4_rows(C.byref(bad), P, P, 0, 1, None))
    assert refused(lib.l3m_k_kv4_append(C.byref(bad), P, 9 * P, 4096, 1, 1, None, None, 0.0, 0, 0, None, None))
    assert refused(lib.l3m_k_kv4_attend(P, 9 * P, C.byref(bad), 1, 2, 0, P, BIG, None))
    assert lib.l3m_kv4_work_bytes(C.byref(bad), 1, 2) == 0


def test_init_refuses_memory():
    c = A.KV4()
    assert refused(lib.l3m_kv4_init(C.byref(c), Q4_0, 1, 64, 8, None))
    assert refused(lib.l3m_kv4_init(C.byref(c), Q4_0, 1, 64, 8, P + 8))
    assert refused(lib.l3m_kv4_init(None, Q4_0, 1, 64, 8, P))


@pytest.mark.parametrize("change", [{"kq": None}, {"ks": None}, {"vq": None}, {"vs": None}, {"kq": P + 4}, {"vs": P + 8}])
def test_planes_refused(change):
    c = cache(**change)
    assert refused(lib.l3m_k_kv4_rows(C.byref(c), P, P, 0, 1, None))
    assert refused(lib.l3m_k_kv4_attend(P, 9 * P, C.byref(c), 1, 2, 0, P, BIG, None))


@pytest.mark.parametrize("pos, n", [(-1, 1), (0, 0), (0, -1), (100, 1), (99, 2), (0, 101), (2 ** 31 - 1, 1), (50, 2 ** 31 - 1), (101, 0)])
def test_positions_refused(pos, n):
    c = C.byref(cache())
    assert refused(lib.l3m_k_kv4_rows(c, P, P, pos, n, None))
    assert refused(lib.l3m_k_kv4_append(c, P, 9 * P, 4096, n, 1, None, None, 0.0, 0, pos, None, None))
    assert refused(lib.l3m_k_kv4_attend(P, 9 * P, c, n, 2, pos, P, BIG, None))


def rope(q=P, k=2 * P, rows=9 * P, stride=640, n=4, nq=4, nkv=2, hd=64, wq=P, wk=P, eps=1e-5, pos=0, table=P):
    return lib.l3m_k_qk_norm_rope(q, k, rows, stride, n, nq, nkv, hd, wq, wk, eps, 0, pos, table, None)


@pytest.mark.parametrize("change", [
    {"q": None}, {"k": None}, {"rows": None}, {"stride": 383}, {"n": 0}, {"n": -3}, {"nq": -1}, {"nkv": -1}, {"nq": 0, "nkv": 0}, {"hd": 0}, {"hd": 63},
    {"hd": 258}, {"hd": -2}, {"eps": -1.0}, {"eps": float("nan")}, {"pos": -1}, {"pos": 2 ** 31 - 2}, {"q": P + 2}, {"k": P + 1}, {"rows": P + 2},
    {"wq": P + 2}, {"table": P + 2}, {"n": 2 ** 25, "nq": 65536, "nkv": 0, "hd": 2, "stride": 2 ** 18}, {"nq": 65537, "stride": 2 ** 30},
    {"q": 9 * P}, {"q": 9 * P + 4 * 640}, {"k": 9 * P + 4 * 256}, {"q": P, "k": P + 16}, {"q": 9 * P + 4, "n": 1}, {"k": 9 * P, "n": 1}],
    ids=lambda c: " ".join(f"{k}={v}" for k, v in c.items()))
def test_rope_refused(change):
    assert refused(rope(**change))


def append(c=None, q=P, rows=9 * P, stride=640, n=4, nq=4, eps=1e-5, pos=0):
    return lib.l3m_k_kv4_append(C.byref(c or cache()), q, rows, stride, n, nq, P, P, eps, 1, pos, P, None)


@pytest.mark.parametrize("change", [{"q": None}, {"rows": None}, {"stride": 511}, {"nq": -1}, {"nq": 65537, "stride": BIG}, {"eps": -1e-9}, {"q": 9 * P},
                                    {"q": 9 * P + 8, "n": 1}, {"rows": 9 * P + 1}], ids=str)
def test_append_refused(change):
    assert refused(append(**change))


@pytest.mark.parametrize("change", [{"nq": 0}, {"nq": 3}, {"nq": -2}, {"out": None}, {"q": None}, {"out": P + 2}, {"q": 9 * P + 1}, {"out": 9 * P + 4}, {"work": None},
                                    {"work": P + 4}, {"size": 0}, {"work": P + 4096 - 16}, {"work": 9 * P + 16}], ids=str)
def test_attend_refused(change):
    a = {"out": P, "q": 9 * P, "n": 4, "nq": 4, "pos": 3, "work": P, "size": BIG, **change}
    assert refused(lib.l3m_k_kv4_attend(a["out"], a["q"], C.byref(cache()), a["n"], a["nq"], a["pos"], a["work"], a["size"], None))


def test_work_bytes():
    c = cache(cap=10000)
    size = [lib.l3m_kv4_work_bytes(C.byref(c), n, 4) for n in (1, 2, 7, 64, 1000, 10000)]
    assert size[0] > 0 and size == sorted(size)               # a larger call's serves a smaller one
    assert [lib.l3m_kv4_work_bytes(C.byref(c), n, 4) for n in (0, -1, 10001)] == [0, 0, 0]
    assert lib.l3m_kv4_work_bytes(C.byref(c), 1, 3) == 0 and lib.l3m_kv4_work_bytes(None, 1, 4) == 0


def test_read_back_refused():
    c = C.byref(cache())
    assert refused(lib.l3m_k_kv4_rows(c, None, None, 0, 1, None))
    assert refused(lib.l3m_k_kv4_rows(c, P + 2, P, 0, 1, None))
    assert refused(lib.l3m_k_kv4_rows(None, P, P, 0, 1, None))
    assert refused(lib.l3m_k_kv4_rows(c, P, P, 0, 1, None))
    assert refused(lib.l3m_k_kv4_rows(c, P + 4 * 2 * 64 - 4, P, 0, 1, None))
