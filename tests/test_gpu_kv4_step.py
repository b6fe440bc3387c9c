"""The 4-bit K/V cache behind the framework's other kernels, as a program composes a layer of them."""
import ctypes as C

import numpy as np
import pytest

from test_gpu_kv4 import DTYPES, attended, clean, near, stored, table_of, turned  # noqa: F401 (clean: a fixture)
from weights import Q4_0
from weights import rows as block_rows

pytestmark = pytest.mark.gpu


@DTYPES
def test_step_from_matrix(dev, dtype):
    """A decode step as a program composes it, on device pointers: the norm, the fused q/k/v product over block weights, the append, the attention; four
    steps behind a prompt."""
    nq, nkv, hd, dim, cap = 6, 2, 64, 256, 80
    rng = np.random.default_rng(12)
    heads = nq + 2 * nkv
    m = dev.matrix(Q4_0, block_rows(Q4_0, heads * hd, dim, 3), dim)
    wn, wq, wk = ((1 + rng.standard_normal(s) / 8).astype(np.float32) for s in (dim, hd, hd))
    table = table_of(cap, hd)
    dn, dq, dk, dt = (dev.put(x) for x in (wn, wq, wk, table))
    c = dev.kv4(dtype, nkv, hd, cap)
    k, v = (rng.standard_normal((70, nkv, hd)) for _ in range(2))
    dev.kv4_append(c, np.concatenate([k, v], 1).reshape(70, -1).astype(np.float32), 0, 0)
    k, v = (x.astype(np.float64) for x in dev.kv4_rows(c, 0, 70))
    h, act, fused = dev.alloc(4 * dim), dev.alloc(dev.lib.l3m_act_bytes(Q4_0, dim)), dev.alloc(4 * heads * hd)
    size = dev.lib.l3m_kv4_work_bytes(C.byref(c), 1, nq)
    work, out = dev.alloc(size), dev.alloc(4 * nq * hd)
    for pos in range(70, 74):
        x = dev.put(rng.standard_normal(dim).astype(np.float32) * 3)
        L = dev.lib
        assert L.l3m_k_rmsnorm(h, x, dn, dim, 1e-5, None) == 0
        assert L.l3m_k_prep(Q4_0, h, dim, act, None) == 0
        assert L.l3m_k_gemv(C.byref(m), act, dim, fused, None) == 0
        rows = dev.get(fused, (1, heads, hd), np.float32)
        assert L.l3m_k_kv4_append(C.byref(c), fused, fused, heads * hd, 1, nq, dq, dk, 1e-6, 1, pos, dt, None) == 0   # the queries in place
        assert L.l3m_k_kv4_attend(out, fused, C.byref(c), 1, nq, pos, work, size, None) == 0
        q64 = turned(rows[:, :nq], wq, 1e-6, True, table[pos:pos + 1])
        k = np.concatenate([k, stored(dtype, turned(rows[:, nq:nq + nkv], wk, 1e-6, True, table[pos:pos + 1]).astype(np.float32))])
        v = np.concatenate([v, stored(dtype, rows[:, nq + nkv:])])
        q = dev.get(fused, (1, heads, hd), np.float32)[:, :nq]
        assert np.all(np.abs(q - q64) <= np.abs(q64) * 2.0 ** -24 * (1 + 1e-6) + 1e-13) and np.abs(q).max() > 0.1
        near(dev.get(out, (1, nq, hd), np.float32), *attended(dtype, q, k, v, pos))


@DTYPES
@pytest.mark.parametrize("n, pos", [(1, 20), (1, 4000), (37, 100)])
def test_floats_need_no_more_than_their_alignment(dev, dtype, n, pos):
    """Rows, queries, outputs, weights and table 4 bytes off: the results of aligned ones, bit for bit."""
    nq, nkv, hd = 4, 2, 40
    rng = np.random.default_rng(pos)
    c, table = dev.kv4(dtype, nkv, hd, pos + n), table_of(pos + n, hd)
    dev.kv4_append(c, rng.standard_normal((pos + n, 2 * nkv * hd)).astype(np.float32), 0, 0)
    rows = rng.standard_normal((n, (nq + 2 * nkv) * hd)).astype(np.float32)
    w = (1 + rng.standard_normal(hd) / 8).astype(np.float32)
    q = dev.kv4_append(c, rows, nq, pos, w, w, 1e-6, True, dev.put(table))
    out, (k, v) = dev.kv4_attend(c, q, pos), dev.kv4_rows(c, pos, n)

    def off(x):
        return dev.put(np.concatenate([np.zeros(1, np.float32), x.ravel()])) + 4
    drows, dw, dt, dq, do, dk, dv = off(rows), off(w), off(table), *(off(np.zeros(x.size, np.float32)) for x in (q, out, k, v))
    L, r = dev.lib, C.byref(c)
    size = L.l3m_kv4_work_bytes(r, n, nq)
    assert L.l3m_k_kv4_append(r, dq, drows, rows.shape[1], n, nq, dw, dw, 1e-6, 1, pos, dt, None) == 0
    assert L.l3m_k_kv4_attend(do, dq, r, n, nq, pos, dev.alloc(size), size, None) == 0
    assert L.l3m_k_kv4_rows(r, dk, dv, pos, n, None) == 0
    for p, want in ((dq, q), (do, out), (dk, k), (dv, v)):
        assert np.array_equal(dev.get(p, want.shape, np.float32), want)
    assert L.l3m_k_qk_norm_rope(dq, dk, drows, rows.shape[1], n, nq, nkv, hd, dw, dw, 1e-6, 1, pos, dt, None) == 0
    assert np.array_equal(dev.get(dq, q.shape, np.float32), q)
