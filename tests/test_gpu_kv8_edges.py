"""The paged 8-bit K/V cache (l3m_k_kv8_attend) where it can go wrong: values that read as infinities, and the forms of a call by its runs, rows and heads."""
import numpy as np
import pytest

from serve import attended
from test_gpu_kv8 import DTYPES, Cache, typed, values

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
