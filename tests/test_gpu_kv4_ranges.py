"""The attention over the 4-bit K/V cache where ranges end: scores far below zero."""
import numpy as np
import pytest

from test_gpu_kv4 import DTYPES, attended, clean, near  # noqa: F401 (clean: a fixture)

pytestmark = pytest.mark.gpu


def cache_of(dev, dtype, k, v):
    """A cache of rows k, v [n][nkv][hd], and the values it holds."""
    n, nkv, hd = k.shape
    c = dev.kv4(dtype, nkv, hd, n)
    dev.kv4_append(c, np.concatenate([k, v], 1).reshape(n, -1).astype(np.float32), 0, 0)
    return (c,) + tuple(x.astype(np.float64) for x in dev.kv4_rows(c, 0, n))


# ---------------------------------------------------------------- scores

@DTYPES
@pytest.mark.parametrize("hd, nq, nkv", [(64, 3, 3), (128, 8, 2), (8, 1, 1), (200, 4, 1)])
@pytest.mark.parametrize("pos, n", [(0, 1), (39, 1), (2999, 1), (69999, 1), (0, 70), (1500, 5)])
@pytest.mark.parametrize("low", [60, 100, 1000, 30000])
def test_attend_low_scores(dev, dtype, hd, nq, nkv, pos, n, low):
    """Every key opposite to the queries, scores of some -low: softmax does not mind a common offset."""
    rng = np.random.default_rng(low + pos)
    side = np.where(rng.standard_normal(hd) < 0, -1.0, 1.0)
    k = rng.standard_normal((pos + n, nkv, hd)) * 0.1 - side * 2
    v = rng.standard_normal((pos + n, nkv, hd))
    c, k, v = cache_of(dev, dtype, k, v)
    q = ((rng.standard_normal((n, nq, hd)) * 0.1 + side) * low / (2 * np.sqrt(hd))).astype(np.float32)
    near(dev.kv4_attend(c, q, pos), *attended(dtype, q, k, v, pos))


@DTYPES
@pytest.mark.parametrize("seen, n", [(300, 1), (9000, 1), (300, 300)])
@pytest.mark.parametrize("at", [0, 64, 288])
def test_attend_a_low_tile(dev, dtype, seen, n, at):
    """Ordinary scores but for the 32 positions of one tile, which lie at some -300: they count for nothing."""
    nq, nkv, hd = 4, 2, 128
    rng = np.random.default_rng(at)
    side = np.where(rng.standard_normal(hd) < 0, -1.0, 1.0)
    k = rng.standard_normal((seen, nkv, hd)) * 0.3
    k[at:at + 32] -= side * 2
    c, k, v = cache_of(dev, dtype, k, rng.standard_normal((seen, nkv, hd)))
    q = (rng.standard_normal((n, nq, hd)) * 0.3 + side * 150 / np.sqrt(hd)).astype(np.float32)
    near(dev.kv4_attend(c, q, seen - n), *attended(dtype, q, k, v, seen - n))
