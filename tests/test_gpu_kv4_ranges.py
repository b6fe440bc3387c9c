"""The attention over the 4-bit K/V cache where ranges end: scores far below zero, values whose sizes change along
the cache; its precision at ordinary sizes; and heads beside one that is not finite."""
import numpy as np
import pytest

from test_cpu_kv4_precision import LIMIT, apart, ordinary
from test_gpu_kv4 import DTYPES, attended, clean, each_near, filled, near  # noqa: F401 (clean: a fixture)
from weights import MXFP4, Q4_0

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


@DTYPES
def test_attend_lowest_scores(dev, dtype):
    """A score at the end of what float32 holds, in base 2, alone: the answer is the position's value. The other wavefronts have seen nothing, which is
    less. mxfp4's stops at 3.1e38: a partial sum leaves float32 above 3.2e38, since the first part of q is q rounded to 1/4 of [2, 4), up to
    1/16 more, and 17/16 of 3.2e38 is 3.4e38."""
    hd = 8
    k = -8 * 65504.0 if dtype == Q4_0 else -6 * 2.0 ** 60
    for score in (3.2e38, 3.39e38) if dtype == Q4_0 else (3.05e38, 3.1e38):
        x, y = np.zeros((1, 1, hd)), np.arange(1.0, hd + 1)[None, None]
        x[..., 0] = k
        c, kk, v = cache_of(dev, dtype, x, y)
        q = np.zeros((1, 1, hd), np.float32)
        q[..., 0] = score / -kk[0, 0, 0] * np.sqrt(hd) / 1.44269504
        got = dev.kv4_attend(c, q, 0)
        assert np.all(np.abs(got - v) <= np.abs(v) * 2.0 ** -21), got


# ---------------------------------------------------------------- values' sizes

def shares(q, k, v):
    """One token's output over keys whose scores are exact (their codes have one dimension other than zero), and its error's bound: a weight is off
    by the roundings of its own score, of the maxima it was taken against (three moves of them) and of its parts, and a share ends at 2^-32 of the largest weight
    times the largest value."""
    s = (q.astype(np.float64) @ k.T) / np.sqrt(len(q))
    p = np.exp(s - s.max())
    p /= p.sum()
    off = (4 * np.abs(s) + 3 * 1.45 * np.abs(s).max() + 32) * 2.0 ** -24
    out = p @ v
    sums = (len(k) / 32 + 64) * 2.0 ** -24 * (p @ np.abs(v))
    return out, (p * off) @ np.abs(v) + (p @ off) * np.abs(out) + sums + (len(k) * p.max() + 1) * 2.0 ** -32 * np.abs(v).max()


@pytest.mark.parametrize("up", [3.0, 5.4, 7.5, 7.9])
@pytest.mark.parametrize("below", [0.3, 0.55, 0.8])
def test_attend_range_after_lowering(dev, up, below):
    """q4_0, three tiles of one wavefront: small values; then a weight near the end of its range on values 2^13 times larger, which lowers the row's
    range; then the largest weights, on small values again. Those keep their 2^-32."""
    hd, seen = 64, 384                                                # twelve tiles, three for a wavefront
    tile = np.arange(seen) // 32
    level = np.where(tile % 3 == 1, -40.0 + up, -40.0)                # log2 of the weights
    level[-32:] = -below
    level[-32] = 0
    d = np.where(tile % 3 == 1, 2.0 ** 7, 2.0 ** -6)
    k, v = np.zeros((seen, 1, hd)), np.full((seen, 1, hd), 7.0)
    k[:, 0, 0] = level
    v[:, :, ::32] = -8
    c, k, v = cache_of(dev, Q4_0, k, v * d[:, None, None])
    q = np.zeros((1, 1, hd), np.float32)
    q[..., 0] = np.sqrt(hd) * np.log(2)
    want, tol = shares(q[0, 0], k[:, 0], v[:, 0])
    near(dev.kv4_attend(c, q, seen - 1)[0, 0], want, tol)


@pytest.mark.parametrize("e", [-24, -23, -22, -20, -18, -14, -10, 0])
def test_attend_small_scales_shares(dev, e):
    """q4_0 values down to f16's subnormal scales: many small weights count beside a large one."""
    hd, seen = 64, 1500
    rng = np.random.default_rng(-e)
    v = rng.integers(-7, 8, (1, hd)) * 2.0 ** e
    v[:, ::32] = -8 * 2.0 ** e
    v = np.tile(v, (seen, 1))
    v[0] = 0
    k = np.zeros((seen, 1, hd))
    k[1:, 0, 0] = -18.45
    c, k, v = cache_of(dev, Q4_0, k, v[:, None])
    q = np.zeros((1, 1, hd), np.float32)
    q[..., 0] = np.sqrt(hd) * np.log(2)
    want, tol = shares(q[0, 0], k[:, 0], v[:, 0])
    near(dev.kv4_attend(c, q, seen - 1)[0, 0], want, tol)


SIZES = [(-20, -30, -30), (-22, -40, -26), (-20, 0, -30), (-100, -40, -110), (100, 30, -100), (-22, -110, -22), (-110, 120, -20), (120, 60, 0)]


@pytest.mark.parametrize("sizes", SIZES, ids=str)
@pytest.mark.parametrize("hd, n, seen", [(64, 1, 900), (128, 1, 20000), (96, 70, 90), (40, 5, 200), (64, 40, 930)])
def test_attend_value_sizes_down(dev, hd, n, seen, sizes):
    """mxfp4 V rows of 2^sizes in the first, middle and last third, smaller ones behind larger ones: a value counts
    down to 2^-32 of the largest that its token sees."""
    nq, nkv = 3, 1
    rng = np.random.default_rng(seen)
    third = -(-seen // 3)
    scale = np.repeat([2.0 ** s for s in sizes], third)[:seen]
    v = np.abs(rng.standard_normal((seen, nkv, hd))) * scale[:, None, None]
    c, k, v = cache_of(dev, MXFP4, rng.standard_normal((seen, nkv, hd)), v)
    q = (rng.standard_normal((n, nq, hd)) * np.array([2.0 ** -12, 2.0 ** -5, 1])[:, None]).astype(np.float32)   # weights alike, and not
    each_near(MXFP4, dev.kv4_attend(c, q, seen - n), q, k, v, seen - n)


@pytest.mark.parametrize("e", [0, -20, -40, -120])
@pytest.mark.parametrize("hd, n, seen", [(64, 1, 40), (128, 1, 3000), (128, 40, 60)])
def test_attend_blocks_of_zeros(dev, hd, n, seen, e):
    """mxfp4 values of 2^e among blocks and rows of zeros, in every tile: zeros have no size."""
    nq, nkv = 2, 1
    rng = np.random.default_rng(seen)
    v = rng.standard_normal((seen, nkv, hd)) * 2.0 ** e
    v[::5] = 0
    v[::3, :, 32:] = 0
    c, k, v = cache_of(dev, MXFP4, rng.standard_normal((seen, nkv, hd)), v)
    assert not v[::5].any() and v[1::5].any(-1).all()
    q = rng.standard_normal((n, nq, hd)).astype(np.float32)
    each_near(MXFP4, dev.kv4_attend(c, q, seen - n), q, k, v, seen - n)


@pytest.mark.parametrize("sizes", [(None, -40, -40), (None, -100, -60), (-110, None, -120), (0, None, -20), (-20, None, -30), (None, None, -120), (None, 20, -30), (None, None, None)],
                         ids=str)
@pytest.mark.parametrize("hd, n, seen", [(64, 1, 900), (128, 1, 20000), (96, 70, 90), (40, 5, 200), (64, 40, 930), (32, 64, 64)])
def test_attend_value_sizes_and_zeros(dev, hd, n, seen, sizes):
    """As above, None for rows of zeros: what lies beside or behind them counts as if they were not there."""
    nq, nkv = 3, 1
    rng = np.random.default_rng(seen)
    third = -(-seen // 3)
    scale = np.repeat([0.0 if s is None else 2.0 ** s for s in sizes], third)[:seen]
    v = np.abs(rng.standard_normal((seen, nkv, hd))) * scale[:, None, None]
    c, k, v = cache_of(dev, MXFP4, rng.standard_normal((seen, nkv, hd)), v)
    q = (rng.standard_normal((n, nq, hd)) * np.array([2.0 ** -12, 2.0 ** -5, 1])[:, None]).astype(np.float32)
    each_near(MXFP4, dev.kv4_attend(c, q, seen - n), q, k, v, seen - n)


# ---------------------------------------------------------------- precision

@DTYPES
@pytest.mark.parametrize("hd", [8, 32, 48, 64, 80, 96, 128, 160, 200, 224, 256])
@pytest.mark.parametrize("pos, n, nq, nkv", [(39, 1, 8, 2), (999, 1, 8, 2), (20000, 1, 8, 2), (0, 150, 4, 2), (600, 40, 6, 3), (0, 300, 64, 64)])
def test_attend_precision(dev, dtype, hd, pos, n, nq, nkv):
    """Inputs of ordinary size: as near the formula as float32 sums are (LIMIT), which a lost part of the weights or the queries is not."""
    q, k, v = ordinary(hd, pos, n, nq, nkv)
    c, k, v = cache_of(dev, dtype, k, v)
    got = dev.kv4_attend(c, q, pos)
    heads = sorted({0, nkv // 2, nkv - 1})
    g = nq // nkv
    for h in heads:
        part = slice(h * g, (h + 1) * g)
        want = attended(dtype, q[:, part], k[:, h:h + 1], v[:, h:h + 1], pos)[0]
        assert apart(got[:, part], want) <= LIMIT, (h, apart(got[:, part], want))


@DTYPES
@pytest.mark.parametrize("pos, n", [(0, 1), (37, 1), (20, 40), (0, 70), (3000, 2)])
def test_attend_head_beside_nan(dev, dtype, pos, n):
    """A key or value row of NaN in kv head 1, head 0's row there as it was: head 0's outputs stay bit for bit."""
    nq, nkv, hd = 6, 2, 128
    c, k, v, rng = filled(dev, dtype, nkv, hd, pos + n, 5)
    q = rng.standard_normal((n, nq, hd)).astype(np.float32)
    want = dev.kv4_attend(c, q, pos)
    at = pos + n // 2
    for plane in (0, 1):
        rows = np.stack([k[at], v[at]]).astype(np.float32)
        rows[plane, 1, 7] = np.nan
        dev.kv4_append(c, rows.reshape(1, -1), 0, at)
        back = dev.kv4_rows(c, at, 1)
        assert np.array_equal(back[0][0, 0], k[at, 0].astype(np.float32)) and np.array_equal(back[1][0, 0], v[at, 0].astype(np.float32))
        got = dev.kv4_attend(c, q, pos)
        assert np.array_equal(got[:, :nq // 2], want[:, :nq // 2])
        assert np.array_equal(got[:at - pos], want[:at - pos])
        bad = got[at - pos:, nq // 2:] if plane == 0 else got[at - pos:, nq // 2:, :32]
        assert np.isnan(bad).all()
