"""The 4-bit K/V cache: norm and rotation of query and key heads, the writer, the read-back and the attention, each against its formula
in 64 bits, and a prompt with decode steps behind it through all of them."""
import ctypes as C

import numpy as np
import pytest

import l3m_amd as A
from weights import MXFP4, Q4_0

pytestmark = pytest.mark.gpu
DTYPES = pytest.mark.parametrize("dtype", [Q4_0, MXFP4], ids=["q4_0", "mxfp4"])
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6])


@pytest.fixture(autouse=True)
def clean(dev):
    yield
    dev.free_all()


def stored(dtype, x):
    """The values the cache holds for rows x [..., hd], by the file formats' quantizer (l3m_quantize_row) on zero-padded blocks."""
    hd = x.shape[-1]
    b = np.zeros(x.shape[:-1] + (-(-hd // 32) * 32,), np.float32)
    b[..., :hd] = x
    raw = A.quantize_rows(dtype, b.reshape(-1, 32))
    if dtype == Q4_0:
        d, q = raw[:, :2].copy().view(np.float16).astype(np.float64), raw[:, 2:]
    else:
        d, q = np.exp2(raw[:, :1].astype(np.float64) - 127), raw[:, 1:]
    c = np.concatenate([q & 15, q >> 4], 1).astype(np.int64)
    v = (c - 8.0 if dtype == Q4_0 else E2M1[c]) * d
    return v.reshape(b.shape)[..., :hd]


def turned(x, w, eps, halves, table):
    """Norm (w None: none) and rotation (table [n][hd / 2][2] None: none) of x [n][heads][hd] in 64 bits."""
    y = x.astype(np.float64)
    if w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * w
    if table is not None:
        c, s = (table[:, None, :, i].astype(np.float64) for i in (0, 1))
        hd = x.shape[-1]
        a, b = (y[..., :hd // 2], y[..., hd // 2:]) if halves else (y[..., 0::2], y[..., 1::2])
        a, b = a * c - b * s, a * s + b * c
        y = np.concatenate([a, b], -1) if halves else np.stack([a, b], -1).reshape(y.shape)
    return y


def table_of(ctx, hd):
    t = np.zeros(ctx * hd, np.float32)
    A.lib().l3m_rope_table(t.ctypes.data_as(C.POINTER(C.c_float)), ctx, hd, 10000.0)
    return t.reshape(ctx, hd // 2, 2)


def summed(dtype, x):
    """The magnitude of the terms a sum over x's codes is made of. mxfp4: |x|. q4_0: x = (u - 8) d is summed as u d, u in 0..15, and -8 d; the
    block's largest value has u = 0, so |8 d| is its magnitude, and a partial sum's terms are at most |u d| + |8 d| <= |x| + 2 |8 d|."""
    if dtype == MXFP4:
        return np.abs(x)
    wide = np.abs(x)
    for b in range(0, x.shape[-1], 32):
        wide[..., b:b + 32] += 2 * wide[..., b:b + 32].max(-1, keepdims=True)
    return wide


def attended(dtype, q, k, v, pos):
    """out and the bound of its error: q [n][nq][hd], k, v [pos + n][nkv][hd] in 64 bits.

    A score is a sum of hd products in float32: off by (hd + 16) 2^-24 of the sum of its terms' magnitudes at most; a weight by twice that
    (itself and the sum's). A weight (q4_0: with its scale) is held in two parts of 11 bits, half a step of the second being 2^-22, and no
    less than 2^-25 where the largest is 2^7 at least: 2^-32 of the largest weight times the largest value for each position; mxfp4's values
    are exact down to 2^-33 of the largest. And a float32 rounding of its terms for each of the sums' steps: 32 positions each, and those
    that join partial results."""
    n, nq, hd = q.shape
    nkv, g = k.shape[1], q.shape[1] // k.shape[1]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for h in range(nq):
        kh, vh, qh = k[:, h // g], v[:, h // g], q[:, h].astype(np.float64)
        s = qh @ kh.T / np.sqrt(hd)
        mag = np.abs(qh) @ summed(dtype, kh).T / np.sqrt(hd)
        late = np.arange(len(k))[None] > pos + np.arange(n)[:, None]
        s[late], mag[late] = -np.inf, 0
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        out[:, h] = p @ vh
        off = 2 * (hd + 16) * 2.0 ** -24 * mag.max(1) + 2.0 ** -21
        least = (len(k) * p.max(1) + 1) * 2.0 ** -32 * np.abs(vh).max()
        tol[:, h] = off[:, None] * (p @ np.abs(vh)) + (len(k) / 32 + 64) * 2.0 ** -24 * (p @ summed(dtype, vh)) + least[:, None] + 1e-42
    return out, tol


def near(got, want, tol):
    off = np.abs(got - want) / tol
    assert np.isfinite(got).all() and off.max() <= 1, off.max()


# ---------------------------------------------------------------- norm and rotation

@pytest.mark.parametrize("norm, rot", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("hd", [2, 6, 48, 64, 80, 128, 130, 254, 256])
@pytest.mark.parametrize("halves", [False, True])
def test_qk_norm_rope(dev, hd, halves, norm, rot):
    for n, nq, nkv, pos, gap in ((1, 3, 1, 0, 0), (7, 4, 2, 13, 0), (33, 5, 0, 3, 5), (2, 0, 3, 100, 1)):
        rng = np.random.default_rng(hd + n)
        rows = (rng.standard_normal((n, (nq + nkv) * hd + gap)) * 3).astype(np.float32)
        wq, wk = ((1 + rng.standard_normal(hd) / 4).astype(np.float32) for _ in range(2))
        table = table_of(pos + n, hd)
        q, k = dev.qk_norm_rope(rows, nq, nkv, hd, wq if norm else None, wk if norm else None, 1e-5, halves, pos, dev.put(table) if rot else None)
        x = rows[:, :(nq + nkv) * hd].reshape(n, nq + nkv, hd)
        for got, part, w in ((q, x[:, :nq], wq), (k, x[:, nq:], wk)):
            want = turned(part, w if norm else None, 1e-5, halves, table[pos:] if rot else None)
            # one rounding to float32, off by half a step; what 64 bits lose is below 1e-13
            assert np.all(np.abs(got - want) <= np.abs(want) * 2.0 ** -24 * (1 + 1e-6) + 1e-13)


def test_qk_norm_rope_special(dev):
    """In place for one token; rows of zeros (s = 1 / sqrt(eps)); values whose squares leave float32; not finite values stay in their head."""
    rng = np.random.default_rng(1)
    hd, nq, nkv = 64, 3, 2
    rows = rng.standard_normal((1, 7 * hd)).astype(np.float32)
    rows[0, :hd] = 0
    rows[0, hd:2 * hd] *= 1e30
    rows[0, 3 * hd + 5] = np.nan
    w, table = (1 + rng.standard_normal(hd) / 4).astype(np.float32), table_of(9, hd)
    p, dw = dev.put(rows), dev.put(w)
    assert dev.lib.l3m_k_qk_norm_rope(p, p + 4 * nq * hd, p, 7 * hd, 1, nq, nkv, hd, dw, dw, 1e-5, 0, 8, dev.put(table), None) == 0
    got = dev.get(p, (7, hd), np.float32)
    want = turned(rows.reshape(1, 7, hd), w, 1e-5, False, table[8:])[0]
    assert np.all(got[0] == 0) and np.isnan(got[3]).all() and np.array_equal(got[5:], rows.reshape(7, hd)[5:])
    for i in (1, 2, 4):
        assert np.all(np.abs(got[i] - want[i]) <= np.abs(want[i]) * 2.0 ** -24 * (1 + 1e-6) + 1e-13)


# ---------------------------------------------------------------- writer and read-back

@DTYPES
@pytest.mark.parametrize("hd", [8, 32, 40, 64, 80, 128, 200, 256])
def test_append_rows(dev, dtype, hd):
    """Rows go in at odd places, over what was there, and come back as the file formats hold them; the other positions stay as they were."""
    rng = np.random.default_rng(hd)
    nkv, cap, nq = 3, 77, 2
    c = dev.kv4(dtype, nkv, hd, cap)
    held = np.zeros((2, cap, nkv, hd))
    w, table = (1 + rng.standard_normal(hd) / 4).astype(np.float32), table_of(cap, hd)
    for pos, n, plain in ((0, 77, True), (5, 3, True), (7, 2, False), (8, 8, True), (30, 40, False), (76, 1, False), (64, 13, True), (3, 1, True)):
        rows = rng.standard_normal((n, (nq + 2 * nkv) * hd + 3)).astype(np.float32)
        x = rows[:, :-3].reshape(n, nq + 2 * nkv, hd)
        q = dev.kv4_append(c, rows, nq, pos, *((None, None) if plain else (w, w)), 1e-5, True, None if plain else dev.put(table))
        turn = (lambda y: y.astype(np.float64)) if plain else (lambda y: turned(y, w, 1e-5, True, table[pos:pos + n]))
        assert np.array_equal(q, turn(x[:, :nq]).astype(np.float32))
        held[0, pos:pos + n] = stored(dtype, turn(x[:, nq:nq + nkv]).astype(np.float32))
        held[1, pos:pos + n] = stored(dtype, x[:, nq + nkv:])
        k, v = dev.kv4_rows(c, 0, cap)
        assert np.array_equal(k, held[0].astype(np.float32)) and np.array_equal(v, held[1].astype(np.float32)), (pos, n)
    k, v = dev.kv4_rows(c, 31, 5)
    assert np.array_equal(k, held[0, 31:36].astype(np.float32)) and np.array_equal(v, held[1, 31:36].astype(np.float32))


@DTYPES
def test_append_edges(dev, dtype):
    """Blocks of zeros, equal largest values of both signs, values halfway between two codes, the smallest and largest scales, and values that
    are not finite (their block reads NaN, no other)."""
    hd, nkv = 64, 1
    x = np.zeros((8, hd), np.float32)
    x[1, :32] = np.where(np.arange(32) % 2, 1.5, -1.5)
    x[2, :32] = -x[1, :32]
    x[3, :32] = np.arange(32) / 4 - 4                                 # halfway values of both formats
    x[4, :32] = np.linspace(-1, 1, 32) * 2.0 ** -120
    x[4, 32:] = 2.0 ** -149
    x[5, :32] = np.linspace(-1, 1, 32) * (3e5 if dtype == Q4_0 else 2.0 ** 127)
    x[6, 3], x[6, 40] = np.nan, 2
    x[7, :32], x[7, 63] = 1, np.inf
    want = stored(dtype, np.where(np.isfinite(x), x, 0))
    if dtype == MXFP4:
        want[4, 32:] = 0                                             # exponents end at 2^-126
    want[6, :32], want[7, 32:] = np.nan, np.nan
    c = dev.kv4(dtype, nkv, hd, 8)
    dev.kv4_append(c, np.concatenate([x, x], 1), 0, 0)
    for got in dev.kv4_rows(c, 0, 8):
        assert np.array_equal(got[:, 0], want.astype(np.float32), equal_nan=True)
    if dtype == Q4_0:                                                # past f16's scales: the largest scale
        c2 = dev.kv4(dtype, 1, 32, 1)
        y = np.zeros((1, 64), np.float32)
        y[0, 0], y[0, 32] = 1e9, -1e9
        dev.kv4_append(c2, y, 0, 0)
        k, v = dev.kv4_rows(c2, 0, 1)
        assert k[0, 0, 0] == 8 * 65504 and v[0, 0, 0] == -8 * 65504 and not k[0, 0, 1:].any()


# ---------------------------------------------------------------- attention

def filled(dev, dtype, nkv, hd, n, seed, cap=None, dirty=False):
    """A cache with n positions and what it holds [n][nkv][hd]."""
    rng = np.random.default_rng(seed)
    c = dev.kv4(dtype, nkv, hd, cap or n)
    if dirty:
        size = dev.lib.l3m_kv4_bytes(dtype, nkv, hd, cap or n)
        assert dev.lib.l3m_dev_upload(c.kq, np.full(size, 0xFF, np.uint8).ctypes.data, size) == 0
    rows = rng.standard_normal((n, 2 * nkv * hd)).astype(np.float32)
    dev.kv4_append(c, rows, 0, 0)
    k, v = dev.kv4_rows(c, 0, n)
    return c, k.astype(np.float64), v.astype(np.float64), rng


@DTYPES
@pytest.mark.parametrize("hd", [8, 32, 48, 64, 96, 128, 160, 200, 224, 256])
@pytest.mark.parametrize("nq, nkv", [(1, 1), (12, 12), (9, 3), (8, 1), (34, 2)])
def test_attend_one_token(dev, dtype, hd, nq, nkv):
    for seen in (1, 2, 31, 32, 33, 64, 127, 300, 1025):
        c, k, v, rng = filled(dev, dtype, nkv, hd, seen, hd + seen)
        q = rng.standard_normal((1, nq, hd)).astype(np.float32) * 2
        near(dev.kv4_attend(c, q, seen - 1), *attended(dtype, q, k, v, seen - 1))
        dev.free_all()


@DTYPES
@pytest.mark.parametrize("hd, nq, nkv", [(64, 9, 3), (128, 8, 2), (80, 10, 2), (48, 6, 6), (256, 4, 1), (8, 3, 3), (160, 17, 1)])
@pytest.mark.parametrize("pos, n", [(0, 2), (0, 33), (0, 300), (1, 5), (31, 17), (100, 64), (998, 5), (600, 130)])
def test_attend_tokens(dev, dtype, hd, nq, nkv, pos, n):
    c, k, v, rng = filled(dev, dtype, nkv, hd, pos + n, pos + n)
    q = rng.standard_normal((n, nq, hd)).astype(np.float32) * 2
    got = dev.kv4_attend(c, q, pos)
    near(got, *attended(dtype, q, k, v, pos))
    assert np.array_equal(got, dev.kv4_attend(c, q, pos))            # the same sums in the same order


@DTYPES
@pytest.mark.parametrize("seen", [4001, 20011, 70000])
def test_attend_long(dev, dtype, seen):
    nq, nkv, hd = 8, 2, 128
    c, k, v, rng = filled(dev, dtype, nkv, hd, seen, seen)
    q = rng.standard_normal((1, nq, hd)).astype(np.float32) * 2
    near(dev.kv4_attend(c, q, seen - 1), *attended(dtype, q, k, v, seen - 1))
    q = rng.standard_normal((3, nq, hd)).astype(np.float32)
    near(dev.kv4_attend(c, q, seen - 3), *attended(dtype, q, k, v, seen - 3))


@DTYPES
@pytest.mark.parametrize("hd", [40, 128])
def test_attend_leaves_out_what_follows(dev, dtype, hd):
    """Memory that was never cleared (every bit set: scales that are not finite) and rows that are not finite, behind a token's position,
    leave its output bit for bit what it is over a clean cache; at its position and before, they reach it."""
    nq, nkv = 6, 2
    for pos, n in ((0, 1), (37, 1), (20, 40), (0, 70)):
        seen = pos + n
        q = np.random.default_rng(9).standard_normal((n, nq, hd)).astype(np.float32)
        c0, k, v, _ = filled(dev, dtype, nkv, hd, seen, 5, cap=seen + 90)
        c1 = filled(dev, dtype, nkv, hd, seen, 5, cap=seen + 90, dirty=True)[0]
        want = dev.kv4_attend(c0, q, pos)
        near(want, *attended(dtype, q, k, v, pos))
        assert np.array_equal(dev.kv4_attend(c1, q, pos), want)
        at = pos + n // 2                                             # a key of NaN in the middle, for kv head 1
        bad = np.zeros((1, 2 * nkv * hd), np.float32)
        bad[0, hd] = np.nan
        dev.kv4_append(c0, bad, 0, at)
        got = dev.kv4_attend(c0, q, pos)
        assert np.array_equal(got[:, :nq // 2], dev.kv4_attend(c0, q, pos)[:, :nq // 2]) and np.isfinite(got[:, :nq // 2]).all()
        assert np.array_equal(got[:at - pos], want[:at - pos]) and np.isnan(got[at - pos:, nq // 2:]).all()


def test_attend_value_not_finite(dev):
    """A V row that is not finite reaches the tokens from its position on, in its block of dimensions and kv head alone."""
    nq, nkv, hd, n = 4, 2, 64, 50
    c, k, v, rng = filled(dev, Q4_0, nkv, hd, n, 3)
    q = rng.standard_normal((n, nq, hd)).astype(np.float32)
    want = dev.kv4_attend(c, q, 0)
    rows = np.concatenate([k[20], v[20]]).reshape(1, -1).astype(np.float32)
    rows[0, (nkv + 1) * hd + 40] = np.inf
    dev.kv4_append(c, rows, 0, 20)
    got = dev.kv4_attend(c, q, 0)
    assert np.array_equal(got[:20], want[:20]) and np.isnan(got[20:, 2:, 32:]).all()
    assert np.isfinite(got[20:, :2]).all() and np.isfinite(got[20:, 2:, :32]).all()


@DTYPES
@pytest.mark.parametrize("hd", [40, 128, 200])
def test_attend_position_never_written(dev, dtype, hd):
    """A position in the middle that was never written, its memory holding infinite f16 scales: the call ends, and the tokens before it are
    what they are over the whole cache."""
    nq, nkv, n = 4, 2, 40
    size, rng = dev.lib.l3m_kv4_bytes(dtype, nkv, hd, n), np.random.default_rng(4)
    rows, q = rng.standard_normal((n, 2 * nkv * hd)).astype(np.float32), rng.standard_normal((n, nq, hd)).astype(np.float32)
    whole, c = dev.kv4(dtype, nkv, hd, n), dev.kv4(dtype, nkv, hd, n)
    assert dev.lib.l3m_dev_upload(c.kq, np.full(size // 2, 0x7C00, np.uint16).ctypes.data, size) == 0
    dev.kv4_append(whole, rows, 0, 0)
    dev.kv4_append(c, rows[:20], 0, 0)
    dev.kv4_append(c, rows[21:], 0, 21)
    got, want = dev.kv4_attend(c, q, 0), dev.kv4_attend(whole, q, 0)
    assert np.array_equal(got[:20], want[:20])
    if dtype == Q4_0:
        assert not np.isfinite(got[20:]).any()


@DTYPES
@pytest.mark.parametrize("hd", [32, 64, 128, 200])
def test_attend_query_not_finite(dev, dtype, hd):
    """A query that holds a NaN or an infinity gives NaN, its neighbours' outputs stay as they are."""
    nq, nkv, n = 6, 2, 40
    for bad in (np.nan, np.inf, -np.inf):
        c, k, v, rng = filled(dev, dtype, nkv, hd, n, 3)
        q = rng.standard_normal((n, nq, hd)).astype(np.float32)
        want = dev.kv4_attend(c, q, 0)
        q[17, 4, hd - 3] = bad
        got = dev.kv4_attend(c, q, 0)
        assert np.isnan(got[17, 4]).all()
        got[17, 4] = want[17, 4]
        assert np.array_equal(got, want)
        dev.free_all()


@DTYPES
def test_attend_query_sizes(dev, dtype):
    """Queries of very different sizes, in a row and between rows, down to subnormal ones and zeros."""
    nq, nkv, hd, seen = 8, 1, 128, 100
    c, k, v, rng = filled(dev, dtype, nkv, hd, seen, 6)
    q = rng.standard_normal((1, nq, hd)).astype(np.float32) * np.exp2(rng.integers(-20, 1, (1, nq, hd))).astype(np.float32)
    q[0, 1] *= 2.0 ** -110
    q[0, 2] *= 2.0 ** -130
    q[0, 3] = 0
    q[0, 4] *= 2.0 ** 6
    near(dev.kv4_attend(c, q, seen - 1), *attended(dtype, q, k, v, seen - 1))


@DTYPES
def test_attend_large_scores(dev, dtype):
    """Scores of hundreds, the largest in any part of the cache: the others' weights vanish."""
    nq, nkv, hd, seen = 2, 1, 64, 3000
    for at in (0, 40, 1499, 2999):
        rng = np.random.default_rng(at)
        rows = rng.standard_normal((seen, 2 * hd)).astype(np.float32)
        rows[at, :hd] *= 20
        c = dev.kv4(dtype, nkv, hd, seen)
        dev.kv4_append(c, rows, 0, 0)
        k, v = (x.astype(np.float64) for x in dev.kv4_rows(c, 0, seen))
        q = np.stack([k[at, 0], -k[at, 0]])[None].astype(np.float32)
        near(dev.kv4_attend(c, q, seen - 1), *attended(dtype, q, k, v, seen - 1))


@DTYPES
def test_attend_mixed_scales(dev, dtype):
    """V rows of very different sizes (2^-20 .. 2^10), keys near zero: every position counts alike."""
    nq, nkv, hd, seen = 3, 1, 96, 200
    rng = np.random.default_rng(4)
    rows = rng.standard_normal((seen, 2, hd)).astype(np.float32)
    rows[:, 0] *= 1e-3
    rows[:, 1] *= np.exp2(rng.integers(-20, 11, (seen, 1)))
    c = dev.kv4(dtype, nkv, hd, seen)
    dev.kv4_append(c, rows.reshape(seen, -1), 0, 0)
    k, v = (x.astype(np.float64) for x in dev.kv4_rows(c, 0, seen))
    q = rng.standard_normal((1, nq, hd)).astype(np.float32)
    near(dev.kv4_attend(c, q, seen - 1), *attended(dtype, q, k, v, seen - 1))


@DTYPES
@pytest.mark.parametrize("sizes", [(-100, -100, -100), (-15, -15, -15), (100, 100, 100), (14, 14, 14), (-100, 0, 90), (-15, 0, 14), (90, 0, -100), (14, -3, -15), (0, 14, 0)],
                         ids=str)
def test_attend_value_sizes(dev, dtype, sizes):
    """V rows of 2^sizes in the first, middle and last third, past what f16 holds (mxfp4) and at the ends of f16 scales (q4_0, whose sizes end
    there): one token, and a prompt, whose rows see more and more of them."""
    if dtype == Q4_0 and max(map(abs, sizes)) > 15:
        pytest.skip("past q4_0's f16 scales")
    nq, nkv, hd = 3, 1, 64
    for seen, n in ((1500, 1), (200, 200)):
        rng = np.random.default_rng(seen)
        rows = rng.standard_normal((seen, 2, hd)).astype(np.float32)
        rows[:, 1] *= np.exp2(np.repeat(np.float32(sizes), -(-seen // 3))[:seen])[:, None]
        c = dev.kv4(dtype, nkv, hd, seen)
        dev.kv4_append(c, rows.reshape(seen, -1), 0, 0)
        k, v = (x.astype(np.float64) for x in dev.kv4_rows(c, 0, seen))
        q = rng.standard_normal((n, nq, hd)).astype(np.float32)
        near(dev.kv4_attend(c, q, seen - n), *attended(dtype, q, k, v, seen - n))
        dev.free_all()


def each_near(dtype, got, q, k, v, pos):
    """Every token against what it sees alone: the bound of its error knows nothing of the positions behind it."""
    for t in range(len(q)):
        near(got[t:t + 1], *attended(dtype, q[t:t + 1], k[:pos + t + 1], v[:pos + t + 1], pos + t))


@DTYPES
@pytest.mark.parametrize("sizes", ["high", "low", "rising", "top"])
@pytest.mark.parametrize("nq, nkv, hd, n", [(6, 2, 64, 50), (2, 1, 200, 70), (64, 64, 96, 250)], ids=str)
def test_attend_sizes_behind(dev, dtype, nq, nkv, hd, n, sizes):
    """V rows whose size changes from one position of a tile to the next, up to the ends of what the scales hold: a token is as near its formula as
    if the positions behind it were not there, whether the call's own tokens wrote them or an earlier, longer sequence did. (64, 64, 96, 250: two
    columns of rows a workgroup.)"""
    top, bottom = (14, -14) if dtype == Q4_0 else (123, -110)
    rng, at = np.random.default_rng(n), np.arange(n)
    e = {"high": np.where(at < 20, 0, top), "low": np.where(at < 20, 0, bottom), "rising": bottom + (top - bottom) * at // n, "top": np.full(n, top)}[sizes]
    rows = rng.standard_normal((n, 2, nkv, hd)).astype(np.float32)
    rows[:, 1] *= np.exp2(e.astype(np.float64)).astype(np.float32)[:, None, None]
    assert np.isfinite(rows).all()
    c = dev.kv4(dtype, nkv, hd, n)
    dev.kv4_append(c, rows.reshape(n, -1), 0, 0)
    k, v = (x.astype(np.float64) for x in dev.kv4_rows(c, 0, n))
    q = rng.standard_normal((n, nq, hd)).astype(np.float32)
    g = nq // nkv
    all_heads = dev.kv4_attend(c, q, 0)
    few = dev.kv4_attend(c, q[10:15], 10)
    for h in sorted({0, nkv // 2, nkv - 1}):
        heads = slice(h * g, (h + 1) * g)
        each_near(dtype, all_heads[:, heads], q[:, heads], k[:, h:h + 1], v[:, h:h + 1], 0)
        each_near(dtype, few[:, heads], q[10:15, heads], k[:15, h:h + 1], v[:15, h:h + 1], 10)


@DTYPES
@pytest.mark.parametrize("hd", [40, 64, 96, 128])
def test_attend_many_rows(dev, dtype, hd):
    """As many rows as take two columns a workgroup (mxfp4): heads of their own formula, a K and a V row that are not finite for the tokens
    from theirs on alone."""
    nq, nkv, n = 128, 64, 150
    c, k, v, rng = filled(dev, dtype, nkv, hd, n, hd)
    q = rng.standard_normal((n, nq, hd)).astype(np.float32)
    got = dev.kv4_attend(c, q, 0)
    for h in (0, 31, 63):
        near(got[:, 2 * h:2 * h + 2], *attended(dtype, q[:, 2 * h:2 * h + 2], k[:, h:h + 1], v[:, h:h + 1], 0))
    rows = np.concatenate([k[50], v[50]]).reshape(1, -1).astype(np.float32)
    rows[0, 3 * hd], rows[0, (nkv + 5) * hd] = np.nan, np.inf
    dev.kv4_append(c, rows, 0, 50)
    bad = dev.kv4_attend(c, q, 0)
    assert np.array_equal(bad[:50], got[:50])
    assert np.isnan(bad[50:, 6:8]).all() and np.isnan(bad[50:, 10:12, :32]).all()
    others = [h for h in range(nq) if h // 2 not in (3, 5)]
    assert np.isfinite(bad[:, others]).all() and np.isfinite(bad[:, 10:12, 32:]).all()


def test_out_may_be_q(dev):
    nq, nkv, hd = 8, 2, 128
    for n, seen in ((1, 5000), (70, 100)):
        c, k, v, rng = filled(dev, MXFP4, nkv, hd, seen, 8)
        q = rng.standard_normal((n, nq, hd)).astype(np.float32)
        want = dev.kv4_attend(c, q, seen - n)
        p, size = dev.put(q), dev.lib.l3m_kv4_work_bytes(C.byref(c), n, nq)
        assert dev.lib.l3m_k_kv4_attend(p, p, C.byref(c), n, nq, seen - n, dev.alloc(size), size, None) == 0
        assert np.array_equal(dev.get(p, q.shape, np.float32), want)


def test_nothing_past_the_outputs(dev):
    nq, nkv, hd, n, seen = 5, 5, 48, 3, 50
    c, k, v, rng = filled(dev, Q4_0, nkv, hd, seen, 8)
    q, fence = rng.standard_normal((n, nq, hd)).astype(np.float32), np.full(64, 7, np.float32)
    p = dev.put(np.concatenate([np.zeros(q.size, np.float32), fence]))
    size = dev.lib.l3m_kv4_work_bytes(C.byref(c), n, nq)
    work = dev.put(np.full(size + 256, 0xAB, np.uint8))
    assert dev.lib.l3m_k_kv4_attend(p, dev.put(q), C.byref(c), n, nq, seen - n, work, size, None) == 0
    assert np.all(dev.get(p, q.size + 64, np.float32)[q.size:] == 7) and np.all(dev.get(work, size + 256, np.uint8)[size:] == 0xAB)
    for call in (lambda: dev.lib.l3m_k_kv4_rows(C.byref(c), p, None, 47, 3, None), lambda: dev.lib.l3m_k_kv4_rows(C.byref(c), None, p, 47, 3, None)):
        assert call() == 0
        assert np.all(dev.get(p, q.size + 64, np.float32)[n * nkv * hd:][-64:] == 7)


@DTYPES
def test_planes_past_32_bits(dev, dtype):
    """Heads whose planes begin past 4 GiB, and positions past 4 GiB of one head's."""
    hd = 256
    for nkv, cap, spots in ((5, 1 << 23, (0, (1 << 23) - 40)), (1, (1 << 25) + 100, (0, (1 << 25) + 60))):
        mem = dev.lib.l3m_kv4_bytes(dtype, nkv, hd, cap)
        c = dev.kv4(dtype, nkv, hd, cap)
        assert mem > 8 << 30
        rng = np.random.default_rng(cap)
        for pos in spots:
            x = rng.standard_normal((40, 2, nkv, hd)).astype(np.float32)
            dev.kv4_append(c, x.reshape(40, -1), 0, pos)
            k, v = dev.kv4_rows(c, pos, 40)
            assert np.array_equal(k, stored(dtype, x[:, 0]).astype(np.float32)) and np.array_equal(v, stored(dtype, x[:, 1]).astype(np.float32))
            if pos == 0:
                q = rng.standard_normal((3, nkv, hd)).astype(np.float32)
                near(dev.kv4_attend(c, q, 37), *attended(dtype, q, k.astype(np.float64), v.astype(np.float64), 37))
        dev.free_all()


@DTYPES
def test_attend_past_32_bits(dev, dtype):
    """One head's positions past 4 GiB of codes: rows of zeros but for 90, whose scores stand out. Weights add up over the whole length, outputs over
    the 90."""
    hd, nq, cap, step = 256, 2, (1 << 25) + 100, 1 << 18
    c, rng = dev.kv4(dtype, 1, hd, cap), np.random.default_rng(1)
    zeros = dev.alloc(8 * hd * step)
    assert dev.lib.l3m_dev_upload(zeros, np.zeros(2 * hd * step, np.float32).ctypes.data, 8 * hd * step) == 0
    for pos in range(0, cap, step):
        assert dev.lib.l3m_k_kv4_append(C.byref(c), None, zeros, 2 * hd, min(step, cap - pos), 0, None, None, 0.0, 0, pos, None, None) == 0
    ks, vs = [], []
    for pos in (5, (1 << 24) + 17, cap - 30):
        dev.kv4_append(c, (rng.standard_normal((30, 2, hd)) * [[[4], [1]]]).astype(np.float32).reshape(30, -1), 0, pos)
        k, v = dev.kv4_rows(c, pos, 30)
        ks.append(k[:, 0].astype(np.float64)), vs.append(v[:, 0].astype(np.float64))
    k, v, q = np.concatenate(ks), np.concatenate(vs), (rng.standard_normal((1, nq, hd)) * 1.5).astype(np.float32)
    got = dev.kv4_attend(c, q, cap - 1)
    s = q[0].astype(np.float64) @ k.T / 16
    p = np.exp(s)
    p /= p.sum(1, keepdims=True) + cap - 90
    off = 2 * (hd + 16) * 2.0 ** -24 * (np.abs(q[0].astype(np.float64)) @ summed(dtype, k).T / 16).max(1) + 2.0 ** -21 + (cap / 32 + 64) * 2.0 ** -24
    near(got[0], p @ v, off[:, None] * (p @ summed(dtype, v)) + 91 * 2.0 ** -32 * np.abs(v).max())


# ---------------------------------------------------------------- streams, graphs, and all of them together

def test_streams_and_capture(dev):
    """Two streams at once, each with its workspace; then a decode step's calls recorded into a graph and replayed between eager calls."""
    hip = C.CDLL("libamdhip64.so")
    nq, nkv, hd, seen = 8, 2, 128, 6000
    sets = [filled(dev, dt, nkv, hd, seen, 20 + i) for i, dt in enumerate((Q4_0, MXFP4))]
    qs = [s[3].standard_normal((1, nq, hd)).astype(np.float32) for s in sets]
    want = [dev.kv4_attend(s[0], q, seen - 1) for s, q in zip(sets, qs)]
    streams, size = [], dev.lib.l3m_kv4_work_bytes(C.byref(sets[0][0]), 1, nq)
    for _ in sets:
        st = C.c_void_p()
        assert hip.hipStreamCreateWithFlags(C.byref(st), 1) == 0
        streams.append(st)
    bufs = [(dev.alloc(q.nbytes), dev.put(q), dev.alloc(size)) for q in qs]
    for _ in range(20):
        for (o, q, w), s, st in zip(bufs, sets, streams):
            assert dev.lib.l3m_k_kv4_attend(o, q, C.byref(s[0]), 1, nq, seen - 1, w, size, st) == 0
    assert hip.hipDeviceSynchronize() == 0
    for b, x in zip(bufs, want):
        assert np.array_equal(dev.get(b[0], x.shape, np.float32), x)
    rng = np.random.default_rng(2)
    rows = rng.standard_normal((1, (nq + 2 * nkv) * hd)).astype(np.float32)
    w, table = dev.put(np.ones(hd, np.float32)), dev.rope_table(seen, hd, 10000.0)
    c, st, p, dq = sets[0][0], streams[0], dev.put(rows), dev.alloc(4 * nq * hd)

    def step(stream):
        assert dev.lib.l3m_k_kv4_append(C.byref(c), dq, p, rows.size, 1, nq, w, w, 1e-5, 0, seen - 1, table, stream) == 0
        assert dev.lib.l3m_k_kv4_attend(bufs[0][0], dq, C.byref(c), 1, nq, seen - 1, bufs[0][2], size, stream) == 0

    graph, ex = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(st, 1) == 0
    step(st)
    assert hip.hipStreamEndCapture(st, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0)) == 0
    for _ in range(4):
        rows = rng.standard_normal(rows.shape).astype(np.float32)
        assert dev.lib.l3m_dev_upload(p, rows.ctypes.data, rows.nbytes) == 0
        step(None)
        eager = dev.get(bufs[0][0], want[0].shape, np.float32)
        assert hip.hipGraphLaunch(ex, st) == 0 and hip.hipStreamSynchronize(st) == 0
        assert np.array_equal(dev.get(bufs[0][0], want[0].shape, np.float32), eager) and not np.array_equal(eager, want[0])
    assert hip.hipGraphExecDestroy(ex) == 0 and hip.hipGraphDestroy(graph) == 0
    for s in streams:
        assert hip.hipStreamDestroy(s) == 0


@DTYPES
def test_prompt_then_steps(dev, dtype):
    """A prompt of 70 tokens and 6 steps behind it, each through the writer and the attention, against the formulas in 64 bits; and the prompt in
    chunks gives what it gives at once."""
    rng = np.random.default_rng(11)
    nq, nkv, hd, cap = 6, 2, 64, 128
    w = [(1 + rng.standard_normal(hd) / 8).astype(np.float32) for _ in range(2)]
    table = table_of(cap, hd)
    dt = dev.put(table)
    c = dev.kv4(dtype, nkv, hd, cap)
    k, v = np.zeros((2, 0, nkv, hd))
    prompt = None
    for n in (70, 1, 1, 1, 1, 1, 1):
        pos = len(k)
        rows = rng.standard_normal((n, (nq + 2 * nkv) * hd)).astype(np.float32) * 2
        x = rows.reshape(n, -1, hd)
        q = dev.kv4_append(c, rows, nq, pos, *w, 1e-6, False, dt)
        k = np.concatenate([k, stored(dtype, turned(x[:, nq:nq + nkv], w[1], 1e-6, False, table[pos:pos + n]).astype(np.float32))])
        v = np.concatenate([v, stored(dtype, x[:, nq + nkv:])])
        q64 = turned(x[:, :nq], w[0], 1e-6, False, table[pos:pos + n])
        assert np.all(np.abs(q - q64) <= np.abs(q64) * 2.0 ** -24 * (1 + 1e-6) + 1e-13)
        got = dev.kv4_attend(c, q, pos)
        near(got, *attended(dtype, q, k, v, pos))
        prompt = (rows, got) if prompt is None else prompt
    c2, at = dev.kv4(dtype, nkv, hd, cap), 0
    for n in (1, 13, 32, 24):
        q = dev.kv4_append(c2, prompt[0][at:at + n], nq, at, *w, 1e-6, False, dt)
        want, tol = attended(dtype, q, k[:at + n], v[:at + n], at)
        got = dev.kv4_attend(c2, q, at)
        near(got, want, tol)
        assert np.all(np.abs(got - prompt[1][at:at + n]) <= 2 * tol)
        at += n
    assert all(np.array_equal(a, b) for a, b in zip(dev.kv4_rows(c2, 0, 70), dev.kv4_rows(c, 0, 70)))
