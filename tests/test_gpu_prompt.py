"""Causal attention over packed prompts (l3m_k_attend_packed) against its formula in 64 bits."""
import ctypes as C

import numpy as np
import pytest

from serve import attended, bf16, from_bf16

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean(dev):
    yield
    dev.free_all()


def rows(rng, n, h, hd, size=1.0):
    return bf16(rng.standard_normal((n, h, hd)) * size)


def check(got, q, k, v, lens, pick=None):
    """Rows of each prompt (of long ones some) within the bound: a weight's rounding to bf16 is off by 2^-8 of it, the result's by 2^-8. A weight is a
    float32 2^(s - m), its largest 1 at least: one of less than 2^-126 of the largest is no normal number and may be zero, off by less than that."""
    at = 0
    for n in lens:
        part = slice(at, at + n)
        t = np.arange(n) if pick is None or n <= pick else np.unique(np.linspace(0, n - 1, pick).astype(int))
        qx, kx, vx = (from_bf16(x[part]) for x in (q, k, v))
        want, tol = attended(qx[t], kx, vx, t + 1, 2.0 ** -8, 2.0 ** -126)
        tol = tol + 2.0 ** -8 * (np.abs(want) + tol)
        off = np.abs(from_bf16(got[part][t]) - want) - tol
        assert np.all(off <= 0), (n, off.max())
        at += n


@pytest.mark.parametrize("hd", [8, 32, 40, 64, 80, 96, 128, 160, 192, 224, 256])
def test_heads(dev, hd):
    """Head sizes, one or several query heads a kv head; prompts of none, one, and around a tile's and a wavefront's ends."""
    rng = np.random.default_rng(hd)
    for nkv, g, lens in ((1, 1, [1, 0, 31, 32, 33, 0, 63, 64, 65, 129]), (2, 3, [5, 128, 0, 70]), (3, 4, [200, 1, 1, 17]), (1, 17, [40, 66])):
        n = sum(lens)
        q, k, v = rows(rng, n, nkv * g, hd), rows(rng, n, nkv, hd), rows(rng, n, nkv, hd)
        check(dev.attend_packed(q, k, v, dev.batch(np.cumsum([0] + lens))), q, k, v, lens)
        dev.free_all()


@pytest.mark.parametrize("hd, nkv, g, lens", [(64, 3, 3, [1000, 2, 333]), (128, 2, 4, [1537, 64]), (128, 1, 8, [2100]), (256, 1, 2, [700, 90]), (64, 1, 1, [4099])])
def test_long(dev, hd, nkv, g, lens):
    rng = np.random.default_rng(len(lens))
    n = sum(lens)
    q, k, v = rows(rng, n, nkv * g, hd), rows(rng, n, nkv, hd), rows(rng, n, nkv, hd)
    check(dev.attend_packed(q, k, v, dev.batch(np.cumsum([0] + lens))), q, k, v, lens, pick=40)


def test_sizes(dev):
    """Scores so large that one position takes all weight, rising and falling along the prompt, and so small that all take the same."""
    rng = np.random.default_rng(1)
    n, hd = 300, 64
    for size in (1e-30, 1e-2, 6.0, 60.0):
        q, v = rows(rng, n, 2, hd, size), rows(rng, n, 1, hd)
        for ramp in (np.ones(n), np.linspace(0, 3, n), np.linspace(3, 0, n)):
            k = bf16(rng.standard_normal((n, 1, hd)) * ramp[:, None, None])
            check(dev.attend_packed(q, k, v, dev.batch([0, n])), q, k, v, [n])
        dev.free_all()
    v = bf16(np.exp(rng.uniform(-60, 60, (n, 1, hd))))
    check(dev.attend_packed(q, k, v, dev.batch([0, n])), q, k, v, [n])


def test_many_prompts(dev):
    """More prompts than a wavefront has lanes, most of them of one row."""
    rng = np.random.default_rng(2)
    lens = [int(x) for x in rng.choice([0, 1, 1, 1, 2, 40], 700)]
    n = sum(lens)
    q, k, v = rows(rng, n, 4, 64), rows(rng, n, 2, 64), rows(rng, n, 2, 64)
    check(dev.attend_packed(q, k, v, dev.batch(np.cumsum([0] + lens))), q, k, v, lens)


@pytest.mark.parametrize("hd", [40, 128, 256])
def test_not_finite(dev, hd):
    """NaN and infinities reach the rows that see them and change no bit of those before them, in other prompts or heads."""
    rng = np.random.default_rng(3)
    lens = [100, 90]
    q, k, v = rows(rng, 190, 4, hd), rows(rng, 190, 2, hd), rows(rng, 190, 2, hd)
    b = dev.batch([0, 100, 190])
    none = from_bf16(dev.attend_packed(q, k, v, b))
    vv, kk, qq = v.copy(), k.copy(), q.copy()
    vv[70, 1, 3], vv[99, 0, 5], vv[100, 0, 7] = 0x7F80, 0x7FC0, 0xFF80
    got = from_bf16(dev.attend_packed(q, k, vv, b))
    for rows_, heads, d in ((slice(70, 100), slice(2, 4), 3), (slice(99, 100), slice(0, 2), 5), (slice(100, 190), slice(0, 2), 7)):
        assert not np.isfinite(got[rows_, heads, d]).any()
        got[rows_, heads, d] = none[rows_, heads, d]
    # the rows before a value in their own tile are computed another way: bf16 of sums in another order, half a step each
    near = (slice(64, 70), slice(2, 4)), (slice(64, 99), slice(0, 2))
    for at in near:
        want, tol = attended(from_bf16(q[:100]), from_bf16(k[:100]), from_bf16(v[:100]), range(1, 101), 2.0 ** -8, 0.0)
        assert np.all(np.abs(got[at] - want[at]) <= (tol + 2.0 ** -8 * (np.abs(want) + tol))[at])
        got[at] = none[at]
    assert np.array_equal(got, none)
    kk[50, 0, 2] = 0x7FC0
    qq[120, 1, 0] = 0x7FC0
    got = from_bf16(dev.attend_packed(qq, kk, v, b))
    assert np.isnan(got[50:100, :2]).all() and np.isnan(got[120, 1]).all()
    got[50:100, :2], got[120, 1] = none[50:100, :2], none[120, 1]
    assert np.array_equal(got, none)


def test_strides(dev):
    """q, k and v as columns of fused rows with a gap, out in q's place; rows of no prompt and other columns left as they were."""
    rng = np.random.default_rng(4)
    n, nq, nkv, hd, width = 150, 6, 2, 48, 10 * 48 + 16
    x = bf16(rng.standard_normal((n, width)))
    b = dev.batch([10, 60, 60, 140], n=n)
    p = dev.put(x)
    lib, qw, kw = dev.lib, nq * hd, nkv * hd
    assert lib.l3m_k_attend_packed(p, width, p, width, p + 2 * qw, p + 2 * (qw + kw), width, C.byref(b), nq, nkv, hd, None) == 0
    got = dev.get(p, x.shape, np.uint16)
    q, k, v = x[:, :qw].reshape(n, nq, hd), x[:, qw:qw + kw].reshape(n, nkv, hd), x[:, qw + kw:qw + 2 * kw].reshape(n, nkv, hd)
    want = dev.attend_packed(q, k, v, b).reshape(n, qw)
    assert np.array_equal(got[:, qw:], x[:, qw:]) and np.array_equal(got[:10], x[:10]) and np.array_equal(got[140:], x[140:])
    assert np.array_equal(got[10:140, :qw], want[10:140])
    check(want[10:140].reshape(130, nq, hd), q[10:140], k[10:140], v[10:140], [50, 80])


def test_very_large_scores(dev):
    """Scores of 10^4 to 10^34, positive and negative, the largest ones apart by far or the same: one position takes all the weight, or several take equal parts."""
    rng = np.random.default_rng(5)
    n, hd = 300, 64
    for sign in (1, -1):
        top = 1.0 if sign > 0 else 2.0 ** -7
        k = np.zeros((n, 1, hd), np.float32)
        k[:, 0, 5] = 2.0 ** -rng.integers(1, 7, n)
        best = [0, 7, 133, 280]
        k[best, 0, 5] = top
        v = rows(rng, n, 1, hd)
        for e in (20, 40, 70, 100, 113):
            q = np.zeros((n, 3, hd), np.float32)
            q[..., 5] = sign * 2.0 ** e * (1 + np.arange(3) / 4)
            got = from_bf16(dev.attend_packed(bf16(q), bf16(k), v, dev.batch([0, n])))
            for t in range(n):
                want = from_bf16(v)[[b for b in best if b <= t], 0]
                # weights are alike or 0; sums of four, a quotient, and the rounding to bf16. And each weight's rounding to bf16, 2^-8, which its part of the
                # sum of weights does not have: the largest weight is 2^(s c - m), m the rounded s c, which is off by up to 1/2 for m below 2^24, so no power of two
                tol = (2.0 ** -8 + 6 * 2.0 ** -24) * np.abs(want).mean(0)
                tol = tol + 2.0 ** -8 * (np.abs(want.mean(0)) + tol)
                assert np.all(np.abs(got[t] - want.mean(0)) <= tol), (sign, e, t)
        dev.free_all()


@pytest.mark.parametrize("hd", [8, 32, 40, 64, 80, 96, 128])
def test_many_groups(dev, hd):
    """Enough rows that workgroups take groups of their own tiles, and few enough that wavefronts share them: lengths around the borders."""
    rng = np.random.default_rng(hd + 1)
    for nkv, g, lens in ((4, 4, [1100, 300, 65]), (2, 2, [900, 1, 31]), (1, 3, [1705]), (1, 1, [257, 0, 256, 255])):
        n = sum(lens)
        q, k, v = rows(rng, n, nkv * g, hd), rows(rng, n, nkv, hd), rows(rng, n, nkv, hd)
        check(dev.attend_packed(q, k, v, dev.batch(np.cumsum([0] + lens))), q, k, v, lens, pick=60)
        dev.free_all()


def test_not_finite_long(dev):
    """A NaN and infinities among the values of a prompt whose tiles several wavefronts share: they reach the rows from them on and no others."""
    rng = np.random.default_rng(9)
    n, hd = 700, 64
    q, k, v = rows(rng, n, 2, hd), rows(rng, n, 1, hd), rows(rng, n, 1, hd)
    b = dev.batch([0, n])
    none = from_bf16(dev.attend_packed(q, k, v, b))
    vv = v.copy()
    vv[300, 0, 3], vv[613, 0, 5] = 0x7F80, 0x7FC0
    got = from_bf16(dev.attend_packed(q, k, vv, b))
    assert not np.isfinite(got[300:, :, 3]).any() and not np.isfinite(got[613:, :, 5]).any()
    got[300:, :, 3], got[613:, :, 5] = none[300:, :, 3], none[613:, :, 5]
    for lo, hi in ((256, 300), (576, 613)):                           # computed another way in those tiles
        want, tol = attended(from_bf16(q[lo:hi]), from_bf16(k), from_bf16(v), range(lo + 1, hi + 1), 2.0 ** -8, 0.0)
        same = np.arange(hd) != 3 if lo == 576 else np.ones(hd, bool)
        assert np.all((np.abs(got[lo:hi] - want) <= tol + 2.0 ** -8 * (np.abs(want) + tol))[..., same])
        got[lo:hi] = none[lo:hi]
    assert np.array_equal(got, none)


@pytest.mark.parametrize("nkv, g, hd", [(2, 3, 48), (3, 2, 128), (8, 4, 64)])
def test_strides_long(dev, nkv, g, hd):
    """As above for a prompt of several tiles: fused rows, out in q's place, what no prompt names left as it was; and the same result apart."""
    rng = np.random.default_rng(10)
    n, nq = 420, nkv * g
    width, qw, kw = (nq + 2 * nkv) * hd + 24, nq * hd, nkv * hd
    x = bf16(rng.standard_normal((n, width)))
    b = dev.batch([10, 10, 390, 399], n=n)
    p = dev.put(x)
    assert dev.lib.l3m_k_attend_packed(p, width, p, width, p + 2 * qw, p + 2 * (qw + kw), width, C.byref(b), nq, nkv, hd, None) == 0
    got = dev.get(p, x.shape, np.uint16)
    q, k, v = x[:, :qw].reshape(n, nq, hd), x[:, qw:qw + kw].reshape(n, nkv, hd), x[:, qw + kw:qw + 2 * kw].reshape(n, nkv, hd)
    want = dev.attend_packed(q, k, v, b).reshape(n, qw)
    assert np.array_equal(got[:, qw:], x[:, qw:]) and np.array_equal(got[:10], x[:10]) and np.array_equal(got[399:], x[399:])
    assert np.array_equal(got[10:399, :qw], want[10:399])
    check(want[10:399].reshape(389, nq, hd), q[10:399], k[10:399], v[10:399], [380, 9])
