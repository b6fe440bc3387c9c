"""Attention over packed prompts (l3m_k_attend_packed) where it can go wrong: sums of rounded weights, infinities among keys, values behind a token."""
import ctypes as C
import time

import numpy as np
import pytest

import l3m_amd as A
from serve import attended, bf16, from_bf16

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean(dev):
    yield
    dev.free_all()


def rows(rng, n, h, hd, size=1.0):
    return bf16(rng.standard_normal((n, h, hd)) * size)


def equal_parts(rng, n, hd, sign, e):
    """Queries and keys of one dimension, so that the positions `best` share all of a row's weight in equal parts; scores of some 2^e."""
    k = np.zeros((n, 1, hd), np.float32)
    k[:, 0, 5] = 2.0 ** -rng.integers(1, 7, n)
    best = [b for b in (0, 7, 133, 280) if b < n]
    k[best, 0, 5] = 1.0 if sign > 0 else 2.0 ** -7
    q = np.zeros((n, 3, hd), np.float32)
    q[..., 5] = sign * 2.0 ** e * (1 + np.arange(3) / 4)
    return bf16(q), bf16(k), best


@pytest.mark.parametrize("hd, n", [(64, 300), (64, 60), (160, 300)])
@pytest.mark.parametrize("sign", [1, -1])
def test_equal_weights(dev, sign, hd, n):
    """Positions that share all weight in equal parts: a weight's rounding to bf16 stands in the sum that the result is divided by as well, so it cancels, and what is
    left is float32's steps (four terms, the sum, a quotient) and the result's rounding, 2^-8."""
    rng = np.random.default_rng(hd + n)
    v = rows(rng, n, 1, hd)
    for e in (17, 20, 40, 70, 113):
        q, k, best = equal_parts(rng, n, hd, sign, e)
        got = from_bf16(dev.attend_packed(q, k, v, dev.batch([0, n])))
        for t in range(n):
            want = from_bf16(v)[[b for b in best if b <= t], 0]
            tol = 6 * 2.0 ** -24 * np.abs(want).mean(0)
            tol = tol + 2.0 ** -8 * (np.abs(want.mean(0)) + tol)
            assert np.all(np.abs(got[t] - want.mean(0)) <= tol), (sign, e, t)


@pytest.mark.parametrize("hd, n", [(64, 300), (64, 60), (160, 300)])
@pytest.mark.parametrize("sign", [1, -1])
def test_large_scores_before_values_not_finite(dev, sign, hd, n):
    """The same with a NaN and an infinity among the values: rows before them in their tile, computed by themselves, are what they are without."""
    rng = np.random.default_rng(hd + n + 1)
    v = rows(rng, n, 1, hd)
    vv, bad = v.copy(), [(50, 3, 0x7FC0), (n - 2, 9, 0xFF80)]
    for t, d, u in bad:
        vv[t, 0, d] = u
    for e in (17, 20, 40, 70, 113):
        q, k, best = equal_parts(rng, n, hd, sign, e)
        got = from_bf16(dev.attend_packed(q, k, vv, dev.batch([0, n])))
        for t in range(n):
            want = from_bf16(v)[[b for b in best if b <= t], 0]
            tol = 6 * 2.0 ** -24 * np.abs(want).mean(0)
            tol = tol + 2.0 ** -8 * (np.abs(want.mean(0)) + tol)
            keep = np.ones(hd, bool)
            keep[[d for at, d, _ in bad if at <= t]] = False
            assert np.all((np.abs(got[t] - want.mean(0)) <= tol)[:, keep]) and not np.isfinite(got[t][:, ~keep]).any(), (sign, e, t)


def without(q, k, v, gone):
    """The attention where the keys of positions `gone` score -inf, so that they have no weight, and its bound. Rows that see no other are NaN."""
    n = len(q)
    keep = np.ones(n, bool)
    keep[gone] = False
    want, tol = attended(from_bf16(q), from_bf16(k)[keep], from_bf16(v)[keep], np.cumsum(keep), 2.0 ** -8, 2.0 ** -126)
    want[np.cumsum(keep) == 0] = np.nan
    return want, tol + 2.0 ** -8 * (np.abs(want) + tol)


@pytest.mark.parametrize("hd, n", [(64, 300), (128, 60), (160, 200)])
def test_first_score_of_minus_infinity(dev, hd, n):
    """A first position whose score is -inf has no weight, in rows that are computed by themselves too."""
    rng = np.random.default_rng(hd)
    q, k, v = rows(rng, n, 2, hd), rows(rng, n, 1, hd), rows(rng, n, 1, hd)
    q[..., 2] &= 0x7FFF
    k[0, 0, 2] = 0xFF80
    want, tol = without(q, k, v, [0])
    for at in (None, 40):
        if at:
            v[at, 0, 7] = 0x7FC0
        got = from_bf16(dev.attend_packed(q, k, v, dev.batch([0, n])))
        assert np.isnan(got[0]).all()
        end = at or n
        assert np.all(np.abs(got[1:end] - want[1:end]) <= tol[1:end])


@pytest.mark.parametrize("hd", [8, 16, 24, 40, 48, 72, 80, 104, 120, 128, 136, 176, 200, 256])
@pytest.mark.parametrize("lens", [[300], [60, 1, 33]])
def test_infinite_keys(dev, hd, lens):
    """Infinities among a key's last eight values and its first ones: -inf as a score has no weight, +inf is NaN in the rows that see it and in no others."""
    rng = np.random.default_rng(hd)
    n = sum(lens)
    q, k, v = rows(rng, n, 4, hd), rows(rng, n, 2, hd), rows(rng, n, 2, hd)
    for d in (hd - 1, hd - 6, 0):
        q[..., d] &= 0x7FFF
    for head in (0, 1):
        k[[5, 30, 59], head, [hd - 1, hd - 6, 0]] = 0xFF80
    k[41, 1, hd - 6] = 0x7F80
    got, at = from_bf16(dev.attend_packed(q, k, v, dev.batch(np.cumsum([0] + lens)))), 0
    for m in lens:
        part = slice(at, at + m)
        gone = [t - at for t in (5, 30, 59) if at <= t < at + m]
        want, tol = without(q[part], np.where(k[part] == 0x7F80, 0, k[part]), v[part], gone)
        nan = np.zeros(want.shape, bool)
        if at <= 41 < at + m:
            nan[41 - at:, 2:] = True
        assert np.isnan(got[part][nan]).all() and np.all(np.abs(got[part] - want)[~nan] <= tol[~nan])
        at += m


@pytest.mark.parametrize("every", [1, 50])
def test_time_of_poisoned_values(dev, every):
    """Values of which a dimension is NaN at every position, or every 50th: rows that are NaN there for their own values' sake are not made anew for those behind
    them, which at this size takes some hundred times as long."""
    rng = np.random.default_rng(11)
    n, nq, nkv, hd = 4096, 16, 4, 128
    q, k, v = rows(rng, n, nq, hd), rows(rng, n, nkv, hd), rows(rng, n, nkv, hd)
    poisoned = v.copy()
    poisoned[::every, :, 77] = 0x7FC0
    b, out = dev.batch([0, n]), dev.alloc(q.nbytes)
    dq, dk = dev.put(q), dev.put(k)
    results, times = [], []
    for x in (v, poisoned):
        dv, least = dev.put(x), []
        for _ in range(5):
            assert dev.lib.l3m_dev_sync() == 0
            start = time.perf_counter()
            assert dev.lib.l3m_k_attend_packed(out, nq * hd, dq, nq * hd, dk, dv, nkv * hd, C.byref(b), nq, nkv, hd, None) == 0 and dev.lib.l3m_dev_sync() == 0
            least.append(time.perf_counter() - start)
        times.append(min(least))
        results.append(from_bf16(dev.get(out, q.shape, np.uint16)))
    assert times[1] < 10 * times[0], times
    clean, got = results
    assert np.isnan(got[..., 77]).all()
    got[..., 77] = clean[..., 77]
    assert np.array_equal(got, clean)


@pytest.mark.parametrize("hd, nkv, g", [(64, 1, 1), (40, 1, 3), (32, 2, 1)])
def test_many_longer_prompts(dev, hd, nkv, g):
    """More prompts than a wavefront has lanes, of one tile or several, whose groups are few enough that wavefronts share them."""
    rng = np.random.default_rng(hd + 70)
    lens = [int(x) for x in rng.choice([0, 1, 63, 64, 65, 130, 190], 75)]
    lens[7] = 700
    n = sum(lens)
    assert n > 64 * len(lens) and (n * g // 128 + len(lens)) * nkv < 256
    q, k, v = rows(rng, n, nkv * g, hd), rows(rng, n, nkv, hd), rows(rng, n, nkv, hd)
    got, at = from_bf16(dev.attend_packed(q, k, v, dev.batch(np.cumsum([0] + lens)))), 0
    for m in lens:
        part = slice(at, at + m)
        want, tol = without(q[part], k[part], v[part], [])
        assert np.all(np.abs(got[part] - want) <= tol)
        at += m


@pytest.mark.parametrize("hd, runs", [(64, 4), (80, 70)])
def test_captured(dev, hd, runs):
    """A call recorded once and replayed: each replay takes the prompts' ends and the rows that it finds, between eager calls, and gives their bits."""
    rng, hip, n, nq, nkv = np.random.default_rng(hd + 2), C.CDLL("libamdhip64.so"), 600, 4, 2
    q, k, v = rows(rng, n, nq, hd), rows(rng, n, nkv, hd), rows(rng, n, nkv, hd)
    dq, dk, dv, out, starts = dev.put(q), dev.put(k), dev.put(v), dev.alloc(q.nbytes), dev.alloc(4 * (runs + 1))
    b, st, graph, ex = A.Batch(None, starts, runs, n), C.c_void_p(), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamCreateWithFlags(C.byref(st), 1) == 0 and hip.hipStreamBeginCapture(st, 1) == 0
    assert dev.lib.l3m_k_attend_packed(out, nq * hd, dq, nq * hd, dk, dv, nkv * hd, C.byref(b), nq, nkv, hd, st) == 0
    assert hip.hipStreamEndCapture(st, C.byref(graph)) == 0 and hip.hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0)) == 0
    for i in range(4):
        ends = np.int32(np.sort(rng.integers(0, n + 1, runs + 1)))
        if i == 2:
            ends[1:] = n                                             # one prompt and empty ones
        q = rows(rng, n, nq, hd)
        for at, x in ((starts, ends), (dq, q), (out, np.full(q.shape, 0x41, np.uint16))):
            assert dev.lib.l3m_dev_upload(at, C.c_void_p(x.ctypes.data), x.nbytes) == 0
        assert dev.lib.l3m_dev_sync() == 0 and hip.hipGraphLaunch(ex, st) == 0 and hip.hipStreamSynchronize(st) == 0
        got, want = dev.get(out, q.shape, np.uint16), dev.attend_packed(q, k, v, dev.batch(ends, n=n))
        named = slice(ends[0], ends[-1])
        assert np.array_equal(got[named], want[named]) and np.all(got[:ends[0]] == 0x41) and np.all(got[ends[-1]:] == 0x41)
    assert hip.hipGraphExecDestroy(ex) == 0 and hip.hipGraphDestroy(graph) == 0 and hip.hipStreamDestroy(st) == 0
