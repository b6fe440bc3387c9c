"""Rotary positions (l3m_k_rotary) against the formula in extended precision."""
import numpy as np
import pytest

import l3m_amd as A
from serve import bf16, from_bf16, typed, values

pytestmark = pytest.mark.gpu
LD = np.longdouble
TWO_PI = LD("6.283185307179586476925286766559")


@pytest.fixture(autouse=True)
def clean(dev):
    yield
    dev.free_all()


def frequencies(rd, theta, scaling, factor, low, high, trained):
    i = np.arange(rd // 2).astype(LD)
    base = LD(theta) * LD(factor) ** (LD(rd) / (rd - 2)) if scaling == "base" else LD(theta)
    f = base ** (-2 * i / rd) if rd else i
    if scaling == "linear":
        f = f / factor
    if scaling == "index":
        at = [rd * np.log(trained / (LD(t) * TWO_PI)) / (2 * np.log(base)) for t in (high, low)]
        a, b = max(np.floor(at[0]), 0), min(np.ceil(at[1]), rd - 1)
        slow = np.clip((i - a) / max(b - a, LD("0.001")), 0, 1)
        f = f * (1 - slow) + f / factor * slow
    if scaling == "turns":
        keep = np.clip((trained * f / TWO_PI - low) / (LD(high) - low), 0, 1)
        f = f * keep + f / factor * (1 - keep)
    return f, 0.1 * np.log(factor) + 1 if scaling == "index" else 1.0


def turned(x, pos, f, mag, rd, halves):
    """x [n][heads][hd] turned, and the sum of its terms' magnitudes."""
    a = np.asarray(pos).astype(LD)[:, None] * f
    c, s = ((mag * fn(a - np.round(a / TWO_PI) * TWO_PI)).astype(np.float64)[:, None] for fn in (np.cos, np.sin))
    x = x.astype(np.float64)
    u, w = (x[..., :rd // 2], x[..., rd // 2:rd]) if halves else (x[..., 0:rd:2], x[..., 1:rd:2])
    y, size = [u * c - w * s, u * s + w * c], [abs(u * c) + abs(w * s), abs(u * s) + abs(w * c)]
    join = (lambda p: np.concatenate(p, -1)) if halves else (lambda p: np.stack(p, -1).reshape(*p[0].shape[:-1], rd))
    amp = join([abs(u) + abs(w)] * 2)
    return np.concatenate([join(y), x[..., rd:]], -1), np.concatenate([3 * 2.0 ** -24 * join(size) * (1 + 1e-6) + 2e-9 * mag * amp, 0 * x[..., rd:]], -1)


def check(got, want, tol, out):
    tol = tol + (2.0 ** -8 * abs(want) * (1 + 1e-6) + 1e-40 if out == A.BF16 else 0)
    assert np.all(np.abs(values(got) - want) <= tol), np.max(np.abs(values(got) - want) - tol)


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("hd, rd", [(64, 64), (128, 64), (80, 80), (96, 32), (256, 256), (6, 4), (66, 66), (40, 24), (64, 0), (1, 0), (8, 8), (16, 16)])
def test_shapes(dev, hd, rd, halves):
    """Types, head counts, strides with a gap, rows from one to many, one position each."""
    for n, nq, nkv, gap, dtype, out in ((1, 3, 1, 0, "f32", A.F32), (7, 4, 2, 8, "bf16", A.BF16), (33, 5, 0, 3, "f32", A.BF16), (1300, 0, 2, 0, "bf16", A.F32)):
        rng = np.random.default_rng(hd + n)
        rows, vals = typed(rng.standard_normal((n, (nq + nkv) * hd + gap)) * 3, dtype)
        pos = rng.integers(0, 5000, n).astype(np.int32)
        q, k = dev.rotary(dev.rotary_plan(hd, rd, halves), rows, nq, nkv, pos, out=out)
        f, mag = frequencies(rd, 10000.0, "plain", 1.0, 1, 4, 1)
        want, tol = turned(vals[:, :(nq + nkv) * hd].reshape(n, nq + nkv, hd), pos, f, mag, rd, halves)
        check(q, want[:, :nq], tol[:, :nq], out)
        check(k, want[:, nq:], tol[:, nq:], out)
        dev.free_all()


@pytest.mark.parametrize("scaling", list(A.ROTARY_SCALINGS))
@pytest.mark.parametrize("theta, factor, trained", [(10000.0, 4.0, 2048), (500000.0, 8.0, 8192), (10000.0, 1.0, 4096), (100.0, 2.5, 64)])
def test_scalings(dev, scaling, theta, factor, trained):
    low, high = 1.0, 32.0 if scaling == "index" else 4.0
    for rd in (128, 32):
        plan = dev.rotary_plan(128, rd, True, theta, scaling, factor, low, high, trained)
        f, mag = frequencies(rd, theta, scaling, factor, low, high, trained)
        turns = np.array([int(t) for t in plan.turn[:rd // 2]], np.uint64).astype(LD) / LD(2) ** 64
        # a turn more or less is none; the plan's rounding is 2^-65, the powers' a few 2^-63
        off = np.abs(turns - f / TWO_PI)
        assert np.all(np.minimum(off, np.abs(off - 1)) < 2.0 ** -58) and abs(plan.mag - mag) <= 2.0 ** -23
        rng = np.random.default_rng(rd)
        x, pos = rng.standard_normal((9, 3 * 128)).astype(np.float32), np.int32([0, 1, 2, 63, 64, 4097, 131071, 1 << 20, 5])
        q, k = dev.rotary(plan, x, 2, 1, pos)
        want, tol = turned(x.reshape(9, 3, 128), pos, f, mag, rd, True)
        check(np.concatenate([q, k], 1), want, tol, A.F32)


def test_far_and_negative_positions(dev):
    """Any int32 is a position; one turned and then turned by its negative is where it was."""
    pos = np.int32([0, -1, 2 ** 31 - 1, -2 ** 31, -2 ** 31 + 1, 1 << 30, 12345678, -12345678])
    rng = np.random.default_rng(1)
    x = rng.standard_normal((8, 2 * 64)).astype(np.float32)
    plan, (f, _) = dev.rotary_plan(64, halves=True), frequencies(64, 10000.0, "plain", 1.0, 1, 4, 1)
    q, k = dev.rotary(plan, x, 1, 1, pos)
    # the plan's 2^-65 of a turn times 2^31 is below 2e-9
    want, tol = turned(x.reshape(8, 2, 64), pos, f, 1.0, 64, True)
    check(np.concatenate([q, k], 1), want, tol, A.F32)
    back = np.int32(-np.int64(pos[[1, 2, 4, 5, 6, 7]]))
    q2, _ = dev.rotary(plan, q.reshape(8, 64)[[1, 2, 4, 5, 6, 7]], 1, 0, back)
    assert np.abs(q2[:, 0] - x[[1, 2, 4, 5, 6, 7], :64]).max() < 2e-6


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd, rd, width", [(64, 32, 6 * 64 + 8), (62, 30, 6 * 62 + 1)])
def test_in_place_and_neighbours(dev, dtype, hd, rd, width):
    """The rows' own heads turned where they are: what lies behind them, and the part that does not turn, keep their bits. q and k as columns of one output."""
    rng = np.random.default_rng(3)
    n, nq, nkv, size = 20, 3, 2, 4 if dtype == "f32" else 2
    rows, vals = typed(rng.standard_normal((n, width)), dtype)
    code = A.F32 if dtype == "f32" else A.BF16
    plan = dev.rotary_plan(hd, rd)
    p = dev.put(rows)
    assert dev.lib.l3m_k_rotary(plan, p, width, p + size * nq * hd, width, code, p, width, code, n, nq, nkv, None, 40, None) == 0
    got = dev.get(p, rows.shape, rows.dtype)
    q, k = dev.rotary(plan, rows, nq, nkv, np.arange(40, 40 + n, dtype=np.int32), out=code)
    both = np.concatenate([q, k], 1)
    assert np.array_equal(got[:, :(nq + nkv) * hd].reshape(both.shape), both) and np.array_equal(got[:, (nq + nkv) * hd:], rows[:, (nq + nkv) * hd:])
    assert np.array_equal(both[..., rd:], rows[:, :(nq + nkv) * hd].reshape(both.shape)[..., rd:])
    o = dev.put(np.full((n, width), 7, rows.dtype))
    assert dev.lib.l3m_k_rotary(plan, o + size * nkv * hd, width, o, width, code, dev.put(rows), width, code, n, nq, nkv, None, 40, None) == 0
    got = dev.get(o, rows.shape, rows.dtype)
    assert np.array_equal(got[:, :nkv * hd].reshape(k.shape), k) and np.array_equal(got[:, nkv * hd:(nq + nkv) * hd].reshape(q.shape), q) and np.all(got[:, (nq + nkv) * hd:] == 7)


def test_not_finite(dev):
    """NaN and infinities stay in their pairs; a row of the largest values."""
    x = np.ones((1, 64), np.float32)
    x[0, 4], x[0, 9], x[0, 20] = np.nan, np.inf, 3e38
    q, _ = dev.rotary(dev.rotary_plan(64), x, 1, 0, pos0=3)
    good = [i for i in range(64) if i // 2 not in (2, 4, 10)]
    assert np.isnan(q[0, 0, 4:6]).all() and not np.isfinite(q[0, 0, 8:10]).any() and np.isfinite(q[0, 0, good]).all() and np.abs(q[0, 0, good]).max() < 1.5
    q, _ = dev.rotary(dev.rotary_plan(64), bf16(x), 1, 0, pos0=3, out=A.BF16)
    assert np.isnan(from_bf16(q[0, 0, 4:6])).all() and np.isfinite(from_bf16(q[0, 0, good])).all()
