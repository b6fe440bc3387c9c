"""How near the attention over the 4-bit K/V cache has to come at inputs of ordinary size, and that the limit tells a lost part from a whole one: the formula
with its weights or queries rounded further passes it for no head size."""
import numpy as np
import pytest

# Relative error, 2-norm of a head's outputs. A score of ordinary size (|s| a few units, partial sums of q4_0's codes, 0 .. 15, some three times that) is summed in
# float32 with errors of some 2^-24 of the partial sums at each of up to eight blocks: 2^-24 * 8 * sqrt(8) and less, 1.4e-6, in the worst head, a third of that
# elsewhere; a weight in two f16 parts is off by 2^-22 and the sums by less, 2.4e-7 and random. 2e-6 leaves those room.
LIMIT = 2e-6


def apart(got, want):
    return float(np.linalg.norm((got - want).astype(np.float64)) / np.linalg.norm(want))


def ordinary(hd, pos, n, nq, nkv):
    rng = np.random.default_rng(hd * 7 + pos)
    return rng.standard_normal((n, nq, hd)).astype(np.float32), rng.standard_normal((pos + n, nkv, hd)), rng.standard_normal((pos + n, nkv, hd))


def bits(x, n):
    """x to n significant bits."""
    m, e = np.frexp(x)
    return np.ldexp(np.round(m * 2.0 ** n) * 2.0 ** -n, e)


def formula(q, k, v, weights=None, queries=None):
    s = (bits(q, queries) if queries else q) @ k.T / np.sqrt(q.shape[1])
    p = np.exp(s - s.max(1, keepdims=True))
    return (bits(p, weights) if weights else p) @ v / p.sum(1, keepdims=True)


@pytest.mark.parametrize("hd", [8, 32, 48, 64, 80, 96, 128, 160, 200, 224, 256])
@pytest.mark.parametrize("seen", [40, 1000, 20000])
def test_limit_tells_a_lost_part(hd, seen):
    q, k, v = ordinary(hd, seen - 1, 1, 4, 1)
    q, k, v = q[0].astype(np.float64), k[:, 0], v[:, 0]
    want = formula(q, k, v)
    assert apart(formula(q, k, v, weights=11), want) > 5 * LIMIT
    assert apart(formula(q, k, v, queries=11), want) > 5 * LIMIT
    assert apart(formula(q, k, v, queries=15), want) > LIMIT           # of mxfp4's five parts of a query, three
    assert apart(formula(q.astype(np.float32), k.astype(np.float32), v.astype(np.float32)), want) < LIMIT / 2
