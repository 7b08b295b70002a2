"""Attention over pages at the ends of its numbers: scores whose last place is more than one, queries that are not finite."""
import numpy as np
import pytest

from crabml_b200 import paged
from tests import paged_ref as R
from tests.test_paged_ops import Case, dev, give, take                                      # noqa: F401 (dev: the fixture)

pytestmark = pytest.mark.gpu


def attend(c, q, scale, **kw):
    """q [T, H, dk] -> [T, H, dv]"""
    T, H = q.shape[:2]
    y = paged.attention(c.plan(), c.cache, give(c.dev, q.reshape(T, -1)), H, scale, **kw)
    return take(c.dev, y).reshape(T, H, c.dv)


def refill(c):
    c.cache = paged.PagedCache(**{n: give(c.dev, a) for n, a in c.ref.a.items()})


# ---- large scores ---------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
@pytest.mark.parametrize("n", [1, 8, 40, 300])
@pytest.mark.parametrize("size", [2.0 ** 18, 1.3 * 2.0 ** 20, 1.9 * 2.0 ** 24, 1.1 * 2.0 ** 26, 1.03 * 2.0 ** 27, 1.4 * 2.0 ** 27, 1.9 * 2.0 ** 27, 1.3 * 2.0 ** 28, 1e9, 1.7 * 2.0 ** 33])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_large_numbers(dev, size, sign, n, i8):  # noqa: F811
    """Keys that are whole multiples c of one: scores c s with s up to thousands of millions.  Those of the best multiple that a query sees are equal to the last bit (the same
    operations on the same numbers), all others lie size / 5 or more below them, which no rounding bridges: the result is the mean of the best ones' values"""
    P, d, pos0 = 16, 32, 70
    c = Case(dev, P, 1, d, d, i8, [pos0], [n], seed=11)
    r, a, end = c.rng, c.ref.a, pos0 + n
    base = r.integers(1, 13, d) * r.choice([-1, 1], d)
    times = r.integers(1, 6, end)
    k = (times[:, None] * base).astype(np.float64)
    for p in range(end):
        b = p // P
        open_ = i8 and (b + 1) * P > end
        at = (2 * c.slot(0) + b % 2, 0, p % P) if open_ else (c.table[0][b], 0, p % P)
        a["k_open" if open_ else "k"][at] = k[p]
    if i8:
        a["k_scale"][:] = 1
        a["v_scale"][:] = np.float32(1 / 60)
    refill(c)
    q = np.abs(r.normal(size=(n, 1, d))) + 0.1
    q = q * np.sign(base)                                    # every product is positive: s = q . base > 0
    q = (q / (q @ base)[..., None] * (sign * size / 5 / np.log2(np.e))).astype(np.float32)
    got = attend(c, q, 1.0)
    v = c.ref.rows("v", c.table[0], end, c.slot(0))[0]
    for t in range(n):
        see = times[:pos0 + t + 1]
        best = np.flatnonzero(see == (see.max() if sign > 0 else see.min()))
        want, mass = v[best].mean(0), np.abs(v[best]).mean(0)
        tol = R.attention_bound(mass[None, None], np.zeros((1, 1)), d, pos0 + t + 1)[0, 0]
        assert (np.abs(got[t, 0] - want) <= tol).all(), (t, got[t, 0][:4], want[:4])


# ---- queries that are not finite ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
@pytest.mark.parametrize("n", [5, 40, 150])
@pytest.mark.parametrize("window,kw", [(1, {}), (2, {}), (6, {}), (0, {}), (3, dict(softcap=5.0)), (4, dict(sink=True)), (0, dict(softcap=5.0, sink=True))])
def test_queries_that_are_not_finite(dev, window, kw, n, i8):  # noqa: F811
    """their results are NaN, all of them; the other queries' stay as they are"""
    P, d, Rh, pos0 = 16, 48, 1, 23
    c = Case(dev, P, 1, d, d, i8, [pos0], [n], seed=5)
    if i8:
        c.ref.a["k_scale"] /= np.float32(60)
        c.ref.a["v_scale"] /= np.float32(60)
        refill(c)
    q = c.rng.normal(size=(n, Rh, d)).astype(np.float32)
    kw = dict(kw, window=window)
    if kw.pop("sink", False):
        kw["sink"] = give(dev, np.zeros(Rh, np.float32))
    clean = attend(c, q, 0.2, **kw)
    assert np.isfinite(clean).all()
    for what in (np.nan, np.inf, -np.inf):
        for first in (0, 1):
            x, hit = q.copy(), np.arange(first, n, 2)
            x[hit, 0, hit % d] = what
            got = attend(c, x, 0.2, **kw)
            assert np.isnan(got[hit]).all(), (what, np.argwhere(~np.isnan(got[hit]))[:3])
            rest = np.arange(1 - first, n, 2)
            np.testing.assert_array_equal(got[rest], clean[rest])
