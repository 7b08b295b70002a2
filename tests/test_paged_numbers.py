"""Attention over pages at the ends of its numbers: scores whose last place is more than one, queries that are not finite, value factors that differ by orders of magnitude."""
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


# ---- value factors ----------------------------------------------------------------------------------------------------------------------------
def check(c, q, scale, window=0):
    """Against 64 bits.  Beside what attention_bound counts: a weight is two 16-bit numbers, whose last place is 2^-24 where the row's largest product of a weight and its block's
    factor stands at 2^8 or more (16-bit pages: the largest weight): off by 2^-25 / 2^8 of that for every key, times a code of up to 127 of that block (16 bits: the value)"""
    got, at = attend(c, q, scale, window=window), 0
    for i, n in enumerate(c.counts):
        end = c.pos0[i] + n
        k, v = (c.ref.rows(m, c.table[i], end, c.slot(i)) for m in ("k", "v"))
        want, mass, reach = R.attention(q[at:at + n], k, v, c.pos0[i], float(np.float32(scale)), window)
        tol = R.attention_bound(mass, reach, c.dk, end)
        big = np.abs(v).max(2)                               # [G, keys]: the largest number of a key's block
        for b in range((end + c.P - 1) // c.P):
            if c.i8 and (b + 1) * c.P <= end:
                big[:, b * c.P:(b + 1) * c.P] = 127 * c.ref.a["v_scale"][c.table[i][b]].astype(np.float64)[:, None]
        for t in range(n):
            lo = max(0, c.pos0[i] + t - window + 1) if window else 0
            for h in range(q.shape[1]):
                g = h // (q.shape[1] // c.G)
                kk, bb = k[g, lo:c.pos0[i] + t + 1], big[g, lo:c.pos0[i] + t + 1]
                s = kk @ q[at + t, h].astype(np.float64) * float(np.float32(scale))
                w = np.exp(s - s.max()) if c.i8 else np.ones(len(s))
                tol[t, h] += 2.0 ** -33 * len(s) * (w * bb).max() * (1 + 2 * reach[t, h] * 2.0 ** -18)
        bad = ~(np.abs(got[at:at + n] - want) <= tol)
        assert not bad.any(), (i, np.argwhere(bad)[:3], got[at:at + n][bad][:3], want[bad][:3], tol[bad][:3])
        at += n


@pytest.mark.parametrize("q_scale", [1.0, 8.0])
@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("P", [16, 128])
@pytest.mark.parametrize("pos0,counts", [([60, 3], [40, 130]), ([95, 255], [5, 1])], ids=["many", "few"])
def test_small_values_beside_an_open_block(dev, pos0, counts, P, size, q_scale):  # noqa: F811
    """values far below one, in blocks of codes and in the open one, which share a step of keys"""
    d = 32
    c = Case(dev, P, 1, d, d, True, pos0, counts, seed=31)
    c.ref.a["k_scale"] /= np.float32(60)
    c.ref.a["v_scale"] *= np.float32(size / 60)
    c.ref.a["v_open"] = (c.ref.a["v_open"].astype(np.float32) * np.float32(size)).astype(np.float16)
    refill(c)
    q = (c.rng.normal(size=(sum(counts), 1, d)) * q_scale).astype(np.float32)
    check(c, q, d ** -0.5)


@pytest.mark.parametrize("q_scale", [1e-4, 1.0, 8.0, 30.0])
@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("counts", [[1, 3], [10, 75]], ids=["few", "many"])
def test_value_factors_orders_of_magnitude_apart(dev, counts, window, q_scale):  # noqa: F811
    """factors from 1e-4 to 1e4, blocks of zeros, and open rows of any size: what has a large factor and no weight must not cost the others their bits"""
    P, d, Rh = 16, 32, 4
    c = Case(dev, P, 1, d, d, True, [500, 41], counts, seed=32)
    a = c.ref.a
    a["k_scale"] /= np.float32(60)
    a["v_scale"] *= (10.0 ** c.rng.uniform(-4, 4, a["v_scale"].shape)).astype(np.float32)
    a["v_open"] = (a["v_open"].astype(np.float32) * 10.0 ** c.rng.uniform(-5, 4, a["v_open"].shape[:1])[:, None, None, None]).astype(np.float16)
    zero = c.table[0][3:8:2] + c.table[1][:1]
    a["v_scale"][zero] = 0
    a["v"][zero] = 0
    refill(c)
    q = (c.rng.normal(size=(sum(counts), Rh, d)) * q_scale).astype(np.float32)
    check(c, q, d ** -0.5, window)


@pytest.mark.parametrize("lead", [5.0, 20.0, 50.0, 300.0])
@pytest.mark.parametrize("n", [2, 40])
def test_the_largest_weight_on_zeros(dev, n, lead):  # noqa: F811
    """a block of zeros has the largest score by far: what is left of the others' weights is the whole result"""
    P, d, pos0 = 16, 16, 150
    c = Case(dev, P, 1, d, d, True, [pos0], [n], seed=33)
    a = c.ref.a
    a["k"][:] = 0
    a["k_scale"][:] = 1
    a["k_open"][:] = 0
    a["v_scale"] *= np.float32(1e-2)
    top = c.table[0][2]
    a["v"][top], a["v_scale"][top] = 0, 0
    a["k"][top, 0, 5, 0] = 1
    a["k_scale"][top] = np.float32(lead)
    refill(c)
    q = np.zeros((n, 1, d), np.float32)
    q[..., 0] = 1
    check(c, q, 1.0)


def test_a_factor_that_no_query_of_a_row_sees(dev):  # noqa: F811
    """the bits of a result do not depend on factors of blocks out of its window, nor on blocks behind it"""
    P, d, n, pos0 = 16, 32, 40, 200
    for counts in ([n], [6]):
        c = Case(dev, P, 1, d, d, True, [pos0], counts, seed=34)
        c.ref.a["k_scale"] /= np.float32(60)
        c.ref.a["v_scale"] *= np.float32(1e-4)
        refill(c)
        q = (c.rng.normal(size=(counts[0], 2, d)) * 4).astype(np.float32)
        clean = attend(c, q, d ** -0.5, window=20)
        end = pos0 + counts[0]
        for block in range((pos0 - 19) // P, end // P):
            kept = c.ref.a["v_scale"].copy()
            c.ref.a["v_scale"][c.table[0][block]] = np.float32(400.0)
            refill(c)
            got = attend(c, q, d ** -0.5, window=20)
            c.ref.a["v_scale"] = kept
            unseen = [t for t in range(counts[0]) if pos0 + t < block * P or pos0 + t - 19 >= (block + 1) * P]
            np.testing.assert_array_equal(got[unseen], clean[unseen])
