"""Attention over pages, long caches under many rows: what a call takes of the device's memory, slices of any length, sequences by portions."""
import numpy as np
import pytest

from crabml_b200 import paged
from tests import paged_ref as R
from tests.gpu_common import make_device
from tests.test_paged_ops import Case, check_attention, dev, give, take                     # noqa: F401 (dev: the fixture)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_the_workspace_of_a_long_prompt():
    """8192 tokens over 65536: the sums of slices of 4096 keys alone would be 537 MB"""
    P, G, Rh, d, n, end = 128, 2, 4, 128, 8192, 65536
    dev = make_device()  # noqa: F811
    c = Case(dev, P, G, d, d, True, [end - n], [n], seed=1)
    for m in ("k_scale", "v_scale"):
        c.ref.a[m] /= np.float32(60)
    c.cache = paged.PagedCache(**{m: give(dev, a) for m, a in c.ref.a.items()})
    q = c.rng.normal(size=(n, G * Rh, d)).astype(np.float32)
    qt, plan = give(dev, q.reshape(n, -1)), c.plan()
    dev.synchronize()
    before = torch.cuda.mem_get_info()[0]
    y = paged.attention(plan, c.cache, qt, G * Rh, d ** -0.5)
    got = take(dev, y).reshape(n, G * Rh, d)
    used = before - torch.cuda.mem_get_info()[0] - got.nbytes
    assert used <= 530 << 20, used
    k, v = (c.ref.rows(m, c.table[0], end, c.slot(0)) for m in ("k", "v"))
    for t in (0, 4097, n - 1):
        at = end - n + t
        want, mass, reach = R.attention(q[t:t + 1], k[:, :at + 1], v[:, :at + 1], at, float(np.float32(d ** -0.5)))
        assert (np.abs(got[t:t + 1] - want) <= R.attention_bound(mass, reach, d, at + 1)).all()
    del y, qt, plan, c
    dev.close()


@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
@pytest.mark.parametrize("kw", [{}, dict(window=4500, sink=True), dict(softcap=20.0)], ids=["all", "window", "cap"])
def test_slices_of_thousands_of_keys(kw, i8):
    """on one SM a row's keys are not dealt out: 70 steps, and what stands beside them, one after the other; a number that is not finite in the fiftieth"""
    dev = make_device()  # noqa: F811
    dev.set_sm_limit(1)
    P, d, Rh, pos0, n = 32, 64, 4, 8930, 30
    c, q, clean = check_attention(dev, P, 1, Rh, d, d, i8, [pos0, 20], [n, 40], seed=3, **kw)
    sink = {}
    if "sink" in kw:
        r = np.random.default_rng(9)
        sink = dict(sink=give(dev, r.normal(size=Rh).astype(np.float32)))
    rest = {k: v for k, v in kw.items() if k != "sink"}

    def run():
        cache = paged.PagedCache(**{m: give(dev, a) for m, a in c.ref.a.items()})
        return take(dev, paged.attention(c.plan(), cache, give(dev, q.reshape(n + 40, -1)), Rh, d ** -0.5, **rest, **sink)).reshape(n + 40, Rh, d)
    if sink:
        clean = run()
    bad = pos0 + 10 - 4499 if "window" in kw else 6400      # with the window: the first key of the eleventh new token
    block = bad // P
    if i8:
        c.ref.a["v_scale"][c.table[0][block]] = np.nan
        seen = [t for t in range(n) if "window" not in kw or pos0 + t - 4499 < (block + 1) * P]
    else:
        c.ref.a["v"][c.table[0][block], 0, bad % P, 3] = np.inf
        seen = [t for t in range(n) if "window" not in kw or pos0 + t - 4499 <= bad]
    got = run()
    others = sorted(set(range(n + 40)) - set(seen))
    assert len(seen) >= 11 and len(others) >= 40
    np.testing.assert_array_equal(got[others], clean[others])
    if i8:
        assert np.isnan(got[seen]).all()
    else:
        assert not np.isfinite(got[seen][..., 3]).any()
        np.testing.assert_array_equal(np.delete(got[seen], 3, 2), np.delete(clean[seen], 3, 2))
    dev.close()


@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
def test_sequences_by_portions(dev, i8):  # noqa: F811
    """eight sequences over a common prefix of 120000 tokens: the images of one head are more than are kept at a time"""
    P, d, pos0, seqs = 128, 128, 120000, 8
    counts = [33 + i for i in range(seqs)]
    c = Case(dev, P, 1, d, d, i8, [pos0] + [0] * (seqs - 1), [counts[0]] + [0] * (seqs - 1), spare=seqs, seed=6)
    own, spare = c.table[0][-1], sorted(set(range(c.n_pages)) - set(c.table[0]))
    assert pos0 // P == len(c.table[0]) - 1
    table = [c.table[0][:-1] + [p] for p in [own] + spare[:seqs - 1]]
    plan = paged.PagePlan(dev, P, c.n_pages, table, [pos0] * seqs, counts, c.n_slots, c.slots)
    q = c.rng.normal(size=(sum(counts), 1, d)).astype(np.float32)
    scale = d ** -0.5 / (60 if i8 else 1)
    got, at = take(dev, paged.attention(plan, c.cache, give(dev, q.reshape(-1, d)), 1, scale)), 0
    for i, n in enumerate(counts):
        k, v = (c.ref.rows(m, table[i], pos0 + n, c.slot(i)) for m in ("k", "v"))
        for t in (0, n - 1):
            want, mass, reach = R.attention(q[at + t:at + t + 1], k[:, :pos0 + t + 1], v[:, :pos0 + t + 1], pos0 + t, float(np.float32(scale)))
            assert (np.abs(got[at + t].reshape(1, 1, d) - want) <= R.attention_bound(mass, reach, d, pos0 + t + 1)).all()
        at += n
