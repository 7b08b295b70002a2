"""The plan of a step over several sequences (crabml_b200/csrc/paged_plan.hpp) on the CPU: what is refused, and that the segments cover every new token once, keep what
has to be kept and stand in an order in which no open row is overwritten before it is read.  CPU only."""
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FULL, KEPT = 1, 2


@pytest.fixture(scope="module")
def build(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("plan") / "plan")
    subprocess.run(["g++", "-std=c++17", "-O1", os.path.join(ROOT, "tests", "host", "paged_plan_check.cpp"), "-o", exe], check=True, capture_output=True, timeout=300)

    def run(page, n_pages, table, pos0, counts, n_slots=0, slots=None):
        cols = max([len(r) for r in table], default=0)
        text = [len(counts), page, cols, n_pages, n_slots, int(slots is not None), *pos0, *counts]
        for r in table:
            text += list(r) + [-1] * (cols - len(r))
        text += slots or []
        out = subprocess.run([exe], input=" ".join(map(str, text)), check=True, capture_output=True, text=True, timeout=60).stdout.strip().split("\n")
        if out[0].startswith("wrong"):
            return out[0], []
        keys = ("seq", "block", "page", "token0", "row0", "rows", "half", "flags", "next", "pos0")
        return [int(x) for x in out[0].split()[1:]], [dict(zip(keys, map(int, r.split()))) for r in out[1:]]
    return run


REFUSED = [
    ("page size", dict(page=48, n_pages=4, table=[[0]], pos0=[0], counts=[1]), "pages of 48"),
    ("negative count", dict(page=16, n_pages=4, table=[[0]], pos0=[0], counts=[-1]), "new ones"),
    ("negative position", dict(page=16, n_pages=4, table=[[0]], pos0=[-1], counts=[1]), "new ones"),
    ("position beyond 31 bits", dict(page=16, n_pages=4, table=[[0]], pos0=[1 << 31], counts=[1]), "new ones"),
    ("a page too few", dict(page=16, n_pages=4, table=[[0]], pos0=[16], counts=[1]), "needs more than 1 pages"),
    ("no such page", dict(page=16, n_pages=4, table=[[4]], pos0=[0], counts=[1]), "page 4 of sequence 0"),
    ("no page given", dict(page=16, n_pages=4, table=[[0], [1, 2]], pos0=[16, 0], counts=[1, 1]), "page -1 of sequence 0"),
    ("a read page out of range", dict(page=16, n_pages=4, table=[[9, 1]], pos0=[16], counts=[1]), "page 9 of sequence 0"),
    ("one page for two sequences", dict(page=16, n_pages=4, table=[[0], [0]], pos0=[0, 3], counts=[1, 1]), "page 0 takes tokens"),
    ("one page twice in a row", dict(page=16, n_pages=4, table=[[0, 0]], pos0=[0], counts=[20]), "page 0 takes tokens"),
    ("an older page again", dict(page=16, n_pages=4, table=[[0, 0]], pos0=[16], counts=[2]), "page 0 takes new tokens"),
    ("a page another one reads", dict(page=16, n_pages=4, table=[[0, 1], [1, 2]], pos0=[16, 16], counts=[1, 1]), "page 1 takes new tokens"),
    ("a page that a resting one reads", dict(page=16, n_pages=4, table=[[0, 1], [1, 2]], pos0=[16, 17], counts=[1, 0]), "page 1 takes new tokens"),
    ("no such slot", dict(page=16, n_pages=4, table=[[0]], pos0=[0], counts=[1], n_slots=1, slots=[1]), "slot 1 of sequence 0"),
    ("one slot for two", dict(page=16, n_pages=4, table=[[0], [1]], pos0=[0, 0], counts=[1, 1], n_slots=3, slots=[2, 2]), "two sequences with slot 2"),
    ("more sequences than slots", dict(page=16, n_pages=4, table=[[0], [1]], pos0=[0, 0], counts=[1, 1], n_slots=1), "slot 1 of sequence 1"),
    ("too many tokens", dict(page=128, n_pages=1 << 18, table=[list(range(1 << 17))], pos0=[0], counts=[1 << 24]), "16 million"),
]


@pytest.mark.parametrize("what,plan,text", REFUSED, ids=[r[0] for r in REFUSED])
def test_refused(build, what, plan, text):
    head, _ = build(**plan)
    assert isinstance(head, str) and text in head


def test_allowed(build):
    # a shared prefix that nothing is appended to, a sequence at rest, pages that are not needed, no sequence at all
    assert build(16, 9, [[3, 4], [3, 5]], [16, 20], [1, 2])[0] == [2, 3, 2]
    assert build(16, 9, [[3], [4]], [5, 6], [0, 1])[0] == [1, 1, 1]
    assert build(16, 9, [[3, -1, 99]], [0], [16])[0] == [1, 16, 1]
    assert build(16, 0, [], [], [])[0] == [0, 0, 0]
    assert build(16, 0, [[]], [0], [0], n_slots=1)[0] == [0, 0, 0]


@pytest.mark.parametrize("seed", range(40))
def test_segments(build, seed):
    r = random.Random(seed)
    P, n = r.choice([16, 32, 64, 128]), r.randint(1, 9)
    pos0 = [r.choice([0, r.randint(0, 5 * P), P * r.randint(0, 4), P * r.randint(1, 4) - 1]) for _ in range(n)]
    counts = [r.choice([0, 1, 1, r.randint(1, 6 * P), P, 2 * P]) for _ in range(n)]
    need = [(p + c + P - 1) // P for p, c in zip(pos0, counts)]
    pages = r.sample(range(sum(need) + 5), sum(need))
    table, at = [], 0
    for k in need:
        table.append(pages[at:at + k])
        at += k
    slots = r.sample(range(n + 3), n)
    (items, tokens, n_segments), segs = build(P, sum(need) + 5, table, pos0, counts, n + 3, slots)
    assert tokens == sum(counts) and n_segments == len(segs)
    first, seen = [sum(counts[:i]) for i in range(n)], [0] * tokens
    for g in segs:
        i = g["seq"]
        assert g["page"] == table[i][g["block"]] and g["half"] == 2 * slots[i] + g["block"] % 2
        assert 0 <= g["row0"] and g["rows"] > 0 and g["row0"] + g["rows"] <= P
        assert g["pos0"] == g["block"] * P + g["row0"] == pos0[i] + g["token0"] - first[i]
        end = pos0[i] + counts[i]
        assert bool(g["flags"] & FULL) == ((g["block"] + 1) * P <= end)
        assert bool(g["flags"] & KEPT) == (g["block"] >= end // P - 1)
        for t in range(g["token0"], g["token0"] + g["rows"]):
            seen[t] += 1
    assert seen == [1] * tokens
    # chains: every segment is reached once, and one that writes open rows that another one of its sequence reads stands behind it in the same chain
    reached = []
    for head in range(items):
        chain, at = [], head
        while at >= 0:
            chain.append(segs[at])
            at = segs[at]["next"]
        reached += [id(g) for g in chain]
        for later, g in enumerate(chain):
            assert g["seq"] == chain[0]["seq"] and (later == 0 or g["block"] > chain[later - 1]["block"])
    assert sorted(reached) == sorted(id(g) for g in segs)
    where = {}
    for head in range(items):
        at, place = head, 0
        while at >= 0:
            where[at] = (head, place)
            at, place = segs[at]["next"], place + 1
    for a, g in enumerate(segs):
        for b, h in enumerate(segs):
            reads = h["row0"] > 0 and h["flags"] & FULL
            if a != b and g["flags"] & KEPT and reads and g["half"] == h["half"]:
                assert where[a][0] == where[b][0] and where[a][1] > where[b][1]


def test_numbers_that_are_not_whole_or_too_large():
    """a plan takes them as they are or not at all"""
    import numpy as np

    from crabml_b200 import TensorError, paged
    good = dict(table=[[0, 1]], pos0=[3], counts=[1], slots=[0])
    for bad in (dict(counts=[1.5]), dict(counts=np.array([(1 << 32) + 1])), dict(pos0=[0.5]), dict(slots=np.array([1 << 32])), dict(table=[[0, 1.5]]), dict(table=[[1 << 40]]),
                dict(table=np.array([[1 << 32]])), dict(table=np.array([[0.0]])), dict(pos0=np.array([1 << 63], np.uint64)), dict(slots=[0, 1]), dict(pos0=[0, 0])):
        with pytest.raises(TensorError):
            paged.PagePlan(None, 16, 4, n_slots=1, **{**good, **bad})


@pytest.mark.parametrize("seed", range(12))
def test_where_a_sequence_may_go_back(build, seed):
    """what the header allows, played on the segments: every open row that a block is completed from is the sequence's own, portions that end with a block among them"""
    r = random.Random(seed)
    P, borders = r.choice([16, 32]), 0
    have, half = [], [[None] * P, [None] * P]                # the sequence's tokens as (position, call); what its two open blocks hold
    start = far = 0                                          # where it last went back to a block's start; the furthest since then
    for call in range(60):
        lowest = max(start, P * (far // P - 1))
        at = r.choice([len(have), len(have), min(lowest, len(have)), r.randint(min(lowest, len(have)), len(have)), P * r.randint(0, len(have) // P)])
        n = r.choice([1, 1, r.randint(1, 3 * P), P * ((at + P - 1) // P + r.randint(0, 3)) - at])
        n = max(n, 1)
        if at < lowest:                                      # to the start of a block further back
            start, far = at, at
        have = have[:at] + [(p, call) for p in range(at, at + n)]
        far = max(far, at + n)
        borders += (at + n) % P == 0
        pages = (at + n + P - 1) // P
        (items, _, _), segs = build(P, pages, [list(range(pages))], [at], [n], 1)
        for first in range(items):
            i = first
            while i >= 0:
                g = segs[i]
                own = have[g["block"] * P:(g["block"] + 1) * P]
                rows = half[g["half"]]
                if g["flags"] & FULL:
                    assert rows[:g["row0"]] == own[:g["row0"]], (call, at, n, g)
                if g["flags"] & KEPT:
                    rows[g["row0"]:g["row0"] + g["rows"]] = own[g["row0"]:g["row0"] + g["rows"]]
                i = g["next"]
        if (at + n) % P:                                     # attention reads the open block
            assert half[(at + n) // P % 2][:(at + n) % P] == have[(at + n) // P * P:], (call, at, n)
    assert borders > 5


def test_arguments_that_are_not_whole_or_too_large():
    """a window of 2^32 + 5 would arrive as one of 5: refused before the call, like all that its argument cannot hold"""
    from types import SimpleNamespace

    from crabml_b200 import TensorError, capi, paged
    called = []
    lib = SimpleNamespace(cc_paged_append=lambda *a: called.append(a), cc_paged_attention=lambda *a: called.append(a), cc_page_plan_create=lambda *a: called.append(a))
    dev = SimpleNamespace(lib=lib, handle=None, check=lambda rc: None)
    plan = SimpleNamespace(device=dev, handle=None, tokens=1)
    t = SimpleNamespace(_view=capi.cc_view, shape=lambda: [1, 1, 16, 16])
    cache = paged.PagedCache(t, t)
    wrong = (1 << 32, (1 << 32) + 5, 1 << 31, -(1 << 31) - 1, 1.5, "1", None)
    for x in wrong:
        for kw in (dict(window=x), dict(n_heads=x)):
            with pytest.raises(TensorError):
                paged.attention(plan, cache, t, **{**dict(n_heads=1, scale=1.0), **kw})
        for kw in ("q_col0", "k_col0", "v_col0", "n_heads", "pairing", "offset"):
            with pytest.raises(TensorError):
                paged.append(plan, cache, **{**dict(q_src=t, q_col0=0, k_src=t, k_col0=0, v_src=t, v_col0=0, n_heads=1), kw: x})
        with pytest.raises(TensorError):
            paged.PagePlan(dev, x, 4, [[0]], [0], [1])
    for x in (1 << 63, 1.5):
        for kw in (dict(n_pages=x), dict(n_slots=x)):
            with pytest.raises(TensorError):
                paged.PagePlan(dev, **{**dict(page_size=16, n_pages=4, table=[[0]], pos0=[0], counts=[1]), **kw})
    assert not called
    paged.attention(plan, cache, t, 1, 1.0, window=5.0)
    assert called.pop()[6] == 5


def test_a_pool_of_any_size(build, monkeypatch):
    """a plan takes memory for its step, not for the pages and slots that there are"""
    import resource
    plain, most = subprocess.run, 256 << 20
    monkeypatch.setattr(subprocess, "run", lambda *a, **kw: plain(*a, preexec_fn=lambda: resource.setrlimit(resource.RLIMIT_AS, (most, most)), **kw))
    head, segs = build(16, (1 << 31) - 1, [[(1 << 31) - 2, 7], [(1 << 30) + 3]], [17, 0], [1, 16], (1 << 30) - 1, [(1 << 30) - 2, 5])
    assert head == [2, 17, 2] and sorted(g["page"] for g in segs) == [7, (1 << 30) + 3]
    for table, text in (([[1 << 30, 7], [7]], "page 7 takes"), ([[9, 1 << 30], [1 << 30]], f"page {1 << 30} takes")):
        assert text in build(16, (1 << 31) - 1, table, [17, 0], [1, 16], (1 << 30) - 1, [(1 << 30) - 2, 5])[0]
    assert "two sequences with slot 5" in build(16, (1 << 31) - 1, [[8], [9]], [0, 0], [1, 1], (1 << 30) - 1, [5, 5])[0]


@pytest.mark.parametrize("seed", range(30))
def test_pages_that_two_take(build, seed):
    """a page that takes new tokens stands nowhere else: against a count of every page's places"""
    r = random.Random(1000 + seed)
    P, n = 16, r.randint(1, 6)
    pos0, counts = [r.randint(0, 60) for _ in range(n)], [r.choice([0, 1, r.randint(1, 50)]) for _ in range(n)]
    table = [[r.randrange(r.choice([60, 4000])) * r.choice([1, 1024]) % 4096 for _ in range((p + c + P - 1) // P)] for p, c in zip(pos0, counts)]
    places, new = {}, []
    for i, row in enumerate(table):
        for b, page in enumerate(row):
            places[page] = places.get(page, 0) + 1
            if counts[i] and b >= pos0[i] // P:
                new.append(page)
    head, _ = build(P, 4096, table, pos0, counts)
    assert isinstance(head, str) == any(places[p] > 1 for p in new), (table, pos0, counts)
