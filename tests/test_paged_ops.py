"""Pages of a cache that several sequences share (include/crabml_paged.h): the append and the attention against plain references in 64 bits (tests/paged_ref.py), over
16-bit and 8-bit pages, with the lengths, strides, masks and numbers at which they can go wrong."""
import numpy as np
import pytest

from crabml_b200 import CudaTensor, TensorError, CudaError, TensorStrider, capi, paged, seqops
from tests import paged_ref as R
from tests.gpu_common import make_device

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def dev():
    d = make_device()
    yield d
    d.close()


TYPES = {np.dtype(np.float32): capi.F32, np.dtype(np.float16): capi.F16, np.dtype(np.int8): capi.I8}


def give(dev, a):
    a = np.ascontiguousarray(a)
    t = CudaTensor.alloc(list(a.shape), TYPES[a.dtype], dev)
    dev.synchronize()
    if a.size:
        torch.as_tensor(t, device="cuda").copy_(torch.from_numpy(a))
    torch.cuda.synchronize()
    return t


def take(dev, t):
    dev.synchronize()
    return torch.as_tensor(t, device="cuda").cpu().numpy()


class Case:
    """sequences of given lengths over shuffled pages, beside the reference's cache with the same contents"""

    def __init__(self, dev, P, G, dk, dv, i8, pos0, counts, spare=2, seed=0):
        r = np.random.default_rng(seed)
        self.dev, self.P, self.G, self.dk, self.dv, self.i8, self.pos0, self.counts = dev, P, G, dk, dv, i8, list(pos0), list(counts)
        need = [(p + c + P - 1) // P for p, c in zip(pos0, counts)]
        self.n_pages, self.n_slots = sum(need) + spare, (len(counts) + 1 if i8 else 0)
        pages = r.permutation(self.n_pages)
        cut = np.cumsum([0] + need)
        self.table = [pages[cut[i]:cut[i + 1]].tolist() for i in range(len(need))]
        self.slots = r.permutation(len(counts) + 1)[:len(counts)].tolist() if i8 else None
        self.ref = R.Cache(self.n_pages, G, P, dk, dv, i8, self.n_slots, fill=seed)
        self.cache = paged.PagedCache(**{n: give(dev, a) for n, a in self.ref.a.items()})
        self.rng = r

    def plan(self, pos0=None, counts=None):
        return paged.PagePlan(self.dev, self.P, self.n_pages, self.table, self.pos0 if pos0 is None else pos0, self.counts if counts is None else counts, self.n_slots, self.slots)

    def same(self):
        for n, a in self.ref.a.items():
            got = take(self.dev, getattr(self.cache, n))
            np.testing.assert_array_equal(got.view(np.uint8).reshape(-1), a.view(np.uint8).reshape(-1), err_msg=n) if not np.isnan(a.astype(np.float32)).any() else \
                np.testing.assert_array_equal(got, a, err_msg=n)

    def slot(self, i):
        return self.slots[i] if self.slots is not None else 0


def freqs(n, base=10000.0):
    return (base ** (-np.arange(n) / max(n, 1))).astype(np.float32)


# ---- append -------------------------------------------------------------------------------------------------------------------------------
LENGTHS = [
    ([0], [1]), ([15], [1]), ([16], [1]), ([300], [1]), ([127], [2]), ([0], [128]), ([5], [300]), ([130, 7, 64], [1, 0, 1]), ([0, 0, 40], [0, 33, 100]),
    ([63, 64, 65, 1000], [1, 1, 70, 16]),
]


@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
@pytest.mark.parametrize("P", [16, 32, 64, 128])
@pytest.mark.parametrize("pos0,counts", LENGTHS, ids=[str(i) for i in range(len(LENGTHS))])
def test_append(dev, P, i8, pos0, counts):
    G, H, dk, dv = 2, 6, 48, 32
    c = Case(dev, P, G, dk, dv, i8, pos0, counts, seed=P)
    T = sum(counts)
    # keys, values and queries as column blocks of one matrix, with columns between them
    src = c.rng.normal(size=(T, H * dk + 3 + G * dk + 1 + G * dv + 2)).astype(np.float32)
    kc, vc = H * dk + 3, H * dk + 3 + G * dk + 1
    f = freqs(dk // 2)
    t = give(dev, src)
    q = paged.append(c.plan(), c.cache, t, 0, t, kc, t, vc, H, freq=give(dev, f))
    pos = np.concatenate([np.arange(p, p + n) for p, n in zip(pos0, counts)])
    want = R.turn(src[:, :H * dk].reshape(T, H, dk), pos, f, 0, 0, 1.0).reshape(T, -1)
    k = R.turn(src[:, kc:kc + G * dk].reshape(T, G, dk), pos, f, 0, 0, 1.0).astype(np.float32)
    v = src[:, vc:vc + G * dv].reshape(T, G, dv)
    at = 0
    for i, n in enumerate(counts):
        c.ref.append(c.table[i], pos0[i], c.slot(i), {"k": k[at:at + n], "v": v[at:at + n]})
        at += n
    assert q.shape() == [T, H * dk]
    np.testing.assert_allclose(take(dev, q), want, rtol=2.0 ** -23, atol=1e-14)
    c.same()


@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
@pytest.mark.parametrize("pairing,offset,n,mag", [(0, 0, 40, 1.0), (1, 0, 40, 1.0), (0, 16, 8, 1.25), (1, 3, 17, 0.7), (1, 79, 0, 1.0), (0, 1, 1, 1.0)])
def test_append_turns(dev, i8, pairing, offset, n, mag):
    """both pairings, part of the columns, a factor; at positions where 32 bits lose the angle"""
    G, H, d, P = 1, 3, 80, 16
    pos0, counts = [1000003 // P * P - 5, 31], [23, 1]
    c = Case(dev, P, G, d, d, i8, [p % (40 * P) for p in pos0], counts, seed=n)
    far = 1000000 // P * P                                   # the same rows as if they stood further back: the table needs pages for all positions before
    c.table[0] = [c.table[0][0]] * (far // P) + c.table[0]
    c.pos0[0] += far
    T = sum(counts)
    src = c.rng.normal(size=(T, (H + 2 * G) * d)).astype(np.float32)
    f = freqs(n)
    t = give(dev, src)
    ft = give(dev, f) if n else None
    q = paged.append(c.plan(), c.cache, t, 0, t, H * d, t, (H + G) * d, H, freq=ft, pairing=pairing, offset=offset, mag=mag)
    pos = np.concatenate([np.arange(p, p + m) for p, m in zip(c.pos0, counts)])
    x = R.turn(src[:, :(H + G) * d].reshape(T, H + G, d), pos, f if n else None, pairing, offset, mag)
    np.testing.assert_allclose(take(dev, q).reshape(T, H, d), x[:, :H], rtol=2.0 ** -23, atol=1e-14)
    k, at = x[:, H:].astype(np.float32), 0
    for i, m in enumerate(counts):
        c.ref.append(c.table[i], c.pos0[i], c.slot(i), {"k": k[at:at + m], "v": src[at:at + m, (H + G) * d:].reshape(m, G, d)})
        at += m
    c.same()


def test_append_sources(dev):
    """three matrices of their own, rows of a wider one (row stride), no queries"""
    G, H, dk, dv, P = 3, 3, 16, 64, 16
    c = Case(dev, P, G, dk, dv, True, [10, 3], [9, 40], seed=3)
    T = 49
    q, k, v = (c.rng.normal(size=(T, n)).astype(np.float32) for n in (H * dk, G * dk + 5, G * dv))
    wide = give(dev, k)
    kt = wide.with_strider(TensorStrider([T, G * dk + 3], [G * dk + 5, 1]))
    plan = c.plan()
    out = paged.append(plan, c.cache, give(dev, q), 0, kt, 2, give(dev, v), 0, H)
    np.testing.assert_array_equal(take(dev, out), q)         # no frequencies: as they are
    for again in range(2):                                   # and the same without queries
        assert paged.append(plan, c.cache, None, 0, kt, 2, give(dev, v), 0) is None
    for i, (lo, hi) in enumerate(((0, 9), (9, 49))):
        c.ref.append(c.table[i], c.pos0[i], c.slot(i), {"k": k[lo:hi, 2:2 + G * dk].reshape(-1, G, dk), "v": v[lo:hi].reshape(-1, G, dv)})
    for n in ("k", "v"):                                     # (the second sequence's blocks, which the repeated calls began without the rows they replaced)
        got, want = take(dev, getattr(c.cache, n)), c.ref.a[n]
        for b in c.table[0][:1]:
            np.testing.assert_array_equal(got[b], want[b])


@pytest.mark.parametrize("P", [16, 64])
@pytest.mark.parametrize("portions", [[1] * 150, [150], [7] * 21 + [3], [64, 64, 22], [16, 1, 63, 70]], ids=["tokens", "once", "sevens", "blocks", "mixed"])
def test_portions_make_the_same_cache(dev, P, portions):
    """8-bit pages and open blocks do not depend on the portions that a sequence came in"""
    G, d = 2, 32
    c = Case(dev, P, G, d, d, True, [0], [150], seed=11)
    src = np.random.default_rng(12).normal(size=(150, 2 * G * d)).astype(np.float32)
    t, f, at = give(dev, src), give(dev, freqs(d // 2)), 0
    x = R.turn(src[:, :G * d].reshape(150, G, d), np.arange(150), freqs(d // 2), 0, 0, 1.0).astype(np.float32)
    v = src[:, G * d:].reshape(150, G, d)
    for n in portions:
        part = give(dev, src[at:at + n])
        paged.append(c.plan([at], [n]), c.cache, None, 0, part, 0, part, G * d, freq=f)
        at += n
    c.ref.append(c.table[0], 0, c.slot(0), {"k": x, "v": v})
    for n in ("k", "v"):
        for b in range(150 // P):
            np.testing.assert_array_equal(take(dev, getattr(c.cache, n))[c.table[0][b]], c.ref.a[n][c.table[0][b]])
            np.testing.assert_array_equal(take(dev, getattr(c.cache, n + "_scale"))[c.table[0][b]], c.ref.a[n + "_scale"][c.table[0][b]])
        b = 150 // P
        for half in (b, b - 1):                              # the open block and the one before it
            rows = min(P, 150 - half * P)
            got = take(dev, getattr(c.cache, n + "_open"))[2 * c.slot(0) + half % 2, :, :rows]
            np.testing.assert_array_equal(got, R.f16((x if n == "k" else v)[half * P:half * P + rows]).swapaxes(0, 1))


@pytest.mark.parametrize("back", [1, 3, 8, 16, 19, 20])
def test_going_back(dev, back):
    """drafted tokens are rejected: the sequence goes back, across a block that had been completed, and other tokens take their place"""
    G, d, P, n = 1, 16, 16, 37                               # 37 tokens: two blocks and 5 rows; the block before the open one begins at 16
    c = Case(dev, P, G, d, d, True, [0], [n + 20], seed=back)
    r = np.random.default_rng(back)
    a, b = r.normal(size=(n, 2 * d)).astype(np.float32), r.normal(size=(20, 2 * d)).astype(np.float32)
    for at, m in ((0, 30), (30, n - 30)):
        t = give(dev, a[at:at + m])
        paged.append(c.plan([at], [m]), c.cache, None, 0, t, 0, t, d)
    t = give(dev, b)
    paged.append(c.plan([n - back], [20]), c.cache, None, 0, t, 0, t, d)
    every = np.concatenate([a[:n - back], b])
    c.ref.append(c.table[0], 0, c.slot(0), {"k": every[:, None, :d], "v": every[:, None, d:]})
    end = len(every)
    for name in ("k", "v"):
        pages = c.table[0][:end // P]
        np.testing.assert_array_equal(take(dev, getattr(c.cache, name))[pages], c.ref.a[name][pages])
        got = take(dev, getattr(c.cache, name + "_open"))[2 * c.slot(0) + end // P % 2, :, :end % P]
        np.testing.assert_array_equal(got, c.ref.a[name + "_open"][2 * c.slot(0) + end // P % 2, :, :end % P])


@pytest.mark.parametrize("first", [16, 32, 48, 61])
@pytest.mark.parametrize("back", [0, 1, 15, 16])
def test_going_back_from_the_end_of_a_block(dev, first, back):
    """portions that end with a block, and drafts behind them: from there a sequence goes back by up to a block's tokens, or to the start of any"""
    G, d, P = 1, 16, 16
    r = np.random.default_rng(first + back)
    for at in (64 - back, 0, 16, 48):
        c = Case(dev, P, G, d, d, True, [0], [90], seed=back)
        a, b = r.normal(size=(64, 2 * d)).astype(np.float32), r.normal(size=(21, 2 * d)).astype(np.float32)
        for lo, hi in ((0, first), (first, 64)):
            if hi > lo:
                t = give(dev, a[lo:hi])
                paged.append(c.plan([lo], [hi - lo]), c.cache, None, 0, t, 0, t, d)
        t = give(dev, b)
        paged.append(c.plan([at], [21]), c.cache, None, 0, t, 0, t, d)
        every = np.concatenate([a[:at], b])
        x = {"k": every[:, None, :d], "v": every[:, None, d:]}
        end = len(every)
        for name in ("k", "v"):
            for blk in range(end // P):                      # the reference's block from all of the sequence's rows, not by way of open ones
                code, factor = R.codes(R.f16(x[name][blk * P:(blk + 1) * P, 0]))
                np.testing.assert_array_equal(take(dev, getattr(c.cache, name))[c.table[0][blk], 0], code)
                assert take(dev, getattr(c.cache, name + "_scale"))[c.table[0][blk], 0] == factor
            got = take(dev, getattr(c.cache, name + "_open"))[2 * c.slot(0) + end // P % 2, 0, :end % P]
            np.testing.assert_array_equal(got, R.f16(x[name][end // P * P:, 0]))


def test_numbers_at_the_ends(dev):
    """numbers beyond 16 bits, zeros, subnormal ones, ties, infinities and NaN; blocks of other heads stay clean"""
    G, d, P = 4, 16, 16
    c = Case(dev, P, G, d, d, True, [0], [48], seed=1)
    x = np.random.default_rng(2).normal(size=(48, G, d)).astype(np.float32)
    x[3, 0, 1], x[4, 0, 2] = 1e9, -7e4                       # saturate
    x[:16, 1] = 0.0
    x[16:32, 0] = np.linspace(-3e-8, 6e-8, 16)[:, None]      # subnormal
    x[16:32, 1] = np.arange(-8, 8)[:, None] + np.linspace(-0.5, 0.5, 16).round(1)
    x[16:32, 2] = np.arange(-127, 129).reshape(16, 16) / 2   # codes k + 1/2 with a = 64: 127 x / 64 is no tie, with a = 63.5 it is
    x[16:32, 2][x[16:32, 2] > 63.5] = 63.5
    x[16 + 15, 3, 15], x[17, 2, 0] = np.inf, -63.5
    x[35, 1, 0] = np.nan
    t = give(dev, np.concatenate([x.reshape(48, -1), x.reshape(48, -1)], 1))
    paged.append(c.plan(), c.cache, None, 0, t, 0, t, G * d)
    c.ref.append(c.table[0], 0, c.slot(0), {"k": x, "v": x})
    c.same()
    scale = take(dev, c.cache.k_scale)
    assert np.isnan(scale[c.table[0][1], 3]) and np.isnan(scale[c.table[0][2], 1]) and np.isfinite(np.delete(scale[c.table[0][2]], 1)).all()


# ---- attention -----------------------------------------------------------------------------------------------------------------------------
def check_attention(dev, P, G, Rh, dk, dv, i8, pos0, counts, window=0, softcap=0.0, sink=False, seed=0, q_scale=1.0, mend=None):
    c = Case(dev, P, G, dk, dv, i8, pos0, counts, seed=seed)
    if mend:
        mend(c)
        c.cache = paged.PagedCache(**{n: give(dev, a) for n, a in c.ref.a.items()})
    if i8:                                                   # keys and values of about unit size
        for n in ("k", "v"):
            c.ref.a[n + "_scale"] /= np.float32(60)
            c.cache = paged.PagedCache(**{m: give(dev, a) for m, a in c.ref.a.items()}) if n == "v" else c.cache
    H, T = G * Rh, sum(counts)
    q = (c.rng.normal(size=(T, H, dk)) * q_scale).astype(np.float32)
    s = c.rng.normal(size=H).astype(np.float32) if sink else None
    scale = dk ** -0.5
    y = paged.attention(c.plan(), c.cache, give(dev, q.reshape(T, -1)), H, scale, window=window, softcap=softcap, sink=None if s is None else give(dev, s))
    got, at = take(dev, y).reshape(T, H, dv), 0
    for i, n in enumerate(counts):
        if n:
            k, v = (c.ref.rows(m, c.table[i], pos0[i] + n, c.slot(i)) for m in ("k", "v"))
            want, mass, reach = R.attention(q[at:at + n], k, v, pos0[i], float(np.float32(scale)), window, softcap, s)
            tol = R.attention_bound(mass, reach, dk, pos0[i] + n)
            bad = np.abs(got[at:at + n] - want) > tol
            assert not bad.any(), (i, np.argwhere(bad)[:3], np.abs(got[at:at + n] - want)[bad][:3], tol[bad][:3])
        at += n
    return c, q, got


SHAPES = [  # G, heads a key head, dk, dv
    (1, 1, 16, 16), (2, 4, 64, 64), (2, 1, 128, 128), (1, 8, 128, 128), (1, 5, 80, 96), (2, 3, 96, 48), (1, 2, 256, 256), (1, 16, 64, 128), (1, 7, 192, 128), (1, 4, 32, 256),
]


@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
@pytest.mark.parametrize("shape", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
def test_attention_shapes(dev, shape, i8):
    G, Rh, dk, dv = shape
    check_attention(dev, 32, G, Rh, dk, dv, i8, [0, 100, 31, 32, 700], [1, 1, 1, 2, 1], seed=dk)


TILES = [(1, 1, 16, 16), (2, 4, 64, 64), (1, 8, 128, 128), (2, 3, 80, 96), (1, 5, 96, 48), (1, 2, 32, 128), (1, 7, 112, 16), (1, 2, 256, 128), (1, 1, 64, 256)]


@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
@pytest.mark.parametrize("shape", TILES, ids=["x".join(map(str, s)) for s in TILES])
def test_attention_of_many_rows(dev, shape, i8):
    """prompts of ragged lengths, from the start and late, beside a decoded token and a sequence at rest"""
    G, Rh, dk, dv = shape
    check_attention(dev, 32, G, Rh, dk, dv, i8, [0, 100, 31, 5, 300], [70, 33, 0, 1, 129], seed=dk + dv)


@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
@pytest.mark.parametrize("P,pos0,counts,kw", [(16, [5000], [20], {}), (64, [2999, 10], [17, 300], {}), (128, [4500], [40], dict(window=3000, sink=True)), (32, [0], [600], dict(softcap=20.0)),
                                              (64, [1000], [50], dict(window=1)), (16, [3000], [33], dict(window=130, sink=True, softcap=5.0))],
                         ids=["slices", "mixed", "window", "prompt", "itself", "all"])
def test_attention_of_many_rows_far(dev, P, pos0, counts, kw, i8):
    """few rows over long caches are dealt out in slices; windows that leave most of a cache out"""
    check_attention(dev, P, 1, 8, 64, 64, i8, pos0, counts, seed=P, **kw)


@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
@pytest.mark.parametrize("P", [16, 32, 64, 128])
@pytest.mark.parametrize("pos0,counts", [([0], [1]), ([14, 15, 16], [1, 1, 1]), ([2000], [1]), ([0, 0, 5], [17, 0, 40]), ([127, 128, 129, 640], [3, 1, 2, 64]), ([0], [200])],
                         ids=["first", "ends", "long", "prompts", "drafts", "prompt"])
def test_attention_lengths(dev, P, i8, pos0, counts):
    check_attention(dev, P, 2, 4, 64, 64, i8, pos0, counts, seed=P + len(pos0))


@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
@pytest.mark.parametrize("window,softcap,sink", [(1, 0.0, False), (2, 0.0, True), (16, 5.0, False), (17, 0.0, False), (100, 30.0, True), (5000, 0.0, True), (0, 2.0, True)])
def test_attention_masks(dev, window, softcap, sink, i8):
    check_attention(dev, 32, 1, 4, 64, 48, i8, [0, 33, 500, 64], [1, 5, 1, 90], window=window, softcap=softcap, sink=sink, seed=window)


@pytest.mark.parametrize("q_scale", [1e-30, 1e-4, 30.0, 3000.0])
@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
def test_attention_sizes_of_numbers(dev, q_scale, i8):
    """queries of any size, blocks whose factors differ by orders of magnitude, blocks of zeros"""
    def mend(c):
        r = np.random.default_rng(4)
        if c.i8:
            for n in ("k_scale", "v_scale"):
                c.ref.a[n] *= (10.0 ** r.uniform(-3, 3, c.ref.a[n].shape)).astype(np.float32)
            c.ref.a["v_scale"][c.table[0][:2]] = 0
            c.ref.a["v"][c.table[0][:2]] = 0
        else:
            c.ref.a["v"] = (c.ref.a["v"].astype(np.float32) * 1000).astype(np.float16)
    check_attention(dev, 32, 1, 4, 64, 64, i8, [500, 40], [1, 3], q_scale=q_scale, seed=9, mend=mend)


@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
@pytest.mark.parametrize("counts", [[1, 6], [1, 70], [1, 300]], ids=["few", "many", "more"])
def test_what_a_query_does_not_see(dev, i8, counts):
    """NaN and infinities in keys and values reach the queries that see them and no others; rows behind a sequence's end are not looked at"""
    G, Rh, d, P, pos0 = 1, 4, 64, 32, [40, 100]
    clean = check_attention(dev, P, G, Rh, d, d, i8, pos0, counts, window=50, seed=21)

    def poisoned(bad):
        c = Case(dev, P, G, d, d, i8, pos0, counts, seed=21)
        for n in c.ref.a:
            c.ref.a[n] = clean[0].ref.a[n].copy()
        bad(c.ref.a, c)
        cache = paged.PagedCache(**{n: give(dev, a) for n, a in c.ref.a.items()})
        T, H = sum(counts), G * Rh
        return take(dev, paged.attention(c.plan(), cache, give(dev, clean[1].reshape(T, -1)), H, d ** -0.5, window=50)).reshape(T, H, d)

    end = pos0[1] + counts[1]

    def place(c, name, pos):                                 # array and index of a row of the second sequence
        b = pos // P
        if i8 and (b + 1) * P > end:
            return name + "_open", (2 * c.slot(1) + b % 2, 0, pos % P)
        return (name, (c.table[1][b], 0, pos % P)) if not i8 else (name + "_scale", (c.table[1][b], 0))

    for what in (np.nan, np.inf, -np.inf):
        # 1. rows behind the ends and pages of nobody
        def behind(a, c):
            for n in ("k", "v"):
                for i in range(2):
                    e = pos0[i] + counts[i]
                    if e % P:
                        if i8:
                            a[n + "_open"][2 * c.slot(i) + e // P % 2, :, e % P:] = what
                            a[n + "_scale"][c.table[i][e // P]] = np.nan
                        else:
                            a[n][c.table[i][e // P], :, e % P:] = what
        np.testing.assert_array_equal(poisoned(behind), clean[2])
        for name in ("k", "v"):
            # 2. the last token's row: only it sees it (16 bits, or the open block)
            if not i8 or end % P:
                def last(a, c):
                    n, at = place(c, name, end - 1)
                    a[n][at][3] = what
                got = poisoned(last)
                np.testing.assert_array_equal(got[:-1], clean[2][:-1])
                if name == "v" or np.isnan(what):
                    assert not np.isfinite(got[-1][..., 3]).any()
            # 3. an old row: out of everybody's window but the first one's
            def old(a, c):
                n, at = place(c, name, pos0[1] - 49)
                if i8:
                    a[n][at] = np.nan
                else:
                    a[n][at][3] = what
            got = poisoned(old)
            first = counts[0]
            span = (pos0[1] - 49) // P * P + P - 1 + 50 if i8 else pos0[1] + 1                # queries from here on do not see the block (row)
            np.testing.assert_array_equal(got[:first], clean[2][:first])
            np.testing.assert_array_equal(got[first + max(0, span - pos0[1]):], clean[2][first + max(0, span - pos0[1]):])
            if i8 or np.isnan(what):
                assert np.isnan(got[first][..., 3]).all()


def test_a_shared_prefix(dev):
    """two sequences read the same pages and go on in their own"""
    G, d, P = 2, 32, 16
    c = Case(dev, P, G, d, d, True, [32, 32], [3, 5], seed=5)
    c.table[1][:2] = c.table[0][:2]
    q = c.rng.normal(size=(8, 2 * d)).astype(np.float32)
    got = take(dev, paged.attention(c.plan(), c.cache, give(dev, q), 2, 0.1)).reshape(8, 2, d)
    for i, (lo, hi) in enumerate(((0, 3), (3, 8))):
        k, v = (c.ref.rows(m, c.table[i], 32 + hi - lo, c.slot(i)) for m in ("k", "v"))
        want, mass, reach = R.attention(q[lo:hi].reshape(-1, 2, d), k, v, 32, float(np.float32(0.1)))
        assert (np.abs(got[lo:hi] - want) <= R.attention_bound(mass, reach, d, 40)).all()


def test_many_sequences(dev):
    """more sequences than lanes of a warp, lengths of all kinds, some at rest"""
    r = np.random.default_rng(8)
    pos0, counts = r.integers(0, 90, 70).tolist(), r.choice([0, 1, 1, 1, 2, 12], 70).tolist()
    check_attention(dev, 16, 1, 2, 32, 32, True, pos0, counts, seed=6)


@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
@pytest.mark.parametrize("seed,G,Rh,d,n,top,window", [(1, 3, 4, 64, 20, 1500, 0), (2, 2, 8, 128, 40, 900, 0), (3, 1, 1, 32, 3, 9000, 0), (4, 4, 5, 80, 9, 3000, 700), (5, 1, 2, 256, 12, 2500, 0), (6, 8, 1, 16, 30, 600, 0)])
def test_attention_in_runs(dev, seed, G, Rh, d, n, top, window, i8):
    """few rows over sequences of all lengths: equal runs of keys begin and end anywhere in them"""
    r = np.random.default_rng(seed)
    pos0 = np.where(r.random(n) < 0.3, r.integers(0, 70, n), r.integers(0, top, n)).tolist()
    counts = r.choice([0, 1, 1, 1, 2, 32 // Rh], n).tolist()
    pos0[0], counts[0] = top, 1
    check_attention(dev, 32, G, Rh, d, d, i8, pos0, counts, window=window, seed=seed)


@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
@pytest.mark.parametrize("window,softcap,sink", [(0, 0.0, True), (1500, 30.0, False), (2999, 3.0, True)])
def test_attention_in_runs_masks(dev, window, softcap, sink, i8):
    """a sink's share and capped scores where a row's sums come from several CTAs"""
    check_attention(dev, 16, 2, 3, 48, 80, i8, [4000, 2500, 100, 3100], [1, 3, 2, 10], window=window, softcap=softcap, sink=sink, seed=window)


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("lead", [1.0, 3.0, 4.999, 5.9995, 5.99995, 6.01, 9.0])
def test_attention_of_a_later_larger_score(dev, lead, n):
    """a score that outgrows the ones before it by a little, beside the largest value factor that a power of two leaves room for"""
    P, d, end = 16, 16, 160
    c = Case(dev, P, 1, d, d, True, [end - n], [n], seed=2)
    a = c.ref.a
    a["k"][:] = 0
    a["k_scale"][:] = 1
    a["v_scale"][:] = np.float32(1.9999999)
    a["k"][c.table[0][4], 0, 3, 0] = 1                       # key 67: score of lead * ln 2, the others 0
    a["k_scale"][c.table[0][4]] = np.float32(lead * np.log(2.0))
    c.cache = paged.PagedCache(**{m: give(dev, x) for m, x in a.items()})
    q = np.zeros((n, 1, d), np.float32)
    q[:, 0, 0] = 1
    got = take(dev, paged.attention(c.plan(), c.cache, give(dev, q.reshape(n, -1)), 1, 1.0)).reshape(n, 1, d)
    k, v = (c.ref.rows(m, c.table[0], end, c.slot(0)) for m in ("k", "v"))
    want, mass, reach = R.attention(q, k, v, end - n, 1.0)
    assert (np.abs(got - want) <= R.attention_bound(mass, reach, d, end)).all()


@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
def test_rows_over_thousands_of_keys(dev, i8):
    """eight rows at a time over more keys than a CTA holds page numbers of"""
    d, Rh, pos0, n = 256, 8, 4400, 1190
    c = Case(dev, 16, 1, d, d, i8, [pos0], [n], seed=3)
    q = c.rng.normal(size=(n, Rh, d)).astype(np.float32)
    scale = d ** -0.5 / (60 if i8 else 1)
    got = take(dev, paged.attention(c.plan(), c.cache, give(dev, q.reshape(n, -1)), Rh, scale)).reshape(n, Rh, d)
    k, v = (c.ref.rows(m, c.table[0], pos0 + n, c.slot(0)) for m in ("k", "v"))
    for t in (0, 600, n - 3):
        want, mass, reach = R.attention(q[t:t + 3], k[:, :pos0 + t + 3], v[:, :pos0 + t + 3], pos0 + t, float(np.float32(scale)))
        assert (np.abs(got[t:t + 3] - want) <= R.attention_bound(mass, reach, d, pos0 + t + 3)).all()


@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
def test_many_rows_over_many_keys(dev, i8):
    """many rows whose keys and values, all heads' together, are more than are unpacked at a time"""
    G, d, pos0, n, seqs = 8, 128, 2968, 40, 24
    c = Case(dev, 64, G, d, d, i8, [pos0] + [0] * (seqs - 1), [n] + [0] * (seqs - 1), spare=seqs, seed=4)
    assert (pos0 + n) % 64 == 0
    last, spare = c.table[0][-1], sorted(set(range(c.n_pages)) - set(c.table[0]))
    for name in ("k", "v") + (("k_scale", "v_scale") if i8 else ()):
        c.ref.a[name][spare] = c.ref.a[name][last]
    c.cache = paged.PagedCache(**{m: give(dev, a) for m, a in c.ref.a.items()})
    table = [c.table[0][:-1] + [p] for p in [last] + spare[:seqs - 1]]               # all read the same pages but the last, whose contents are the same
    plan = paged.PagePlan(dev, 64, c.n_pages, table, [pos0] * seqs, [n] * seqs, c.n_slots, c.slots)
    q = c.rng.normal(size=(n, G, d)).astype(np.float32)
    scale = d ** -0.5 / (60 if i8 else 1)
    got = take(dev, paged.attention(plan, c.cache, give(dev, np.tile(q.reshape(n, -1), (seqs, 1))), G, scale)).reshape(seqs, n, G, d)
    k, v = (c.ref.rows(m, c.table[0], pos0 + n, c.slot(0)) for m in ("k", "v"))
    want, mass, reach = R.attention(q, k, v, pos0, float(np.float32(scale)))
    assert (np.abs(got[0] - want) <= R.attention_bound(mass, reach, d, pos0 + n)).all()
    for i in range(1, seqs):
        np.testing.assert_array_equal(got[i], got[0])


@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
@pytest.mark.parametrize("sink", [False, True])
def test_many_slices(dev, sink, i8):
    """a few dozen rows over so many keys that each has more slices than a warp has lanes"""
    check_attention(dev, 128, 1, 1, 16, 32, i8, [140000, 90], [40, 40], sink=sink, seed=17)


@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-20])
def test_attention_scales(dev, scale, i8):
    """the smallest scores are the largest, and every key weighs the same"""
    c = Case(dev, 16, 1, 32, 32, i8, [700, 20], [2, 60], seed=12)
    q = (c.rng.normal(size=(62, 2, 32)) / (60 if i8 else 1)).astype(np.float32)
    got = take(dev, paged.attention(c.plan(), c.cache, give(dev, q.reshape(62, -1)), 2, scale)).reshape(62, 2, 32)
    for i, (lo, hi) in enumerate(((0, 2), (2, 62))):
        end = c.pos0[i] + hi - lo
        k, v = (c.ref.rows(m, c.table[i], end, c.slot(i)) for m in ("k", "v"))
        want, mass, reach = R.attention(q[lo:hi], k, v, c.pos0[i], float(np.float32(scale)))
        assert (np.abs(got[lo:hi] - want) <= R.attention_bound(mass, reach, 32, end)).all()


def test_offsets_beyond_32_bits(dev):
    """pages behind element 2^31 of their tensor"""
    G, d, P, n = 8, 128, 64, 33000
    cache = paged.PagedCache.alloc(dev, n, G, P, d, dtype=capi.I8, n_slots=1)
    assert n * G * P * d > 1 << 31
    src = np.random.default_rng(1).normal(size=(130, 2 * G * d)).astype(np.float32)
    t = give(dev, src)
    plan = paged.PagePlan(dev, P, n, [[n - 1, n - 2, n - 3]], [0], [130], 1)
    paged.append(plan, cache, None, 0, t, 0, t, G * d)
    ref = R.Cache(3, G, P, d, d, True, 1)
    ref.append([2, 1, 0], 0, 0, {"k": src[:, :G * d].reshape(130, G, d), "v": src[:, G * d:].reshape(130, G, d)})
    q = np.random.default_rng(2).normal(size=(130, G * d)).astype(np.float32)
    got = take(dev, paged.attention(plan, cache, give(dev, q), G, 0.1)).reshape(130, G, d)
    want, mass, reach = R.attention(q.reshape(130, G, d)[-2:], ref.rows("k", [2, 1, 0], 130, 0), ref.rows("v", [2, 1, 0], 130, 0), 128, float(np.float32(0.1)))
    assert (np.abs(got[-2:] - want) <= R.attention_bound(mass, reach, d, 130)).all()


def test_nothing_to_do(dev):
    c = Case(dev, 16, 1, 16, 16, True, [5, 0], [0, 0], seed=1)
    before = {n: a.copy() for n, a in c.ref.a.items()}
    empty = CudaTensor.alloc([0, 48], capi.F32, dev)
    assert paged.append(c.plan(), c.cache, empty, 0, empty, 16, empty, 32, 1).shape() == [0, 16]
    assert paged.attention(c.plan(), c.cache, CudaTensor.alloc([0, 16], capi.F32, dev), 1, 1.0).shape() == [0, 16]
    for n, a in before.items():
        np.testing.assert_array_equal(take(dev, getattr(c.cache, n)), a)
    plan = paged.PagePlan(dev, 16, 0, [], [], [])
    assert plan.tokens == 0


def test_a_plan_outlives_nothing(dev):
    """a plan that is released while its work is queued, and plans that take its place in memory at once"""
    G, d, P = 1, 64, 16
    c = Case(dev, P, G, d, d, True, [400, 300], [1, 1], seed=14)
    q = give(dev, c.rng.normal(size=(2, 4 * d)).astype(np.float32))
    want = take(dev, paged.attention(c.plan(), c.cache, q, 4, 0.125))
    outs = []
    for i in range(30):
        plan = c.plan()
        outs.append(paged.attention(plan, c.cache, q, 4, 0.125))
        del plan
        c.plan([16, 17], [1, 1])
    for y in outs:
        np.testing.assert_array_equal(take(dev, y), want)


def test_plans_do_not_wait_for_the_device(dev):
    """a host that makes plans, larger ones too, for many steps ahead while the device is busy; what they say arrives all the same"""
    G, d, P, n = 1, 32, 16, 24
    c = Case(dev, P, G, d, d, True, [200, 40], [1, 1], seed=15)
    q = give(dev, c.rng.normal(size=(2, 2 * d)).astype(np.float32))
    want = [take(dev, paged.attention(c.plan([100 + i, 40 - i], [1, 1]), c.cache, q, 2, 0.1)) for i in range(n)]
    large = [paged.PagePlan(dev, P, 1 << 20, [list(range(30000))], [16 * 30000 - 1], [1], 1) for _ in range(2)]
    dev.synchronize()
    stream = torch.cuda.ExternalStream(dev.stream())
    with torch.cuda.stream(stream):
        torch.cuda._sleep(2_000_000_000)                     # about a second
    busy = stream.record_event()
    plans = [c.plan([100 + i, 40 - i], [1, 1]) for i in range(n)] + [paged.PagePlan(dev, P, 1 << 20, [list(range(30000))], [16 * 30000 - 1], [1], 1)]
    assert not busy.query()
    for i, plan in enumerate(plans[:n]):
        np.testing.assert_array_equal(take(dev, paged.attention(plan, c.cache, q, 2, 0.1)), want[i])
    del large, plans


def test_two_devices_at_once():
    """two threads, a device each, append to blocks of different sizes: one's launches do not depend on what the other asks of the same kernel in between"""
    import threading
    failed, devs, work = [], [make_device(), make_device()], []
    for dev, d in zip(devs, (256, 192)):  # noqa: F402
        P, G = 128, 1
        cache = paged.PagedCache.alloc(dev, 2, G, P, d, dtype=capi.I8, n_slots=1)
        src = give(dev, np.random.default_rng(d).normal(size=(1, 2 * d)).astype(np.float32))
        plan = paged.PagePlan(dev, P, 2, [[0]], [5], [1], 1)
        paged.append(plan, cache, None, 0, src, 0, src, d)
        work.append((plan, cache, src, d))

    def go(plan, cache, src, d):
        try:
            for _ in range(20000):
                paged.append(plan, cache, None, 0, src, 0, src, d)
        except Exception as e:                               # noqa: BLE001
            failed.append(e)
    threads = [threading.Thread(target=go, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for dev in devs:
        dev.synchronize()
    del work
    for dev in devs:
        dev.close()
    assert not failed, failed


# ---- refusals -------------------------------------------------------------------------------------------------------------------------------
def test_refusals(dev):
    G, H, d, P = 2, 4, 32, 16
    c = Case(dev, P, G, d, d, True, [3], [2], seed=1)
    plan, t = c.plan(), give(dev, np.zeros((2, (H + 2 * G) * d), np.float32))
    short = give(dev, np.zeros((1, (H + 2 * G) * d), np.float32))
    q = give(dev, np.zeros((2, H * d), np.float32))
    f = give(dev, freqs(d // 2))

    def append(cache=c.cache, src=t, kc=H * d, vc=(H + G) * d, heads=H, plan=plan, **kw):
        return paged.append(plan, cache, src, 0, src, kc, src, vc, heads, **kw)

    def attend(cache=c.cache, qt=q, heads=H, plan=plan, **kw):
        return paged.attention(plan, cache, qt, heads, 1.0, **kw)

    append(), attend()                                       # as it should be
    a = {n: getattr(c.cache, n) for n in c.ref.a}
    bad = [dict(a, k=a["v"].reshape([c.n_pages, G, P * d, 1])), dict(a, v=give(dev, np.zeros((c.n_pages, G, P, d), np.float16))), dict(a, k_scale=None),
           dict(a, v_scale=give(dev, np.zeros((c.n_pages, G + 1), np.float32))), dict(a, k_open=give(dev, np.zeros((2, G, P, d), np.float16))),
           dict(a, k=give(dev, np.zeros((c.n_pages - 1, G, P, d), np.int8))), dict(a, v_open=give(dev, np.zeros((2 * c.n_slots, G, P, d + 16), np.float16))),
           dict(a, k=give(dev, np.zeros((c.n_pages, G, P, d), np.float32)))]
    for x in bad:
        for call in (append, attend):
            with pytest.raises((TensorError, CudaError)):
                call(cache=paged.PagedCache(**x))
    for call in (append, attend):
        with pytest.raises((TensorError, CudaError)):
            call(heads=8194)
    for kw in (dict(src=short), dict(kc=H * d + 1, vc=(H + G) * d + 1), dict(kc=-1), dict(vc=1 << 30), dict(heads=3), dict(heads=0), dict(pairing=2), dict(freq=f, offset=1),
               dict(freq=f, offset=-1), dict(freq=give(dev, np.zeros(4, np.int8)))):
        with pytest.raises((TensorError, CudaError)):
            append(**kw)
    for kw in (dict(qt=short), dict(heads=3), dict(heads=0), dict(sink=f), dict(qt=give(dev, np.zeros((2, H * d + 1), np.float32))),
               dict(qt=give(dev, np.zeros((2, H * d), np.float16)))):
        with pytest.raises((TensorError, CudaError)):
            attend(**kw)
    with pytest.raises(TensorError):                         # codes need open blocks
        append(plan=paged.PagePlan(dev, P, c.n_pages, c.table, [3], [2]))
    with pytest.raises(TensorError):                         # pages of another size than the plan's
        append(plan=paged.PagePlan(dev, 32, c.n_pages, c.table, [3], [2], 1))
    for sizes in ((24, 32), (272, 32), (32, 8)):
        with pytest.raises(TensorError):
            append(cache=paged.PagedCache.alloc(dev, c.n_pages, G, P, *sizes, dtype=capi.I8, n_slots=c.n_slots))
    for kw in (dict(table=[[0]], pos0=[0, 1], counts=[1]), dict(table=[[0], [1]], pos0=[0], counts=[1]), dict(table=[[7]], pos0=[0], counts=[1]), dict(table=[[0]], pos0=[16], counts=[1])):
        with pytest.raises(TensorError):
            paged.PagePlan(dev, 16, 4, **kw)
    lazy = make_device(lazy=True)
    with pytest.raises(CudaError):
        paged.PagePlan(lazy, 16, 4, [[0]], [0], [1])
    other = make_device()
    with pytest.raises(TensorError):                         # a plan, and a cache, of another device object
        paged.attention(paged.PagePlan(other, P, c.n_pages, c.table, [3], [2], c.n_slots), c.cache, q, H, 1.0)
    for d2 in (lazy, other):
        d2.close()
    append(), attend()


@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
def test_one_tensor_for_keys_and_values(dev, i8):
    """nothing says which of the two would be there in the end: the append refuses it; attention only reads, and may"""
    G, d, P = 2, 32, 16
    c = Case(dev, P, G, d, d, i8, [20], [2], seed=1)
    t = give(dev, np.zeros((2, 2 * G * d), np.float32))
    a = {n: getattr(c.cache, n) for n in c.ref.a}
    for one, other in (("k", "v"), ("k_scale", "v_scale"), ("k_open", "v_open")):
        if one in a:
            with pytest.raises(TensorError):
                paged.append(c.plan(), paged.PagedCache(**dict(a, **{other: a[one]})), None, 0, t, 0, t, G * d)
    both = dict(a, **{n.replace("k", "v", 1): a[n] for n in a if n[0] == "k"})
    q = give(dev, c.rng.normal(size=(2, G * d)).astype(np.float32))
    got = take(dev, paged.attention(c.plan(), paged.PagedCache(**both), q, G, 0.1))
    twice = {n: give(dev, c.ref.a[n if n[0] == "k" else n.replace("v", "k", 1)]) for n in a}
    np.testing.assert_array_equal(got, take(dev, paged.attention(c.plan(), paged.PagedCache(**twice), q, G, 0.1)))
    paged.append(c.plan(), c.cache, None, 0, t, 0, t, G * d)


def test_arrays_of_a_tensor(dev):
    """what other libraries see of a tensor is its memory"""
    a = np.arange(24, dtype=np.float32).reshape(4, 6)
    t = CudaTensor.new(a, [4, 6], dev)
    dev.synchronize()
    np.testing.assert_array_equal(torch.as_tensor(t, device="cuda").cpu().numpy(), a)
    np.testing.assert_array_equal(torch.as_tensor(t.transpose([1, 0]), device="cuda").cpu().numpy(), a.T)
    torch.as_tensor(t, device="cuda").add_(1.0)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(t.export().reshape(4, 6), a + 1)
    first = t.__cuda_array_interface__
    first["data"] = None                                     # what a caller does to it is the caller's
    assert t.__cuda_array_interface__["data"][0] == torch.as_tensor(t, device="cuda").data_ptr()
    u = CudaTensor.new(a, [4, 6], dev)
    assert u.__cuda_array_interface__["shape"] == (4, 6)
    v = u.reshape([6, 4])
    assert v.__cuda_array_interface__["shape"] == (6, 4) and v.__cuda_array_interface__["data"] == u.__cuda_array_interface__["data"]
    gone = make_device()
    w = CudaTensor.new(a, [4, 6], gone)
    assert w.__cuda_array_interface__["data"][0]
    gone.close()
    with pytest.raises(CudaError):
        w.__cuda_array_interface__
    q = CudaTensor.from_cpu(np.zeros(34 * 2, np.uint8), [2, 32], capi.Q8_0, dev)
    assert not hasattr(q, "__cuda_array_interface__")
    assert CudaTensor.alloc([0, 3], capi.I8, dev).__cuda_array_interface__["data"][0] == 0
    with pytest.raises(TensorError):
        CudaTensor.alloc([1, 4], capi.F32, dev).copy_rows_from(CudaTensor.alloc([1, 4], capi.I8, dev), [0])
    assert seqops is not None
