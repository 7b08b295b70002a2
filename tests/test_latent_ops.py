"""Latent rows in pages (include/crabml_paged.h): the append and the attention in both forms against plain references in 64 bits (tests/latent_ref.py), with the lengths,
strides, masks and numbers at which they can go wrong."""
import numpy as np
import pytest

from crabml_b200 import CudaTensor, TensorError, CudaError, TensorStrider, capi, paged
from tests import latent_ref as R
from tests.gpu_common import make_device

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

FORMS = {"absorbed": capi.LATENT_ABSORBED, "expanded": capi.LATENT_EXPANDED}


@pytest.fixture(scope="module")
def dev():
    d = make_device()
    yield d
    d.close()


TYPES = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}


def view(t):
    return torch.as_tensor(t.bits(), device="cuda").view(torch.bfloat16) if t.dtype() == capi.BF16 else torch.as_tensor(t, device="cuda")


def give(dev, a, dtype=None):
    a = torch.from_numpy(np.ascontiguousarray(a))
    a = a if dtype is None else a.to(dtype)
    t = CudaTensor.alloc(list(a.shape), TYPES[a.dtype], dev)
    dev.synchronize()
    if a.numel():
        view(t).copy_(a)
    torch.cuda.synchronize()
    return t


def take(dev, t):
    dev.synchronize()
    return view(t).float().cpu().numpy()


def freqs(n, base=10000.0):
    return (base ** (-np.arange(n) / max(n, 1))).astype(np.float32)


class Case:
    """sequences of given lengths over shuffled pages; what lies behind a sequence's end, and pages that no one has, is NaN"""

    def __init__(self, dev, P, rank, rest, pos0, counts, spare=2, seed=0):
        r = np.random.default_rng(seed)
        self.dev, self.P, self.rank, self.rest, self.pos0, self.counts, self.rng = dev, P, rank, rest, list(pos0), list(counts), r
        need = [(p + c + P - 1) // P for p, c in zip(pos0, counts)]
        self.n_pages = sum(need) + spare
        pages, cut = r.permutation(self.n_pages), np.cumsum([0] + need)
        self.table = [pages[cut[i]:cut[i + 1]].tolist() for i in range(len(need))]
        self.a = np.full((self.n_pages, P, rank + rest), np.nan, np.float16)
        for i in range(len(need)):
            self.put(i, 0, r.normal(size=(pos0[i] + counts[i], rank + rest)).astype(np.float16))

    def put(self, i, pos, rows):
        for j, x in enumerate(rows):
            self.a[self.table[i][(pos + j) // self.P], (pos + j) % self.P] = x

    def rows(self, i, n):
        return np.stack([self.a[self.table[i][j // self.P], j % self.P] for j in range(n)]) if n else np.zeros((0, self.rank + self.rest), np.float16)

    def plan(self):
        return paged.PagePlan(self.dev, self.P, self.n_pages, self.table, self.pos0, self.counts)

    def positions(self):
        return np.concatenate([np.arange(p, p + n) for p, n in zip(self.pos0, self.counts)]) if self.counts else np.zeros(0)


# ---- append -------------------------------------------------------------------------------------------------------------------------------
LENGTHS = [([0], [1]), ([15], [1]), ([16], [1]), ([300], [1]), ([127], [2]), ([0], [128]), ([5], [300]), ([130, 7, 64], [1, 0, 1]), ([0, 0, 40], [0, 33, 100]), ([63, 64, 65, 1000], [1, 1, 70, 16])]


def near16(got, want, steps=1.0):
    """16-bit results of 32-bit steps: half a step of 2^-11 and what the steps before it are off by (2^-22 of the value and its terms: norm and turn are a few operations), beside
    the smallest numbers' 2^-25"""
    want = np.asarray(want, np.float64)
    np.testing.assert_allclose(got, np.clip(want, -65504, 65504), rtol=steps * 2.0 ** -11 + 2.0 ** -19, atol=2.0 ** -25 + 2.0 ** -19)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("P", [16, 64, 128])
@pytest.mark.parametrize("pos0,counts", LENGTHS, ids=[str(i) for i in range(len(LENGTHS))])
def test_append(dev, P, dtype, pos0, counts):
    H, dim, rest, rank = 3, 32, 16, 48
    c = Case(dev, P, rank, rest, pos0, counts, seed=P)
    T, odd = sum(counts), 8 if dtype == torch.float32 else 3                # rows that start at a multiple of 16 bytes, and others
    src = torch.from_numpy(c.rng.normal(size=(T, H * (dim + rest) + odd + rank + rest + 5)) * np.exp(c.rng.normal(size=(T, 1)))).to(dtype)
    kc, w, f = H * (dim + rest) + odd, c.rng.normal(size=rank).astype(np.float32), freqs(rest // 2)
    pages, t = give(dev, c.a), give(dev, src.float().numpy(), dtype)
    q = paged.latent_append(c.plan(), pages, rank, t, kc, norm_w=give(dev, w), eps=1e-5, q_src=t, n_heads=H, dim=dim, freq=give(dev, f))
    x, pos, was = src.double().numpy(), c.positions(), c.a.copy()
    want = x[:, :H * (dim + rest)].reshape(T, H, dim + rest).copy()
    want[..., dim:] = R.turn(want[..., dim:], pos, f, 0, 1.0)
    assert q.shape() == [T, H * (dim + rest)] and q.dtype() == capi.F16
    near16(take(dev, q).reshape(want.shape), want)
    rows, at = R.row(x[:, kc:kc + rank + rest], rank, w, 1e-5, pos, f, 0, 1.0), 0
    got = take(dev, pages)
    for i, n in enumerate(counts):
        for j in range(n):
            p = pos0[i] + j
            near16(got[c.table[i][p // P], p % P], rows[at + j])
            was[c.table[i][p // P], p % P] = got[c.table[i][p // P], p % P]
        at += n
    np.testing.assert_array_equal(got, was.astype(np.float32))               # every other row is as it was


@pytest.mark.parametrize("pairing,n,mag", [(0, 32, 1.0), (1, 32, 1.0), (0, 8, 1.25), (1, 17, 0.7), (1, 0, 1.0), (0, 1, 1.0)])
def test_append_turns(dev, pairing, n, mag):
    """both pairings, part of the columns, a factor; at positions where 32 bits lose the angle"""
    H, dim, rest, rank, P = 2, 16, 64, 16, 16
    pos0, counts = [1000003 // P * P - 5, 31], [23, 1]
    need = [(p + k + P - 1) // P for p, k in zip(pos0, counts)]
    table = [[0] * (need[0] - 3) + [1, 2, 3], [4, 5]]
    r = np.random.default_rng(n)
    T, f = sum(counts), freqs(n)
    src = r.normal(size=(T, H * (dim + rest) + rank + rest)).astype(np.float32)
    pages, t = give(dev, np.zeros((6, P, rank + rest), np.float16)), give(dev, src)
    plan = paged.PagePlan(dev, P, 6, table, pos0, counts)
    q = paged.latent_append(plan, pages, rank, t, H * (dim + rest), eps=0.0, q_src=t, n_heads=H, dim=dim, freq=give(dev, f), pairing=pairing, mag=mag)
    pos = np.concatenate([np.arange(p, p + k) for p, k in zip(pos0, counts)])
    want = src[:, :H * (dim + rest)].reshape(T, H, -1).astype(np.float64)
    want[..., dim:] = R.turn(want[..., dim:], pos, f, pairing, mag)
    near16(take(dev, q).reshape(want.shape), want)
    rows, got = R.row(src[:, H * (dim + rest):], rank, None, 0.0, pos, f, pairing, mag), take(dev, pages)
    for j, p in enumerate(pos):
        i = 0 if j < counts[0] else 1
        near16(got[table[i][p // P], p % P], rows[j])


def test_append_of_extremes(dev):
    """numbers beyond 16 bits become its largest, infinities and NaN stay, rows of zeros stay zeros"""
    rank, rest, P, H, dim = 16, 16, 16, 1, 16
    src = np.zeros((5, dim + rest + rank + rest), np.float32)
    src[0, :4] = [1e6, -7e4, np.inf, np.nan]
    src[0, dim + rest + rank] = 3e38
    src[1, dim + rest + rank + 1] = -np.inf
    src[2, dim + rest + 3] = np.nan                                          # the whole of c
    src[3, dim + rest:dim + rest + rank] = 1e-30                             # squares that vanish
    src[4, dim + rest:dim + rest + rank] = 1e18
    pages, t = give(dev, np.ones((1, P, rank + rest), np.float16)), give(dev, src)
    q = take(dev, paged.latent_append(paged.PagePlan(dev, P, 1, [[0]], [0], [5]), pages, rank, t, dim + rest, eps=1e-6, q_src=t, n_heads=H, dim=dim))
    got = take(dev, pages)[0]
    np.testing.assert_array_equal(q[0, :4], [65504.0, -65504.0, np.inf, np.nan])
    assert got[0, rank] == 65504.0 and got[1, rank + 1] == -np.inf and np.isnan(got[2, :rank]).all() and (got[2, rank:] == 0).all()
    assert (got[0, :rank] == 0).all() and (got[3, :rank] == 0).all() and (np.abs(got[4, :rank] - 1.0) < 1e-3).all()
    assert (got[5:] == 1.0).all()


def test_append_rows_alone(dev):
    c = Case(dev, 32, 32, 0, [3], [40])
    src = c.rng.normal(size=(40, 32)).astype(np.float32)
    pages = give(dev, c.a)
    assert paged.latent_append(c.plan(), pages, 32, give(dev, src), 0, eps=1e-6) is None
    got = take(dev, pages)
    near16(np.stack([got[c.table[0][p // 32], p % 32] for p in range(3, 43)]), R.row(src, 32, None, 1e-6, np.arange(3, 43), [], 0, 1.0))


# ---- attention ----------------------------------------------------------------------------------------------------------------------------
def bound(want, size, q, rows, uk, rank, H, scale, out_eps):
    """How far a result may be off.  2^-11 is half a step of f16.
    a weight: 2^-11 of itself by its rounding, and its score's error e: the query over the latents (absorbed) or the key (expanded) rounded to f16, 2^-11 of a term at most, in a sum of
    terms q_j k_j whose roundings have no common sign: 4 standard deviations of it, 4 x 2^-11 / sqrt(3) x the root of the sum of (q_j k_j)^2, at most |q| |k|; 32-bit sums of up to 576 terms beside
    it.  A score's error multiplies weights by 1 +- e, in the sum and its divisor: 2 e of sum(w |v|).
    values: 2^-11 of sum(w |v|) in the expanded form.  The result: its own rounding, out_eps of itself."""
    e = abs(scale) * 4 * 2.0 ** -11 / 3 ** 0.5 * q                            # (an error has no sign)
    return out_eps * np.abs(want) + (2 * e + 3 * 2.0 ** -11) * size * 1.1 + 2.0 ** -24


def attend(dev, c, q, uk, uv, H, scale, window, sink, form, out_type=capi.BF16):
    y = paged.latent_attention(c.plan(), give(dev, c.a), c.rank, give(dev, q), H, give(dev, uk), give(dev, uv), scale, window=window, sink=None if sink is None else give(dev, sink),
                               form=form, out_type=out_type)
    assert y.shape() == [sum(c.counts), uv.shape[0]] and y.dtype() == out_type
    return take(dev, y)


def check(dev, c, H, dim, vdim, scale, window=0, sink=None, form=capi.LATENT_AUTO, out_type=capi.BF16, q=None, uk=None, uv=None):
    T, rank, rest, r = sum(c.counts), c.rank, c.rest, c.rng
    uk = (r.normal(size=(H * dim, rank)) * rank ** -0.5).astype(np.float16) if uk is None else uk
    uv = (r.normal(size=(H * vdim, rank)) * rank ** -0.5).astype(np.float16) if uv is None else uv
    q = r.normal(size=(T, H * (dim + rest))).astype(np.float16) if q is None else q
    got = attend(dev, c, q, uk, uv, H, scale, window, sink, form, out_type).reshape(T, H, vdim)
    eps, at = 2.0 ** -8 if out_type == capi.BF16 else 2.0 ** -11, 0
    for i, n in enumerate(c.counts):
        rows, mine = c.rows(i, c.pos0[i] + n), q[at:at + n].reshape(n, H, dim + rest)
        want, size = R.attention(rows, c.pos0[i], mine, uk, uv, rank, H, scale, window, sink)
        with np.errstate(invalid="ignore", over="ignore"):
            k = np.concatenate([np.einsum("jr,hdr->hjd", rows[:, :rank].astype(np.float64), uk.astype(np.float64).reshape(H, dim, rank)),
                                np.broadcast_to(rows[None, :, rank:].astype(np.float64), (H, len(rows), rest))], 2) if n else np.zeros((H, 0, dim + rest))
            far = np.sqrt(np.nansum(k ** 2, 2)).max(1) if n else np.zeros(H)       # of keys that are finite
            # absorbed: terms are those of the query over the latents and the row
            over = np.concatenate([np.einsum("thd,hdr->thr", mine[..., :dim].astype(np.float64), uk.astype(np.float64).reshape(H, dim, rank)), mine[..., dim:].astype(np.float64)], 2)
            terms = np.maximum(np.sqrt((mine.astype(np.float64) ** 2).sum(2)) * far[None],
                               np.sqrt((over ** 2).sum(2)) * np.sqrt(np.nanmax(np.where(np.isfinite(rows), rows.astype(np.float64) ** 2, np.nan), initial=0.0)))
        off = np.abs(got[at:at + n] - want)
        lim = bound(want, size, terms[..., None], rows, uk, rank, H, scale, eps)
        bad = ~((off <= lim) | (np.isnan(got[at:at + n]) & np.isnan(want)))
        assert not bad.any(), (i, np.argwhere(bad)[:5].tolist(), got[at:at + n][bad][:5], want[bad][:5], lim[bad][:5])
        at += n
    return got


SHAPES = [  # heads, dim, rest, vdim, rank
    (16, 128, 64, 128, 512), (3, 32, 16, 32, 64), (1, 16, 0, 16, 16), (5, 48, 16, 80, 160), (8, 64, 32, 64, 256), (24, 32, 48, 16, 80), (33, 16, 16, 32, 48),
]
SEQS = [([0], [1]), ([31], [1]), ([32], [1]), ([200], [1]), ([1000, 3, 0, 64], [1, 1, 1, 1]), ([40, 0, 5], [3, 0, 2]), ([0, 100], [9, 6]), ([70], [17]), ([0], [150])]


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("shape", SHAPES, ids=[str(s) for s in SHAPES])
@pytest.mark.parametrize("pos0,counts", SEQS, ids=[str(i) for i in range(len(SEQS))])
def test_attention(dev, form, shape, pos0, counts):
    H, dim, rest, vdim, rank = shape
    c = Case(dev, 16, rank, rest, pos0, counts, seed=H)
    check(dev, c, H, dim, vdim, 1.5 * (dim + rest) ** -0.5, form=FORMS[form])


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("out_type", [capi.F16, capi.BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("window,sink", [(0, False), (1, False), (2, True), (33, False), (100, True), (1000, True)])
@pytest.mark.parametrize("P", [16, 32, 128])
def test_masks(dev, form, P, window, sink, out_type):
    c = Case(dev, P, 64, 16, [300, 0, 64], [7, 1, 33], seed=window)
    check(dev, c, 6, 32, 32, 0.2, window=window, sink=c.rng.normal(size=6).astype(np.float32) if sink else None, form=FORMS[form], out_type=out_type)


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("P,window", [(16, 0), (128, 0), (64, 200)])
@pytest.mark.parametrize("shape", [(2, 128, 64, 128, 512), (3, 32, 16, 32, 64), (2, 80, 32, 112, 96)], ids=str)
def test_prompts(dev, form, P, window, shape):
    """portions of many tokens: several tiles of rows and of keys, beside sequences of one token and of none"""
    H, dim, rest, vdim, rank = shape
    c = Case(dev, P, rank, rest, [0, 333, 70, 9, 1000], [513, 256, 0, 1, 129], seed=P)
    check(dev, c, H, dim, vdim, 1.2 * (dim + rest) ** -0.5, window=window, form=FORMS[form])


def test_both_forms_in_a_call(dev):
    """a step of portions and single tokens, by the rule"""
    c = Case(dev, 32, 64, 16, [100, 7, 0, 40, 300, 5], [1, 300, 64, 65, 1, 200], seed=4)
    check(dev, c, 4, 32, 48, 0.2)


@pytest.mark.parametrize("form", list(FORMS))
def test_sinks_far_away(dev, form):
    """sinks that take all of the weight, none of it, and -inf"""
    c = Case(dev, 16, 32, 16, [50], [3])
    check(dev, c, 4, 16, 16, 0.3, sink=np.array([-np.inf, 80.0, -80.0, 1e30], np.float32), form=FORMS[form])


@pytest.mark.parametrize("form", list(FORMS))
def test_rows_that_are_not_finite(dev, form):
    """they reach the queries that see them and no others: later tokens of the call, windows that have left them, other sequences"""
    for window in (0, 12):
        c = Case(dev, 16, 32, 16, [40, 40, 90], [20, 20, 40], seed=window)
        for i, (at, col, x) in enumerate([(50, 3, np.nan), (45, 35, np.inf), (100, 0, -np.inf)]):
            row = c.rows(i, c.pos0[i] + c.counts[i])[at].copy()
            row[col] = x
            c.put(i, at, row[None])
        H, dim, vdim = 3, 32, 32
        q = np.abs(c.rng.normal(size=(80, H * (dim + 16)))).astype(np.float16)
        uk, uv = (np.abs(c.rng.normal(size=(H * d, 32)) * 0.2).astype(np.float16) for d in (dim, vdim))
        got = attend(dev, c, q, uk, uv, H, 0.2, window, None, FORMS[form]).reshape(80, H, vdim)
        at = 0
        for i, n in enumerate(c.counts):
            want, size = R.attention(c.rows(i, c.pos0[i] + n), c.pos0[i], q[at:at + n].reshape(n, H, -1), uk, uv, 32, H, 0.2, window)
            clean = ~np.isnan(want)
            assert np.isfinite(got[at:at + n][clean]).all()
            np.testing.assert_allclose(got[at:at + n][clean], want[clean], rtol=0.03, atol=0.03)
            # a weight of exactly 0 may drop it: a score of -inf
            lost = ~np.isfinite(got[at:at + n][~clean])
            assert lost.all() or (i > 0 and x == -np.inf)
            at += n


@pytest.mark.parametrize("form", list(FORMS))
def test_queries_that_are_not_finite(dev, form):
    c = Case(dev, 16, 32, 16, [40], [20])
    H, dim = 3, 32
    q = c.rng.normal(size=(20, H * (dim + 16))).astype(np.float16)
    q[3, 5], q[4, dim + 16 + dim + 3], q[19, 2 * (dim + 16)] = np.nan, np.inf, -np.inf
    check(dev, c, H, dim, 32, 0.2, form=FORMS[form], q=q)


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("scale", [0.0, -0.3, 30.0, 3000.0])
def test_scores_of_any_size(dev, form, scale):
    """a score of thousands: one key has all of the weight.  Scores whose difference is far above their errors: the queries pick keys out by their rotated part alone"""
    c = Case(dev, 16, 32, 16, [30], [2], seed=3)
    for j in range(32):                                                      # row j: latents of its own, and the j-th of 32 directions, as +-1 and powers of two
        row = c.rows(0, 32)[j].copy()
        row[32:] = [(1.0 if j >> (b % 5) & 1 else -1.0) * (1.0 + 0.25 * (b // 5)) for b in range(16)]
        c.put(0, j, row[None])
    H, dim, vdim = 2, 16, 32
    q = np.zeros((2, H, dim + 16), np.float16)
    q[..., dim:] = 2.0 * c.rows(0, 32)[13, 32:]
    check(dev, c, H, dim, vdim, scale, form=FORMS[form], q=q.reshape(2, -1))


@pytest.mark.parametrize("form", list(FORMS))
def test_large_and_small_numbers(dev, form):
    """queries and latents near the ends of 16 bits"""
    for big, small in ((60000.0, 1.0 / 60000.0), (1.0 / 4096.0, 4096.0), (1.0, 1.0)):
        c = Case(dev, 16, 32, 16, [60], [3], seed=5)
        q = np.clip(c.rng.normal(size=(3, 2 * 32)) * big / 4, -65504, 65504).astype(np.float16)
        check(dev, c, 2, 16, 32, 0.2 * small * 4, form=FORMS[form], q=q)


def test_strided_and_reused(dev):
    """the same plan for two layers, a call after another, and equal calls give equal bits"""
    c = Case(dev, 32, 64, 16, [500, 90, 2000], [1, 4, 1], seed=9)
    H, dim, vdim = 16, 32, 32
    q, uk, uv = (give(dev, (c.rng.normal(size=s) * k).astype(np.float16)) for s, k in (((6, H * (dim + 16)), 1.0), ((H * dim, 64), 0.125), ((H * vdim, 64), 0.125)))
    plan, pages = c.plan(), give(dev, c.a)
    for form in FORMS.values():
        first = [take(dev, paged.latent_attention(plan, pages, 64, q, H, uk, uv, 0.2, form=form)) for _ in range(3)]
        assert all(np.array_equal(first[0], y) for y in first[1:])


def test_shared_prefix(dev):
    """two sequences over the same pages of a prefix"""
    P, rank, rest, H = 16, 32, 16, 4
    r = np.random.default_rng(1)
    a = r.normal(size=(8, P, rank + rest)).astype(np.float16)
    table, pos0, counts = [[3, 5, 0], [3, 5, 1]], [40, 37], [1, 3]
    q, uk, uv = ((r.normal(size=s) * k).astype(np.float16) for s, k in (((4, H * 32), 1.0), ((H * 16, rank), 0.2), ((H * 16, rank), 0.2)))
    for form in FORMS.values():
        y = take(dev, paged.latent_attention(paged.PagePlan(dev, P, 8, table, pos0, counts), give(dev, a), rank, give(dev, q), H, give(dev, uk), give(dev, uv), 0.2, form=form))
        at = 0
        for i, n in enumerate(counts):
            rows = np.concatenate([a[p] for p in table[i]])[:pos0[i] + n]
            want, _ = R.attention(rows, pos0[i], q[at:at + n].reshape(n, H, 32), uk, uv, rank, H, 0.2)
            np.testing.assert_allclose(y[at:at + n].reshape(want.shape), want, rtol=0.02, atol=0.01)
            at += n


def test_nothing(dev):
    c = Case(dev, 16, 32, 16, [5, 9], [0, 0])
    y = paged.latent_attention(c.plan(), give(dev, c.a), 32, CudaTensor.alloc([0, 64], capi.F16, dev), 2, give(dev, np.ones((32, 32), np.float16)), give(dev, np.ones((64, 32), np.float16)), 1.0)
    assert y.shape() == [0, 64]
    assert paged.latent_append(c.plan(), give(dev, c.a), 32, CudaTensor.alloc([0, 48], capi.F32, dev), 0, q_src=CudaTensor.alloc([0, 64], capi.F32, dev), n_heads=2, dim=16).shape() == [0, 64]


@pytest.mark.parametrize("dim,vdim,rest,rank", [(256, 16, 64, 512), (16, 256, 0, 512), (144, 208, 48, 496)])
def test_wide_heads(dev, dim, vdim, rest, rank):
    """heads that are not expanded"""
    c = Case(dev, 64, rank, rest, [100, 31], [70, 1], seed=7)
    check(dev, c, 3, dim, vdim, 1.2 * (dim + rest) ** -0.5)
    with pytest.raises(TensorError):
        check(dev, c, 3, dim, vdim, 0.1, form=capi.LATENT_EXPANDED)


def test_tokens_by_portions(dev):
    """absorbed: more tokens than the workspace holds queries of, one sequence across two portions, beside one that takes the other form in between"""
    rank, rest, dim, vdim, H = 512, 64, 16, 16, 128
    each = (256 << 20) // (H * (2 * rank + rest) * 4) // 32 * 32
    counts = [each - 40, 1, 90]
    c = Case(dev, 128, rank, rest, [0, 50, 7], counts, seed=2)
    T = sum(counts)
    q, uk, uv = ((c.rng.normal(size=s) * k).astype(np.float16) for s, k in (((T, H * (dim + rest)), 1.0), ((H * dim, rank), 0.05), ((H * vdim, rank), 0.05)))
    y = attend(dev, c, q, uk, uv, H, 0.1, 0, None, capi.LATENT_ABSORBED).reshape(T, H, vdim)
    at = 0
    for i, n in enumerate(counts):
        pick = sorted({0, n // 2, n - 1, *range(max(0, n - 60), n, 7), *range(0, min(n, 60), 9)})
        for t in pick:
            rows = c.rows(i, c.pos0[i] + t + 1)
            want, _ = R.attention(rows, c.pos0[i] + t, q[at + t].reshape(1, H, -1), uk, uv, rank, H, 0.1)
            np.testing.assert_allclose(y[at + t], want[0], rtol=0.02, atol=0.01)
        at += n


def test_far_pages(dev):
    """pages whose numbers lie beyond 2^31 elements, in both forms and the append"""
    P, rank, rest, H, dim, vdim = 128, 512, 64, 4, 32, 32
    n_pages = (1 << 31) // (P * (rank + rest)) + 40
    if torch.cuda.mem_get_info()[0] < 3 * n_pages * P * (rank + rest):
        pytest.skip("no room")
    pages = CudaTensor.alloc([n_pages, P, rank + rest], capi.F16, dev)
    r = np.random.default_rng(0)
    table, pos0, counts = [[n_pages - 1, 3, n_pages - 7], [n_pages - 20]], [300, 0], [3, 100]
    rows = [r.normal(size=(p + n, rank + rest)).astype(np.float16) for p, n in zip(pos0, counts)]
    t = view(pages)
    dev.synchronize()
    for i, x in enumerate(rows):
        for b, page in enumerate(table[i]):
            part = torch.from_numpy(x[b * P:(b + 1) * P]).cuda()
            t[page, :len(part)] = part
    T = sum(counts)
    plan = paged.PagePlan(dev, P, n_pages, table, pos0, counts)
    src = r.normal(size=(T, rank + rest)).astype(np.float32)
    torch.cuda.synchronize()
    paged.latent_append(plan, pages, rank, give(dev, src), 0, eps=1e-6)
    dev.synchronize()
    new, at = R.f16(R.row(src, rank, None, 1e-6, np.zeros(T), [], 0, 1.0)), 0
    for i, n in enumerate(counts):
        got = np.concatenate([t[page].cpu().numpy() for page in table[i]])[pos0[i]:pos0[i] + n]
        near16(got, new[at:at + n].astype(np.float64), 2.0)
        rows[i][pos0[i]:] = got
        at += n
    q, uk, uv = ((r.normal(size=s) * k).astype(np.float16) for s, k in (((T, H * (dim + rest)), 1.0), ((H * dim, rank), 0.05), ((H * vdim, rank), 0.05)))
    for form in FORMS.values():
        y = take(dev, paged.latent_attention(plan, pages, rank, give(dev, q), H, give(dev, uk), give(dev, uv), 0.1, form=form)).reshape(T, H, vdim)
        at = 0
        for i, n in enumerate(counts):
            want, _ = R.attention(rows[i], pos0[i], q[at:at + n].reshape(n, H, -1), uk, uv, rank, H, 0.1)
            np.testing.assert_allclose(y[at:at + n], want, rtol=0.02, atol=0.01)
            at += n


@pytest.mark.parametrize("n", [1, 2, 150, 700])
def test_many_sequences(dev, n):
    """as many sequences as take several looks to find, most of them short; tokens of both forms by turns, more runs of them than a call lists"""
    r = np.random.default_rng(n)
    counts = [int(x) for x in r.choice([0, 1, 1, 2, 70], size=n)]
    c = Case(dev, 16, 32, 16, [int(x) for x in r.integers(0, 60, size=n)], counts, seed=n)
    check(dev, c, 3, 16, 16, 0.25)


@pytest.mark.parametrize("limit", [1, 3])
def test_few_sms(limit):
    """a device that is held to a few SMs: the same attention"""
    d = make_device()
    d.set_sm_limit(limit)
    c = Case(d, 32, 64, 16, [900, 3, 2100], [1, 60, 4], seed=limit)
    for form in (capi.LATENT_AUTO, capi.LATENT_EXPANDED):
        check(d, c, 8, 32, 32, 0.2, form=form)
    d.close()


def test_two_devices_at_once(dev):
    """two handles with streams of their own, calls by turns from two threads"""
    import threading
    other = make_device()
    wrong = []

    def work(d, seed):
        try:
            for k in range(3):
                c = Case(d, 32, 64, 32, [200, 5, 1000], [1, 80, 1], seed=seed + k)
                check(d, c, 8, 32, 32, 0.15)
        except Exception as e:                                               # told by the thread that started this one
            wrong.append(e)
    threads = [threading.Thread(target=work, args=(d, i)) for i, d in enumerate((dev, other))]
    [t.start() for t in threads]
    [t.join() for t in threads]
    other.close()
    assert not wrong, wrong


def test_refusals(dev):
    P, rank, rest, H, dim, vdim = 16, 32, 16, 2, 16, 16
    c = Case(dev, P, rank, rest, [5], [3])
    plan, pages = c.plan(), give(dev, c.a)
    z = lambda *s, t=np.float16: give(dev, np.zeros(s, t))  # noqa: E731
    q, uk, uv, src = z(3, H * (dim + rest)), z(H * dim, rank), z(H * vdim, rank), z(3, 100, t=np.float32)
    other = make_device()
    attention = lambda **k: paged.latent_attention(**{**dict(plan=plan, pages=pages, rank=rank, q=q, n_heads=H, uk=uk, uv=uv, scale=1.0), **k})  # noqa: E731
    append = lambda **k: paged.latent_append(**{**dict(plan=plan, pages=pages, rank=rank, kv_src=src, kv_col0=0, q_src=src, q_col0=36, n_heads=2, dim=16), **k})  # noqa: E731
    attention(), append()
    for f in (attention, append):
        for bad in (dict(rank=33), dict(rank=0), dict(rank=-16), dict(rank=48 + 16), dict(pages=z(c.n_pages, P, rank + rest, t=np.float32)), dict(pages=z(c.n_pages - 1, P, rank + rest)),
                    dict(pages=z(c.n_pages, 2 * P, rank + rest)), dict(pages=z(c.n_pages * P, rank + rest)), dict(n_heads=0), dict(n_heads=8193), dict(rank=2 ** 40), dict(n_heads="2"),
                    dict(pages=z(c.n_pages, P, 40), rank=32), dict(pages=z(c.n_pages, P, 640), rank=512), dict(pages=z(c.n_pages, P, 544), rank=528)):
            with pytest.raises(TensorError):
                f(**bad)
    for bad in (dict(q=z(2, H * (dim + rest))), dict(q=z(3, H * (dim + rest) + 1)), dict(q=z(3, H * (dim + rest), t=np.float32)), dict(n_heads=3), dict(uk=z(H * dim, rank + 1)), dict(uk=z(H * dim + 1, rank)),
                dict(uk=z(H * 8, rank)), dict(uv=z(H * 272, rank)), dict(uv=z(H * vdim, rank, t=np.float32)), dict(sink=z(H + 1, t=np.float32)), dict(sink=z(H)), dict(form=3), dict(form=-1), dict(out_type=capi.F32),
                dict(q=q.with_strider(TensorStrider([3, H * (dim + rest)], [1, 3]))), dict(window=2 ** 31), dict(uk=give(other, np.zeros((H * dim, rank), np.float16)))):
        with pytest.raises(TensorError):
            attention(**bad)
    for bad in (dict(kv_src=z(2, 100, t=np.float32)), dict(kv_col0=-1), dict(kv_col0=53), dict(q_col0=37), dict(q_col0=-1), dict(dim=8), dict(dim=272), dict(pairing=2), dict(norm_w=z(rank)), dict(norm_w=z(rank + 1, t=np.float32)),
                dict(freq=z(9, t=np.float32)), dict(freq=z(4)), dict(kv_src=src.with_strider(TensorStrider([3, 100], [99, 1]))), dict(kv_src=src.with_strider(TensorStrider([3, 100], [101, 1]))),
                dict(kv_src=pages.reshape([c.n_pages * P, rank + rest])), dict(q_src=z(4, 100, t=np.float32)), dict(kv_src=give(other, np.zeros((3, 100), np.float32)))):
        with pytest.raises(TensorError):
            append(**bad)
    with pytest.raises(TensorError):
        attention(pages=give(other, c.a))
    with pytest.raises(TensorError):
        attention(plan=paged.PagePlan(other, P, c.n_pages, c.table, c.pos0, c.counts))
    lazy = make_device(lazy=True)
    with pytest.raises((TensorError, CudaError)):
        paged.PagePlan(lazy, P, c.n_pages, c.table, c.pos0, c.counts)
    lazy.close()
    other.close()
    attention(), append()


def test_a_layer(dev):
    """what a program does in a step: products with their epilogue, the append, the attention and the product back into the residual stream; a prompt in portions and then single tokens for
    two sequences, beside each whole sequence in 64 bits"""
    from crabml_b200 import seqops
    P, width, H, dim, rest, vdim, rank = 32, 192, 4, 32, 16, 32, 64
    r = np.random.default_rng(11)
    cols = H * (dim + rest) + rank + rest
    w = {n: (r.normal(size=s) * s[1] ** -0.5).astype(np.float16) for n, s in (("in", (cols, width)), ("uk", (H * dim, rank)), ("uv", (H * vdim, rank)), ("out", (width, H * vdim)))}
    bias, norm, f = (0.3 * r.normal(size=cols)).astype(np.float32), (1.0 + 0.2 * r.normal(size=rank)).astype(np.float32), freqs(rest // 2)
    d = {n: give(dev, x) for n, x in w.items()}
    db, dn, df = give(dev, bias), give(dev, norm), give(dev, f)
    scale, steps = (dim + rest) ** -0.5, [(70, 3), (1, 90), (65, 0), (1, 1), (1, 1), (0, 4)]
    x = [r.normal(size=(sum(s[i] for s in steps), width)).astype(np.float32) for i in range(2)]
    table = [[4, 1, 6, 9, 2], [0, 8, 3, 5]]
    pages, have, got = give(dev, np.full((10, P, rank + rest), np.nan, np.float16)), [0, 0], [[], []]
    for step in steps:
        plan = paged.PagePlan(dev, P, 10, table, have, step)
        h = give(dev, np.concatenate([x[i][have[i]:have[i] + n] for i, n in enumerate(step)]))
        qkv = seqops.product(d["in"], h, bias=db, out_type=capi.F16)
        q = paged.latent_append(plan, pages, rank, qkv, H * (dim + rest), norm_w=dn, eps=1e-5, q_src=qkv, n_heads=H, dim=dim, freq=df)
        y = paged.latent_attention(plan, pages, rank, q, H, d["uk"], d["uv"], scale, out_type=capi.F16)
        o = take(dev, seqops.product(d["out"], y, residual=h, out_type=capi.F32))
        at = 0
        for i, n in enumerate(step):
            got[i].append(o[at:at + n])
            have[i] += n
            at += n
    for i in range(2):
        n = have[i]
        qkv = x[i].astype(np.float16).astype(np.float64) @ w["in"].astype(np.float64).T + bias
        q = qkv[:, :H * (dim + rest)].reshape(n, H, -1).copy()
        q[..., dim:] = R.turn(q[..., dim:], np.arange(n), f, 0, 1.0)
        rows = R.row(qkv[:, H * (dim + rest):], rank, norm, 1e-5, np.arange(n), f, 0, 1.0)
        y, _ = R.attention(rows, 0, q, w["uk"], w["uv"], rank, H, scale)
        want = x[i] + y.reshape(n, -1) @ w["out"].astype(np.float64).T
        # five roundings to 16 bits, 2^-11 of numbers of size 1 each, and a sum of 128 of them with weights of 128^-1/2
        assert np.abs(np.concatenate(got[i]) - want).max() < 5 * 2.0 ** -11 * 6


@pytest.mark.parametrize("pos0,counts,window,sink", [([9000], [70], 0, False), ([4000, 0, 2500], [300, 65, 130], 0, True), ([6000, 100], [513, 70], 1500, True), ([2000, 0], [129, 90], 0, False)])
def test_cut_items(dev, pos0, counts, window, sink):
    """expanded: few rows over long caches, whose keys several CTAs share; beside sequences that one takes as a whole, and pieces that see nothing"""
    c = Case(dev, 64, 64, 16, pos0, counts, seed=5)
    check(dev, c, 2, 32, 48, 0.2, window=window, sink=c.rng.normal(size=2).astype(np.float32) if sink else None, form=capi.LATENT_EXPANDED)


def test_cut_items_not_finite(dev):
    """expanded, cut: a row of the cache that is not finite reaches those who see it and no others, whichever piece it lies in"""
    pos0, n = 5000, 200
    for bad in (10, 3000, pos0 + 110, pos0 + 119, pos0 + 150):      # also a row's last keys, with steps behind them that it does not see
        c = Case(dev, 64, 64, 16, [pos0], [n], seed=bad)
        q, uk, uv = ((c.rng.normal(size=s) * k).astype(np.float16) for s, k in (((n, 2 * 48), 1.0), ((64, 64), 0.1), ((64, 64), 0.1)))
        clean = attend(dev, c, q, uk, uv, 2, 0.2, 0, None, capi.LATENT_EXPANDED).reshape(n, 2, 32)
        c.a[c.table[0][bad // 64], bad % 64, 3] = np.nan
        got = attend(dev, c, q, uk, uv, 2, 0.2, 0, None, capi.LATENT_EXPANDED).reshape(n, 2, 32)
        sees = max(0, bad - pos0)
        assert np.isnan(got[sees:]).all() and np.array_equal(got[:sees], clean[:sees])


@pytest.mark.parametrize("dim,vdim,rest,rank", [(16, 16, 0, 16), (64, 64, 64, 64), (128, 64, 64, 128), (128, 128, 64, 512)])
def test_equal_calls_of_many_steps(dev, dim, vdim, rest, rank):
    """expanded: heads of which shared memory holds several steps, and those of which it holds one; whole items and pieces: equal calls give equal bits"""
    for pos0, n in ((1200, 300), (7000, 130)):
        c = Case(dev, 128, rank, rest, [pos0], [n], seed=3)
        a = [give(dev, (c.rng.normal(size=s) * k).astype(np.float16)) for s, k in (((n, 4 * (dim + rest)), 1.0), ((4 * dim, rank), rank ** -0.5), ((4 * vdim, rank), rank ** -0.5))]
        plan, pages, first = c.plan(), give(dev, c.a), None
        for _ in range(60):
            y = take(dev, paged.latent_attention(plan, pages, rank, a[0], 4, a[1], a[2], 0.1, form=capi.LATENT_EXPANDED))
            first = y if first is None else first
            assert np.array_equal(y, first) and np.isfinite(y).all()


@pytest.mark.parametrize("rank,rest", [(512, 64), (512, 16), (384, 48), (256, 64)])
def test_equal_calls_of_long_rings(dev, rank, rest):
    """absorbed: rows of which the ring holds an odd number of steps (nine blocks of 64 columns 5, seven 7), and an even one: equal calls give equal bits, with all SMs asking at once"""
    H, dim, vdim = 16, 32, 32
    r = np.random.default_rng(rank + rest)
    pos0 = [int(x) for x in r.integers(20, 1500, size=64)]
    c = Case(dev, 32, rank, rest, pos0, [1] * 64, seed=rest)
    q, uk, uv = ((c.rng.normal(size=s) * k).astype(np.float16) for s, k in (((64, H * (dim + rest)), 1.0), ((H * dim, rank), rank ** -0.5), ((H * vdim, rank), rank ** -0.5)))
    plan, pages, t, first = c.plan(), give(dev, c.a), [give(dev, x) for x in (q, uk, uv)], None
    for _ in range(100):
        y = take(dev, paged.latent_attention(plan, pages, rank, t[0], H, t[1], t[2], 0.15, form=capi.LATENT_ABSORBED))
        first = y if first is None else first
        assert np.array_equal(y, first)
    check(dev, c, H, dim, vdim, 0.15, form=capi.LATENT_ABSORBED, q=q, uk=uk, uv=uv)


@pytest.mark.parametrize("dim,vdim,rest,rank", [(16, 16, 0, 16), (128, 128, 64, 128)])
def test_equal_calls_of_one_step(dev, dim, vdim, rest, rank):
    """expanded: items of a single step of 128 keys, in which each row's base moves and its sum follows at once, and of two: equal calls give equal bits"""
    H = 8
    c = Case(dev, 32, rank, rest, [0, 0, 3, 100, 0, 90], [128, 1, 125, 28, 77, 60], seed=rank)
    q, uk, uv = ((c.rng.normal(size=s) * k).astype(np.float16) for s, k in (((sum(c.counts), H * (dim + rest)), 1.0), ((H * dim, rank), rank ** -0.5), ((H * vdim, rank), rank ** -0.5)))
    plan, pages, t, first = c.plan(), give(dev, c.a), [give(dev, x) for x in (q, uk, uv)], None
    for _ in range(200):
        y = take(dev, paged.latent_attention(plan, pages, rank, t[0], H, t[1], t[2], 0.2, form=capi.LATENT_EXPANDED))
        first = y if first is None else first
        assert np.array_equal(y, first)
    check(dev, c, H, dim, vdim, 0.2, form=capi.LATENT_EXPANDED, q=q, uk=uk, uv=uv)


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("with_sink", [False, True])
@pytest.mark.parametrize("pos0,counts", [([40], [20]), ([5000], [70]), ([0, 3000, 7], [1, 130, 3])])
def test_scores_of_minus_infinity(dev, form, with_sink, pos0, counts):
    """a query with an infinity that makes all of its scores -infinity has the result NaN, beside a sink too, whole or cut into pieces; a query that is finite sees such a key with the weight 0: beside a
    sink 0 where there is no other key, and NaN without one"""
    H, dim, vdim, rank, rest = 3, 32, 32, 64, 16
    c = Case(dev, 64, rank, rest, pos0, counts, seed=sum(pos0))
    for i, n in enumerate(counts):
        rows = c.rows(i, pos0[i] + n)
        rows[:, rank] = -np.abs(rows[:, rank]) - np.float16(0.5)
        c.put(i, 0, rows)
    T = sum(counts)
    q = c.rng.normal(size=(T, H, dim + rest)).astype(np.float16)
    q[-1, 1, dim] = np.inf
    if T > 2:
        q[T - 3, 0, dim], q[T - 2, 2, dim] = np.inf, np.inf
    sink = np.array([0.5, -1.0, 2.0], np.float32) if with_sink else None
    check(dev, c, H, dim, vdim, 0.2, sink=sink, form=FORMS[form], q=q.reshape(T, -1))
    # now keys: every row's r is -infinity in a column that queries weigh by a positive number
    for i, n in enumerate(counts):
        rows = c.rows(i, pos0[i] + n)
        rows[:, rank] = -np.inf
        c.put(i, 0, rows)
    q = np.abs(q) + np.float16(0.25)
    q[~np.isfinite(q)] = 1.0
    uk, uv = ((c.rng.normal(size=s) * rank ** -0.5).astype(np.float16) for s in ((H * dim, rank), (H * vdim, rank)))
    got = attend(dev, c, q.reshape(T, -1), uk, uv, H, 0.2, 0, sink, FORMS[form])
    assert (got == 0).all() if with_sink else np.isnan(got).all()


@pytest.mark.parametrize("with_sink", [False, True])
@pytest.mark.parametrize("pos0,counts,P", [([0], [3], 16), ([20, 0], [4, 2], 32), ([5000], [3], 64), ([700, 40], [2, 6], 16)])
def test_large_scores_beside_rows_that_are_not_finite(dev, pos0, counts, P, with_sink):
    """rows whose neighbours in a tile see a NaN, which they do not: where all their keys have one and the same latent row, the result is its value whatever the scores, here in the hundreds and thousands"""
    H, dim, vdim, rank, rest = 5, 64, 32, 128, 32
    c = Case(dev, P, rank, rest, pos0, counts, seed=P)
    uk, uv = ((c.rng.normal(size=s) * k).astype(np.float16) for s, k in (((H * dim, rank), 0.5), ((H * vdim, rank), rank ** -0.5)))
    T, at = sum(counts), 0
    q = (8.0 * c.rng.normal(size=(T, H, dim + rest))).astype(np.float16)
    sink = np.full(H, -1e30, np.float32) if with_sink else None
    same = []
    for i, n in enumerate(counts):
        row = c.rng.normal(size=rank + rest).astype(np.float16)
        c.put(i, 0, np.tile(row, (pos0[i] + n, 1)))
        c.put(i, pos0[i] + n - 1, np.full((1, rank + rest), np.nan, np.float16))
        same.append(uv.astype(np.float64).reshape(H, vdim, rank) @ row[:rank].astype(np.float64))
    got = attend(dev, c, q.reshape(T, -1), uk, uv, H, 1.0, 0, sink, capi.LATENT_ABSORBED, capi.F16).reshape(T, H, vdim)
    for i, n in enumerate(counts):
        assert np.isnan(got[at + n - 1]).all()
        # the same weights over and under the line: their roundings to f16, 2^-11 each where one has all of the weight, the result's own, and what is left of latents in two f16 numbers
        size = np.abs(uv.astype(np.float64)).reshape(H, vdim, rank).sum(2) * 4
        assert (np.abs(got[at:at + n - 1] - same[i]) <= 2.0 ** -11 * np.abs(same[i]) * 2 + 2.0 ** -20 * size).all()
        at += n


@pytest.mark.parametrize("rank,size", [(512, 1e-5), (512, 1.0), (80, 3e-6), (256, 60000.0)])
@pytest.mark.parametrize("pos0,counts", [([6], [1]), ([3000], [2]), ([20, 0, 90], [1, 3, 2])])
def test_small_latents_keep_their_bits(dev, rank, size, pos0, counts):
    """absorbed: latents whose mean lies where f16 has steps of a hundredth of it, and large ones; queries of zeros, so that all weights are one number and nothing else is rounded"""
    H, dim, vdim = 3, 16, 48
    c = Case(dev, 32, rank, 16, pos0, counts, seed=rank)
    for i, n in enumerate(counts):
        rows = c.rng.normal(size=(pos0[i] + n, rank + 16)) * min(size, 15000.0)
        c.put(i, 0, np.clip(rows, -65504, 65504).astype(np.float16))
    T, at = sum(counts), 0
    uk, uv = c.rng.normal(size=(H * dim, rank)).astype(np.float16), (c.rng.normal(size=(H * vdim, rank)) * rank ** -0.5 * min(200.0 / size ** 0.5, 200.0, 10.0 / size)).astype(np.float16)
    got = attend(dev, c, np.zeros((T, H * (dim + 16)), np.float16), uk, uv, H, 0.1, 0, None, capi.LATENT_ABSORBED, capi.F16).reshape(T, H, vdim)
    V = uv.astype(np.float64).reshape(H, vdim, rank)
    for i, n in enumerate(counts):
        rows = c.rows(i, pos0[i] + n)[:, :rank].astype(np.float64)
        for t in range(n):
            lat = rows[:pos0[i] + t + 1].mean(0)
            want, terms = V @ lat, np.abs(V) @ np.abs(rows[:pos0[i] + t + 1]).mean(0)
            # the result's rounding; sums over up to 3000 keys and 512 columns in 32 bits, of which the tensor cores cut off 2^-23 of the sum after every 16 terms
            lim = 2.0 ** -11 * np.abs(want) + (len(rows) / 16 + rank / 16 + 8) * 2.0 ** -23 * terms + 2.0 ** -25
            assert (np.abs(got[at + t] - want) <= lim).all(), float((np.abs(got[at + t] - want) / lim).max())
        at += n


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("pos0,n", [(120, 1), (3000, 30), (9000, 70)])
def test_a_flat_tail(dev, form, pos0, n):
    """one key stands out, thousands lie 15 below it: their weights count together, and each keeps the bits of a 16-bit number"""
    H, dim, vdim, rank, rest = 2, 16, 32, 16, 16
    c = Case(dev, 64, rank, rest, [pos0], [n])
    rows = np.zeros((pos0 + n, rank + rest), np.float16)
    rows[:, 0], rows[:, rank] = 1.0, -15.0
    rows[7, 0], rows[7, rank] = 0.0, 0.0
    c.put(0, 0, rows)
    q = np.zeros((n, H, dim + rest), np.float16)
    q[..., dim] = 1.0
    uk, uv = np.zeros((H * dim, rank), np.float16), np.ones((H * vdim, rank), np.float16)
    got = attend(dev, c, q.reshape(n, -1), uk, uv, H, 1.0, 0, None, FORMS[form], capi.F16)
    tail = (np.arange(pos0, pos0 + n)) * np.exp(-15.0)
    # a weight is 2^7 e^-15 = 2^-14.6 or more, where f16 has steps of 2^-24: half of one is 2^-10.4 of it; the result's rounding 2^-11 of itself, or half of a step of 2^-24
    assert (np.abs(got - (tail / (1 + tail))[:, None]) <= (2.0 ** -10.4 + 2.0 ** -11) * (tail / (1 + tail))[:, None] + 2.0 ** -25).all()


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("scale", [2.0 ** -12, 1e-3, 0.01, 0.037, 0.1, 0.61, 1.0, -0.05])
@pytest.mark.parametrize("pos0,n", [(0, 100), (700, 40), (6000, 33)])
def test_scores_of_millions(dev, form, scale, pos0, n):
    """scores up to 2^30 and beyond, growing from key to key by a little or a lot: all keys have one value, so that is the result, and no weight leaves its type"""
    H, dim, vdim, rank, rest = 3, 16, 32, 32, 16
    c = Case(dev, 32, rank, rest, [pos0], [n], seed=n)
    rows = np.tile(c.rng.normal(size=rank + rest), (pos0 + n, 1))
    j = np.arange(pos0 + n)
    rows[:, rank] = 30000.0 + 16.0 * (j % 700)
    rows[:, rank + 1] = c.rng.integers(-3, 4, size=pos0 + n)
    c.put(0, 0, rows.astype(np.float16))
    q = c.rng.normal(size=(n, H, dim + rest))
    q[:, 0, dim], q[:, 1, dim], q[:, 2, dim] = 2000.0, 30000.0, 100.0
    uk, uv = ((c.rng.normal(size=s) * 0.2).astype(np.float16) for s in ((H * dim, rank), (H * vdim, rank)))
    got = attend(dev, c, q.astype(np.float16).reshape(n, -1), uk, uv, H, scale, 0, None, FORMS[form], capi.F16).reshape(n, H, vdim)
    V, lat = uv.astype(np.float64).reshape(H, vdim, rank), rows[0, :rank].astype(np.float16).astype(np.float64)
    # roundings of the weights (over the line, not under it), of the expanded values and of the result, 2^-11 each, beside 32-bit sums
    lim = 3 * 2.0 ** -11 * np.abs(V @ lat) + 2.0 ** -17 * (np.abs(V) @ np.abs(lat)) + 2.0 ** -24
    assert (np.abs(got - V @ lat) <= lim).all()


def whole(c, i, q, uk, uv, H, scale, window, sink, leave_out=None):
    """one sequence's results in 64 bits, all tokens at a time; leave_out: keys that are lost"""
    n, rank, rest = c.counts[i], c.rank, c.rest
    rows = c.rows(i, c.pos0[i] + n).astype(np.float64)
    dim, vdim = uk.shape[0] // H, uv.shape[0] // H
    pos, keys = c.pos0[i] + np.arange(n)[:, None], np.arange(len(rows))[None]
    seen = (keys <= pos) & ((pos - keys < window) if window > 0 else True)
    if leave_out is not None:
        seen[:, leave_out] = False
    out = np.zeros((n, H, vdim))
    for h in range(H):
        k = np.concatenate([rows[:, :rank] @ uk[h * dim:(h + 1) * dim].astype(np.float64).T, rows[:, rank:]], 1)
        z = np.where(seen, scale * (q[:, h].astype(np.float64) @ k.T), -np.inf)
        top = np.maximum(z.max(1, keepdims=True), -np.inf if sink is None else float(sink[h]))
        w = np.exp(z - top)
        w /= w.sum(1, keepdims=True) + (0.0 if sink is None else np.exp(float(sink[h]) - top))
        out[:, h] = w @ (rows[:, :rank] @ uv[h * vdim:(h + 1) * vdim].astype(np.float64).T)
    return out


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("out_type", [capi.F16, capi.BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("shape", [(2, 32, 16, 48, 64), (16, 128, 64, 128, 512), (64, 64, 32, 64, 128)], ids=str)
@pytest.mark.parametrize("P,pos0,counts,window,sink", [(64, [5000], [10], 0, False), (16, [1000, 0, 300], [1, 200, 3], 0, True), (32, [2500, 40], [130, 2], 700, False), (128, [3000, 700, 31], [1, 1, 1], 0, False)])
def test_results_as_a_whole(dev, form, out_type, shape, P, pos0, counts, window, sink):
    """the root mean square of a whole result's error: a step of 32 keys that is lost among thousands shows in it, and in F16 results one key, where the bound on single numbers lets it pass"""
    H, dim, rest, vdim, rank = shape
    c = Case(dev, P, rank, rest, pos0, counts, seed=H + P)
    r, T, at = c.rng, sum(counts), 0
    uk, uv = ((r.normal(size=s) * rank ** -0.5).astype(np.float16) for s in ((H * dim, rank), (H * vdim, rank)))
    q, s = r.normal(size=(T, H, dim + rest)).astype(np.float16), r.normal(size=H).astype(np.float32) if sink else None
    scale = (dim + rest) ** -0.5
    got = attend(dev, c, q.reshape(T, -1), uk, uv, H, scale, window, s, FORMS[form], out_type).reshape(T, H, vdim)
    # Relative, of independent errors: the result's rounding, at most half a step of 2^-8 or 2^-11 of it; a weight's and a value's, 2^-11 / sqrt(3) at most each; and a weight by its score, whose terms
    # add up to scores of about 1 with a rounding of 2^-11 / sqrt(3) each.  Three of 2^-11.8 beside the result's own
    own = 2.0 ** -8 if out_type == capi.BF16 else 2.0 ** -11
    lim = (own ** 2 / 3 + 3 * (2.0 ** -11.8) ** 2) ** 0.5 * 1.25
    for i, n in enumerate(counts):
        mine = slice(at, at + n)
        want = whole(c, i, q[mine], uk, uv, H, scale, window, s)
        size = np.sqrt((want ** 2).mean())
        assert np.sqrt(((got[mine] - want) ** 2).mean()) <= lim * size, (i, np.sqrt(((got[mine] - want) ** 2).mean()) / size, lim)
        # .. for every token, whose results are H * vdim numbers
        each = np.sqrt(((got[mine] - want) ** 2).mean((1, 2))) / np.sqrt((want ** 2).mean((1, 2)))
        assert (each <= 1.5 * lim).all(), (i, each.max(), lim)
        if pos0[i] >= 300 and H <= 16:
            key = c.pos0[i] - (100 if window else 200)
            lost = whole(c, i, q[mine], uk, uv, H, scale, window, s, leave_out=slice(key, key + 32) if out_type == capi.BF16 else key)
            assert np.sqrt(((lost - want) ** 2).mean()) > 1.5 * lim * size
        at += n


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("window", [0, 12])
def test_each_row_that_is_not_finite(dev, form, window):
    """a NaN or an infinity in c, and a NaN or the infinity that the query's sign makes +infinity in r: NaN for the queries that see the row.  The other infinity in r: the weight 0"""
    bad = [(50, 3, np.nan), (45, 35, np.inf), (100, 0, -np.inf), (41, 7, np.inf), (60, 40, np.nan), (47, 33, -np.inf)]
    pos0, counts, H, dim, vdim, rank = [40, 40, 90, 40, 50, 40], [20, 20, 40, 3, 33, 20], 3, 32, 32, 32
    c = Case(dev, 16, rank, 16, pos0, counts, seed=window)
    clean = [c.rows(i, pos0[i] + counts[i]).copy() for i in range(len(bad))]
    for i, (at, col, x) in enumerate(bad):
        row = clean[i][at].copy()
        row[col] = x
        c.put(i, at, row[None])
    T = sum(counts)
    q = (np.abs(c.rng.normal(size=(T, H, dim + 16))) + 0.25).astype(np.float16)
    uk, uv = (np.abs(c.rng.normal(size=(H * d, rank)) * 0.2).astype(np.float16) + np.float16(0.01) for d in (dim, vdim))
    got, first = attend(dev, c, q.reshape(T, -1), uk, uv, H, 0.2, window, None, FORMS[form]).reshape(T, H, vdim), 0
    for i, (at, col, x) in enumerate(bad):
        n = counts[i]
        rows, mine = clean[i].copy(), got[first:first + n]
        weightless = col >= rank and x == -np.inf
        if weightless:
            rows[at, col] = -65504.0                                         # x 0.25 x 0.2: a weight of 0 in 64 bits too
        want, size = R.attention(rows, pos0[i], q[first:first + n], uk, uv, rank, H, 0.2, window)
        pos = pos0[i] + np.arange(n)
        sees = (pos >= at) & ((pos - at < window) if window else True) & (not weightless)
        assert np.isnan(mine[sees]).all() and np.isfinite(mine[~sees]).all(), i
        np.testing.assert_allclose(mine[~sees], want[~sees], rtol=0.01, atol=0.01)
        first += n
