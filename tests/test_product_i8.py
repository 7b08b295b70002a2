"""Products in 8-bit integers (cc_product_i8) against their definition in 64 bits, and a layer's attention half in 8 bits: product, append, attention, product."""
import numpy as np
import pytest

from crabml_b200 import CudaError, CudaTensor, TensorError, TensorStrider, capi, paged, seqops
from tests import paged_ref as R
from tests.gpu_common import make_device
from tests.test_paged_ops import freqs, give, take

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = make_device()
    yield d
    d.close()


def weights(r, m, k, low=-127):
    return r.integers(low, 128, (m, k)).astype(np.int8), r.uniform(0.5, 1.5, m).astype(np.float32) / np.float32(60 * np.sqrt(k))


def check(dev, w, ws, x, xt=None):
    got = take(dev, seqops.product_i8(give(dev, w), give(dev, ws), give(dev, x) if xt is None else xt))
    want, _ = R.product(w, ws, x)
    assert got.shape == want.shape
    want = np.where(np.abs(want) > np.finfo(np.float32).max, np.copysign(np.inf, want), want)      # 20 of 1e37 and their like: no 32-bit number
    # the sum is exact until it becomes a 32-bit number; that, two factors of 24 bits and two products: five roundings
    np.testing.assert_allclose(got, want, rtol=5 * 2.0 ** -24, atol=1e-37)
    return got


ROWS = [1, 2, 7, 8, 9, 16, 31, 33, 64, 127, 128, 129, 300]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("m,k", [(1, 1), (5, 16), (128, 128), (129, 64), (256, 1000), (77, 513), (512, 4096), (1000, 130), (300, 2064)])
def test_product(dev, rows, m, k):
    r = np.random.default_rng(rows * 1000 + k)
    w, ws = weights(r, m, k)
    check(dev, w, ws, r.normal(size=(rows, k)).astype(np.float32) * np.float32(10.0 ** r.uniform(-3, 3)))


@pytest.mark.parametrize("rows,m,k", [(129, 19000, 64), (300, 9500, 130), (600, 9217, 272), (1100, 6145, 16), (1500, 13000, 48)])
def test_product_of_many_tiles(dev, rows, m, k):
    """more tiles than pairs of SMs, with a last wave of few, of many, and of tiles that end behind the tokens and the channels"""
    r = np.random.default_rng(m)
    w, ws = weights(r, m, k)
    check(dev, w, ws, r.normal(size=(rows, k)).astype(np.float32))


@pytest.mark.parametrize("rows", [1, 20, 200])
def test_extremes(dev, rows):
    """the largest sums there are, -128 among the weights, rows of zeros, of tiny and of huge numbers"""
    r = np.random.default_rng(rows)
    k = 131072
    w = np.full((9, k), 127, np.int8)
    w[1], w[2] = -128, r.integers(-128, 128, k)
    x = np.ones((rows, k), np.float32)
    x[rows // 2] *= np.float32(-1e-35)
    if rows > 2:
        x[1] = 0
        x[2] = r.normal(size=k).astype(np.float32) * np.float32(1e37)
        x[3, :] = 0
        x[3, 5] = np.float32(1e-38)
    check(dev, w, np.ones(9, np.float32), x)


@pytest.mark.parametrize("rows", [1, 40])
def test_codes_next_to_borders(dev, rows):
    """an identity shows the codes themselves: numbers at and next to k + 1/2, from both sides"""
    k = 4096
    a = np.float32(127.0 * 1.0009765625)
    x = np.zeros((rows, k), np.float32)
    for i in range(rows):
        half = (np.arange(k) % 253 - 126 + 0.5) * np.float64(a) / 127
        x[i] = half.astype(np.float32)
        x[i] = np.where(np.arange(k) % 3 == 0, np.nextafter(x[i], np.float32(-1e9)), np.where(np.arange(k) % 3 == 1, np.nextafter(x[i], np.float32(1e9)), x[i]))
        x[i, i] = a
        x[i, 100:200] = (np.arange(100) - 50 + 0.5).astype(np.float32) * (a / np.float32(127))
    w = np.eye(k, dtype=np.int8)
    got = take(dev, seqops.product_i8(give(dev, w), give(dev, np.full(k, 1, np.float32)), give(dev, x)))
    _, codes = R.product(w, np.ones(k, np.float32), x)
    np.testing.assert_array_equal(np.rint(got / (np.abs(x).max(1, keepdims=True) / np.float32(127))), codes)


@pytest.mark.parametrize("rows", [3, 150])
def test_rows_that_are_not_finite(dev, rows):
    r = np.random.default_rng(0)
    w, ws = weights(r, 70, 300)
    x = r.normal(size=(rows, 300)).astype(np.float32)
    clean = check(dev, w, ws, x)
    x[0, 7], x[1, 299] = np.nan, -np.inf
    got = take(dev, seqops.product_i8(give(dev, w), give(dev, ws), give(dev, x)))
    assert np.isnan(got[:2]).all()
    np.testing.assert_array_equal(got[2:], clean[2:])


def test_a_row_does_not_depend_on_its_call(dev):
    """exact sums: the same bits for a row by itself and among others"""
    r = np.random.default_rng(3)
    w, ws = weights(r, 520, 1040)
    x = r.normal(size=(260, 1040)).astype(np.float32)
    wt, st = give(dev, w), give(dev, ws)
    every = take(dev, seqops.product_i8(wt, st, give(dev, x)))
    for lo, hi in ((0, 1), (7, 9), (100, 117), (100, 190), (3, 260)):
        np.testing.assert_array_equal(take(dev, seqops.product_i8(wt, st, give(dev, x[lo:hi]))), every[lo:hi])


@pytest.mark.parametrize("rows", [1, 5, 140])
def test_rows_of_a_wider_matrix(dev, rows):
    r = np.random.default_rng(rows)
    w, ws = weights(r, 33, 48)
    wide = r.normal(size=(rows, 61)).astype(np.float32)
    t = give(dev, wide).with_strider(TensorStrider([rows, 48], [61, 1]))
    check(dev, w, ws, np.ascontiguousarray(wide[:, :48]), t)


def test_refusals_and_nothing(dev):
    r = np.random.default_rng(0)
    w, ws = weights(r, 8, 32)
    wt, st, x = give(dev, w), give(dev, ws), give(dev, np.zeros((2, 32), np.float32))
    assert seqops.product_i8(wt, st, CudaTensor.alloc([0, 32], capi.F32, dev)).shape() == [0, 8]
    bad = [(x, st, x), (wt, give(dev, ws[:7]), x), (wt, st, give(dev, np.zeros((2, 33), np.float32))), (wt, st, give(dev, np.zeros((2, 32), np.float16))),
           (wt, wt, x), (wt.transpose([1, 0]), st, x), (wt, st, x.reshape([1, 2, 32])), (give(dev, np.zeros((1, 131073), np.int8)), give(dev, ws[:1]), give(dev, np.zeros((1, 131073), np.float32))),
           (wt, st, x.with_strider(TensorStrider([3, 32], [32, 1])))]
    for args in bad:
        with pytest.raises((TensorError, CudaError)):
            seqops.product_i8(*args)
    lazy = make_device(lazy=True)
    with pytest.raises(CudaError):
        seqops.product_i8(CudaTensor.alloc([8, 32], capi.I8, lazy), CudaTensor.alloc([8], capi.F32, lazy), CudaTensor.alloc([2, 32], capi.F32, lazy))
    lazy.close()
    seqops.product_i8(wt, st, x)


@pytest.mark.parametrize("i8", [False, True], ids=["f16", "i8"])
def test_a_layer_step_by_step(dev, i8):
    """product of the stacked projections, append, attention, output product, as a serving program runs them: prompts, then tokens, then a portion, sequences of ragged
    lengths; each step against 64 bits from the step's own inputs"""
    r = np.random.default_rng(4)
    D, H, G, d, P = 192, 6, 2, 32, 16
    w, ws = weights(r, (H + 2 * G) * d, D)
    wo, wos = weights(r, D, H * d)
    wt, st, ot, ost, f = give(dev, w), give(dev, ws), give(dev, wo), give(dev, wos), freqs(d // 2)
    ft = give(dev, f)
    S = 3
    table = [list(range(i, 40, 4)) for i in range(S)]
    cache = paged.PagedCache.alloc(dev, 40, G, P, d, dtype=capi.I8 if i8 else capi.F16, n_slots=S if i8 else 0)
    ref = R.Cache(40, G, P, d, d, i8, S)
    for n in ref.a:
        ref.a[n][...] = 0
    lens = [0] * S
    for counts in ([30, 5, 17], [1, 1, 1], [1, 0, 1], [40, 1, 2], [1, 30, 1]):
        T = sum(counts)
        x = r.normal(size=(T, D)).astype(np.float32)
        plan = paged.PagePlan(dev, P, 40, table, lens, counts, S if i8 else 0)
        qkv = seqops.product_i8(wt, st, give(dev, x))
        q = paged.append(plan, cache, qkv, 0, qkv, H * d, qkv, (H + G) * d, H, freq=ft)
        y = paged.attention(plan, cache, q, H, d ** -0.5)
        out = take(dev, seqops.product_i8(ot, ost, y))
        rows = take(dev, qkv)
        np.testing.assert_allclose(rows, R.product(w, ws, x)[0], rtol=5 * 2.0 ** -24)
        pos = np.concatenate([np.arange(p, p + n) for p, n in zip(lens, counts)])
        turned = R.turn(rows[:, :(H + G) * d].reshape(T, -1, d), pos, f, 0, 0, 1.0)
        np.testing.assert_allclose(take(dev, q).reshape(T, H, d), turned[:, :H], rtol=2.0 ** -23, atol=1e-14)
        at, yy = 0, take(dev, y)
        for i, n in enumerate(counts):
            ref.append(table[i], lens[i], i, {"k": turned[at:at + n, H:].astype(np.float32), "v": rows[at:at + n, (H + G) * d:].reshape(n, G, d)})
            lens[i] += n
            if n:
                want, mass, reach = R.attention(take(dev, q)[at:at + n].reshape(n, H, d), ref.rows("k", table[i], lens[i], i), ref.rows("v", table[i], lens[i], i), lens[i] - n,
                                                float(np.float32(d ** -0.5)))
                assert (np.abs(yy[at:at + n].reshape(n, H, d) - want) <= R.attention_bound(mass, reach, d, lens[i])).all()
            at += n
        np.testing.assert_allclose(out, R.product(wo, wos, yy)[0], rtol=5 * 2.0 ** -24)
    for n, a in ref.a.items():
        np.testing.assert_array_equal(take(dev, getattr(cache, n)), a, err_msg=n)


@pytest.mark.parametrize("limit", [1, 2, 3, 5])
def test_few_sms(limit):
    """a device that is held to one SM has no pairs of them: the same products all the same"""
    d = make_device()
    d.set_sm_limit(limit)
    r = np.random.default_rng(limit)
    for T, m, k in ((1, 300, 640), (20, 300, 640), (129, 300, 640), (300, 700, 416)):
        w, ws = weights(r, m, k)
        check(d, w, ws, r.normal(size=(T, k)).astype(np.float32))
    d.close()
