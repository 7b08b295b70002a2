"""out = act(W x + bias) + residual (cc_product) against the same in 64 bits: types, odd sizes, strides, every activation, numbers at the ends of the types, refusals."""
import numpy as np
import pytest

from crabml_b200 import CudaError, CudaTensor, TensorError, TensorStrider, capi, seqops
from tests.gpu_common import make_device

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F = torch.float64
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = {F32: capi.F32, F16: capi.F16, BF16: capi.BF16}
EPS = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


@pytest.fixture(scope="module")
def dev():
    d = make_device()
    yield d
    d.close()


def view(t):
    return torch.as_tensor(t.bits(), device="cuda").view(BF16) if t.dtype() == capi.BF16 else torch.as_tensor(t, device="cuda")


def give(dev, a):
    t = CudaTensor.alloc(list(a.shape), TYPES[a.dtype], dev)
    dev.synchronize()
    if a.numel():
        view(t).copy_(a)
    torch.cuda.synchronize()
    return t


def take(dev, t):
    dev.synchronize()
    return view(t).clone()


def act64(y, act):
    if act in (capi.ACT_SILU, capi.ACT_SWISH):
        return y * torch.sigmoid(y)
    if act == capi.ACT_GELU_TANH:
        return 0.5 * y * (1.0 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y ** 3)))
    if act == capi.ACT_SIGMOID:
        return torch.sigmoid(y)
    return torch.clamp_min(y, 0.0) ** 2 if act == capi.ACT_RELU_SQUARED else y


def check(dev, w, x, bias=None, act=capi.ACT_NONE, residual=None, out=F32, x_tensor=None):
    y = seqops.product(give(dev, w), give(dev, x) if x_tensor is None else x_tensor, bias=None if bias is None else give(dev, bias), act=act,
                       residual=None if residual is None else give(dev, residual), out_type=TYPES[out])
    assert y.shape() == [x.shape[0], w.shape[0]] and y.dtype() == TYPES[out]
    got = take(dev, y).to(F)
    xr = x if x.dtype == w.dtype else (x.float().clamp(-65504, 65504) if w.dtype == F16 else x).to(w.dtype)
    a, b = xr.to(F), w.to(F)
    z, size = a @ b.T, a.abs() @ b.abs().T
    if bias is not None:
        z, size = z + bias.to(F), size + bias.to(F).abs()
    want = act64(z, act)
    # A sum of k terms in 32 bits: the tensor cores take 16 at a time and cut each partial sum off at 2^-23 of it, every partial sum is at most sum |terms|: one cut in 16 terms and one rounding
    # for each of the few sums that meet; bias and residual one rounding each.
    off = (x.shape[1] / 16 + 12) * 2.0 ** -23 * size
    # activations: slope at most 1.13 (silu, gelu), 0.25 (sigmoid), 2 z (squares); their own 32-bit steps 8 roundings of the result and of z
    if act == capi.ACT_RELU_SQUARED:
        off = 2 * (z.abs() + off) * off
    off = 1.13 * off + (0.0 if act == capi.ACT_NONE else 8 * 2.0 ** -24 * (want.abs() + z.abs()))
    if residual is not None:
        want = want + residual.to(F)
    lim = off + (EPS[out] + 2.0 ** -24) * (want.abs() + off) + 2.0 ** -25
    if out == F16:
        want = want.clamp(-65504, 65504)
    bad = ~((got - want).abs() <= lim)
    assert not bad.any(), (torch.nonzero(bad)[:4].tolist(), got[bad][:4], want[bad][:4], lim[bad][:4], int(bad.sum()))
    return got


def make(rows, m, k, w, x, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    return (r(m, k) * k ** -0.5).to(w), (r(rows, k) * torch.exp(r(rows, 1))).to(x), r(m), r(rows, m)


SIZES = [(1, 1, 1), (1, 16, 16), (1, 4096, 4096), (3, 17, 33), (7, 100, 129), (8, 64, 256), (9, 200, 72), (13, 1000, 520), (16, 48, 4104), (17, 33, 1000), (31, 256, 64), (32, 130, 96), (33, 300, 250),
         (64, 128, 64), (65, 129, 128), (100, 512, 1024), (128, 256, 7), (200, 1111, 640), (300, 77, 2048), (513, 257, 136), (1000, 384, 320)]


@pytest.mark.parametrize("w,x,out", [(BF16, BF16, BF16), (BF16, F32, F32), (F16, F16, F32), (F16, F32, F16), (BF16, F16, BF16), (F16, BF16, F16)], ids=str)
@pytest.mark.parametrize("rows,m,k", SIZES, ids=str)
def test_product(dev, rows, m, k, w, x, out):
    w, x, bias, res = make(rows, m, k, w, x, rows)
    check(dev, w, x, out=out)
    check(dev, w, x, bias=bias, act=capi.ACT_SILU, residual=res.to(out), out=out)


@pytest.mark.parametrize("act", [capi.ACT_NONE, capi.ACT_SILU, capi.ACT_GELU_TANH, capi.ACT_SWISH, capi.ACT_SIGMOID, capi.ACT_RELU_SQUARED])
@pytest.mark.parametrize("rows", [1, 40, 300])
@pytest.mark.parametrize("with_bias,with_res", [(False, False), (True, False), (False, True), (True, True)])
def test_epilogues(dev, rows, act, with_bias, with_res):
    w, x, bias, res = make(rows, 200, 320, BF16, BF16, act)
    check(dev, w, x, bias=bias if with_bias else None, act=act, residual=res if with_res else None, out=F32)


@pytest.mark.parametrize("k", [64, 4096, 14336])
@pytest.mark.parametrize("rows", [1, 20, 150])
def test_long_sums_of_one_sign(dev, rows, k):
    """sums whose terms all have one sign: what each step cuts off adds up, far below the tolerance of 16-bit results"""
    w, x, _, _ = make(rows, 150, k, F16, F16, 1)
    got = check(dev, w.abs(), x.abs(), out=F32)
    want = x.abs().to(F) @ w.abs().to(F).T
    assert float(((got - want).abs() / want).max()) < 1e-5


@pytest.mark.parametrize("rows,m,k", [(1, 37, 98304), (1, 37, 98312), (1, 300, 16385), (2, 300, 8191), (3, 64, 8191), (8, 300, 4096), (9, 300, 4096), (16, 200, 2048), (17, 200, 2048), (16, 130, 1023), (17, 130, 1023),
                                      (200, 500, 4200), (290, 2300, 4200), (600, 2500, 6200), (300, 700, 100), (129, 4100, 1100), (2, 8192, 72), (2, 8200, 72), (20, 500, 8300), (100, 500, 8300)], ids=str)
@pytest.mark.parametrize("w,out", [(BF16, BF16), (F16, F32)], ids=str)
def test_ways(dev, rows, m, k, w, out):
    """either side of the bounds between the kernels, and each number of parts of a depth"""
    a, b, bias, _ = make(rows, m, k, w, w, seed=k)
    check(dev, a, b, bias=bias, out=out)


@pytest.mark.parametrize("rows", [2, 70, 260])
def test_rows_of_a_wider_matrix(dev, rows):
    """x and the residual as column blocks, aligned and not, and a residual that is the same tensor for two calls"""
    for off in (8, 3):
        w, x, _, _ = make(rows, 144, 96, BF16, BF16, off)
        wide = torch.full((rows, 96 + off + 5), float("nan"), device="cuda", dtype=BF16)
        wide[:, :96] = x
        t = give(dev, wide)
        check(dev, w, x, x_tensor=t.with_strider(TensorStrider([rows, 96], [96 + off + 5, 1])))
        res = torch.randn(rows, 144 + off, device="cuda")
        r = give(dev, res)
        y = take(dev, seqops.product(give(dev, w), give(dev, x), residual=r.with_strider(TensorStrider([rows, 144], [144 + off, 1]))))
        np.testing.assert_allclose(y.cpu().numpy(), (x.to(F) @ w.to(F).T + res[:, :144].to(F)).cpu().numpy(), rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("rows", [1, 12, 140])
def test_numbers_that_are_not_finite(dev, rows):
    """an infinity or a NaN in a row of x reaches that row's results and no others; one in a row of W that column's"""
    w, x, _, _ = make(rows, 70, 128, F16, F16, 3)
    x[rows // 2, 5], w[9, 100] = float("nan"), float("inf")
    got = take(dev, seqops.product(give(dev, w), give(dev, x), out_type=capi.F16)).to(F)
    clean = torch.ones(rows, 70, dtype=torch.bool, device="cuda")
    clean[rows // 2], clean[:, 9] = False, False
    assert torch.isfinite(got[clean]).all() and torch.isnan(got[rows // 2]).all() and not torch.isfinite(got[:, 9]).any()


def test_ends_of_the_types(dev):
    """f16 results beyond its range become its largest; 32-bit rows beyond the range of f16 weights too"""
    for rows in (1, 40, 200):
        w = torch.zeros(20, 64, device="cuda", dtype=F16)
        w[:, 0] = torch.arange(20, device="cuda") * 300.0
        x = torch.zeros(rows, 64, device="cuda")
        x[:, 0] = 300.0
        check(dev, w, x, out=F16)
        x[:, 0] = 1e9
        got = take(dev, seqops.product(give(dev, w), give(dev, x), out_type=capi.F32)).to(F)
        assert torch.equal(got, (torch.full_like(x, 65504.0)[:, :1].to(F) * w[:, 0].to(F)[None]))


@pytest.mark.parametrize("limit", [1, 2, 5, 9])
def test_few_sms(limit):
    """a device that is held to a few SMs: the same products"""
    d = make_device()
    d.set_sm_limit(limit)
    for rows, m, k in ((1, 300, 640), (20, 300, 640), (129, 300, 1100), (300, 700, 4100)):
        for t in (BF16, F32):
            w, x, bias, _ = make(rows, m, k, BF16, BF16, rows)
            check(d, w, x, bias=bias, out=t)
    d.close()


@pytest.mark.parametrize("rows,m,k", [(3, 131100, 16400), (2, 131100, 16401), (70000, 32768, 16)], ids=str)
def test_far_numbers(dev, rows, m, k):
    """weights, or results, whose places lie beyond 2^31"""
    if torch.cuda.mem_get_info()[0] < 8 * (m * k + rows * m):
        pytest.skip("no room")
    w, x = CudaTensor.alloc([m, k], capi.BF16, dev), CudaTensor.alloc([rows, k], capi.BF16, dev)
    dev.synchronize()
    g = torch.Generator(device="cuda").manual_seed(k)
    view(w).normal_(0.0, k ** -0.5, generator=g)
    view(x).normal_(0.0, 1.0, generator=g)
    torch.cuda.synchronize()
    y = seqops.product(w, x, out_type=capi.BF16)
    dev.synchronize()
    for t in sorted({0, rows // 2, rows - 1}):
        for c in (0, m // 2, m - 40):
            a, b = view(w)[c:c + 40].double(), view(x)[t].double()
            want, size = a @ b, a.abs() @ b.abs()
            # sums of 16-bit results: 24 bits cut off after every 16 terms, and one rounding to bf16
            lim = want.abs() * 2.0 ** -8 + size * (k / 16 + 1) * 2.0 ** -23
            assert ((view(y)[t, c:c + 40].double() - want).abs() <= lim).all()


def test_bits(dev):
    """16-bit memory for libraries that know no bf16: the same memory, kept by who holds it, and no other type's"""
    t = give(dev, torch.arange(6, device="cuda", dtype=F32).reshape(2, 3).to(BF16))
    held = t.bits()
    at = held.__cuda_array_interface__
    assert at["typestr"] == "<i2" and at["shape"] == (2, 3) and at["data"][0] == t.bits().__cuda_array_interface__["data"][0]
    y = torch.as_tensor(held, device="cuda").view(BF16)
    del t
    assert y.float().tolist() == [[0, 1, 2], [3, 4, 5]]
    with pytest.raises(TensorError):
        give(dev, torch.zeros(2, 3, device="cuda")).bits()
    with pytest.raises(AttributeError):
        give(dev, torch.zeros(2, 3, device="cuda", dtype=BF16)).__cuda_array_interface__


def test_equal_calls(dev):
    for rows in (1, 30, 200):
        w, x, bias, _ = make(rows, 500, 1000, BF16, BF16, 2)
        t = [give(dev, v) for v in (w, x, bias)]
        y = [take(dev, seqops.product(t[0], t[1], bias=t[2])) for _ in range(3)]
        assert torch.equal(y[0], y[1]) and torch.equal(y[0], y[2])


def test_nothing(dev):
    w, _, _, _ = make(1, 20, 64, BF16, BF16)
    assert seqops.product(give(dev, w), CudaTensor.alloc([0, 64], capi.BF16, dev)).shape() == [0, 20]


def test_refusals(dev):
    w, x, bias, res = (give(dev, v) for v in make(4, 20, 64, BF16, BF16))
    other = make_device()
    bad = [
        lambda: seqops.product(give(dev, torch.zeros(20, 63, device="cuda", dtype=BF16)), x), lambda: seqops.product(give(dev, torch.zeros(20, 64, device="cuda")), x), lambda: seqops.product(w, x, bias=give(dev, torch.zeros(19, device="cuda"))),
        lambda: seqops.product(w, x, bias=give(dev, torch.zeros(20, device="cuda", dtype=F16))), lambda: seqops.product(w, x, act=6), lambda: seqops.product(w, x, act=-1),
        lambda: seqops.product(w, x, out_type=capi.I8), lambda: seqops.product(w, x, residual=res, out_type=capi.BF16), lambda: seqops.product(w, x, residual=give(dev, torch.zeros(4, 19, device="cuda"))),
        lambda: seqops.product(w, x, residual=give(dev, torch.zeros(3, 20, device="cuda"))), lambda: seqops.product(w, x.with_strider(TensorStrider([4, 64], [63, 1]))),
        lambda: seqops.product(w, x.with_strider(TensorStrider([4, 64], [65, 1]))), lambda: seqops.product(w.with_strider(TensorStrider([20, 64], [1, 20])), x),
        lambda: seqops.product(w, give(other, torch.zeros(4, 64, device="cuda", dtype=BF16))), lambda: seqops.product(w, CudaTensor.alloc([4, 64], capi.I8, dev)),
        lambda: seqops.product(w, x, act=1 << 32), lambda: seqops.product(w, x, out_type=-(1 << 32)), lambda: seqops.product(w, x, act="silu"), lambda: seqops.product(w, x, act=0.5),
    ]
    for f in bad:
        with pytest.raises(TensorError):
            f()
    other.close()
    check(dev, *make(4, 20, 64, BF16, BF16)[:2])


@pytest.mark.parametrize("w", [F16, BF16], ids=str)
@pytest.mark.parametrize("k", [128, 512, 1000, 1001, 2048, 3000])
@pytest.mark.parametrize("rows", [1, 8, 16, 40, 140])
def test_infinities(dev, rows, k, w):
    """an infinity in a row of x, in its last columns too, gives that row infinities of the weights' signs, by every kernel; one in W its column"""
    a, x, _, _ = make(rows, 70, k, w, w, k)
    a[a == 0] = 1.0
    for at in (k - 1, k - 20, 3):
        b = x.clone()
        b[rows // 2, at], b[0, k // 2] = float("inf"), -float("inf")
        got, want = take(dev, seqops.product(give(dev, a), give(dev, b))).to(F), b.to(F) @ a.to(F).T
        for v in (float("inf"), -float("inf")):
            assert torch.equal(got == v, want == v)
        assert torch.equal(got.isnan(), want.isnan())
    a[9, k - 2] = float("inf")
    got, want = take(dev, seqops.product(give(dev, a), give(dev, x))).to(F), x.to(F) @ a.to(F).T
    assert torch.equal(got == float("inf"), want == float("inf")) and torch.equal(got == -float("inf"), want == -float("inf")) and torch.equal(got.isnan(), want.isnan())


@pytest.mark.parametrize("act", [capi.ACT_NONE, capi.ACT_SILU, capi.ACT_GELU_TANH, capi.ACT_SWISH, capi.ACT_SIGMOID, capi.ACT_RELU_SQUARED])
@pytest.mark.parametrize("out", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("rows", [1, 12, 40, 140])
def test_activations_of_numbers_that_are_not_finite(dev, rows, out, act):
    """a NaN stays one under every activation, an infinity has the activation's limit; with and without a residual"""
    w, x, bias, res = make(rows, 70, 512, F16, F16, 3)
    w = w.abs() + 2.0 ** -10
    x[rows // 2, 500] = float("nan")
    if rows > 2:
        x[0, 500], x[2, 500] = float("inf"), -float("inf")
    for r in (None, res.to(out)):
        got = take(dev, seqops.product(give(dev, w), give(dev, x), bias=give(dev, bias), act=act, residual=None if r is None else give(dev, r), out_type=TYPES[out])).to(F)
        assert got[rows // 2].isnan().all() and torch.isfinite(got[3:rows // 2]).all() and torch.isfinite(got[rows // 2 + 1:] if rows > 2 else got[1:]).all()
        if rows > 2:
            up = 1.0 if act == capi.ACT_SIGMOID else float("inf")
            low = {capi.ACT_NONE: -float("inf"), capi.ACT_SIGMOID: 0.0, capi.ACT_RELU_SQUARED: 0.0}.get(act)
            for row, limit in ((0, up), (2, low)):
                if limit is not None:
                    want = torch.full((70,), limit, dtype=F, device="cuda") + (0.0 if r is None else r[row].to(out).to(F))
                    assert torch.equal(torch.isinf(got[row]), torch.isinf(want)) and torch.equal(got[row].sign(), want.sign())
                    fine = torch.isfinite(want)
                    # one rounding of the sum, beside a 32-bit step of a sigmoid of an infinity
                    assert ((got[row] - want)[fine].abs() <= (EPS[out] + 2.0 ** -23) * want[fine].abs() + 2.0 ** -25).all()


def test_types_that_are_allocated(dev):
    """plain types, as zeros; a refusal names them"""
    for t in (BF16, F16, F32):
        assert (take(dev, CudaTensor.alloc([3, 5], TYPES[t], dev)) == 0).all()
    for t in (capi.Q8_0 if hasattr(capi, "Q8_0") else 8, 99, -1):
        with pytest.raises(TensorError, match="f32, f16, bf16, i32 and i8"):
            CudaTensor.alloc([32], t, dev)


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_after_a_call_that_found_no_memory(dev, rows):
    """memory that is not there is that call's error, and no later one's: a tensor of 32 TB, then products by every kernel, and an older operation"""
    w, x, bias, _ = make(rows, 200, 320, BF16, F32, rows)
    with pytest.raises(CudaError):
        CudaTensor.alloc([1 << 44], capi.F16, dev)
    check(dev, w, x, bias=bias, out=F32)
    with pytest.raises(CudaError):
        CudaTensor.alloc([1 << 44], capi.F16, dev)
    y = CudaTensor.new(np.ones((4, 8), np.float32), [4, 8], dev)
    assert (seqops.activate_inplace(y, capi.ACT_RELU_SQUARED).export() == 1.0).all()
