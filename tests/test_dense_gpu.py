"""The dense-layer operators (norm with residual, conversion, linear) on the GPU against plain
implementations in 64 bits, through the C ABI.  Tolerances are derived where they stand; matrices
are surrounded by NaNs that must neither be read nor be overwritten."""
import math
import threading

import numpy as np
import pytest
import torch

import dense_util as U
from kaldi_amd import _lib, dense

pytestmark = pytest.mark.gpu
U24 = 2.0 ** -24


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(rows, cols, seed):
    return torch.randn((rows, cols), generator=gen(seed), dtype=torch.float64)


# ---- convert ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("tin", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tout", ["f32", "bf16", "f16", "mx8"])
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (3, 31, 1), (5, 32, 0), (2, 33, 3), (7, 360, 8), (65, 129, 5),
                                           (3, 517, 0), (2, 8600, 0)])
def test_convert(amlike_device, tin, tout, rows, cols, pad):
    x = U.rounded(randn(rows, cols, rows + cols) * torch.exp2(torch.arange(rows).double() - 3).unsqueeze(1), tin)
    dx = U.DeviceMatrix(rows, cols, tin, pad, fill=x)
    out = U.DeviceMatrix(rows, cols, tout, pad)
    dense.ConvertDevice(dx.m, rows, cols, out.m)
    torch.cuda.synchronize()
    assert U.same(out.values(), U.rounded(x, tout))  # one rounding of the same number: the same bits
    if tout == "mx8":
        q, s = U.to_mx8(x)
        assert torch.equal(out.scales[:rows, :s.shape[1]].cpu(), s)
    out.assert_rest_untouched()


def test_convert_to_mx8_borders(amlike_device):
    """Scales at their borders, values that are not finite, groups of zeros and of denormals."""
    rows = []
    for top in (448.0, 449.0, 448 * 2.0 ** -127, 448 * 2.0 ** -126, 449 * 2.0 ** -127, 2.0 ** -149, 2.0 ** -130, 3.0e38, 2.0 ** 127,
                1.75, 1.7500001192092896, 0.0, 1e-40):
        row = [top, -top / 2, top / 3, 0.0, -0.0, top * 2.0 ** -9, top * 2.0 ** -14, top * 2.0 ** -20] * 4
        rows.append(row)
    for bad in (math.inf, -math.inf, math.nan):
        rows.append([bad, 1.0, -300.0, 0.0] + [0.5] * 28)
        rows.append([bad] * 32)
        rows.append([bad] + [0.0] * 31)
    x = torch.tensor(rows, dtype=torch.float64).float().double()
    dx, out = U.DeviceMatrix(len(rows), 32, "f32", fill=x), U.DeviceMatrix(len(rows), 32, "mx8")
    dense.ConvertDevice(dx.m, len(rows), 32, out.m)
    torch.cuda.synchronize()
    q, s = U.to_mx8(x)
    assert torch.equal(out.scales[:len(rows), :1].cpu(), s)
    want = U.from_mx8(q, s)
    assert torch.equal(torch.isnan(want), ~torch.isfinite(x)) and U.same(out.values(), want)


def test_convert_16_bit_specials(amlike_device):
    x = torch.tensor([[math.inf, -math.inf, math.nan, 65504.0, 65519.0, 65520.0, -70000.0, 1e-8, 6e-8, 2.0 ** -25, 3.4e38, -0.0]],
                     dtype=torch.float64).float().double()
    for t in ("bf16", "f16"):
        dx, out = U.DeviceMatrix(1, 12, "f32", fill=x), U.DeviceMatrix(1, 12, t)
        dense.ConvertDevice(dx.m, 1, 12, out.m)
        torch.cuda.synchronize()
        assert U.same(out.values(), x.to(U.TORCH[t]).double())


# ---- norm --------------------------------------------------------------------------------------------

def norm_reference(x, r, w, eps):
    s = x + r if r is not None else x
    y = s / torch.sqrt((s * s).mean(1, keepdim=True) + eps)
    return s, y * w if w is not None else y


def norm_error(s, y):
    """Of y before its rounding: s carries half a step; the sum of squares is a chain of at most 32
    products per thread, 6 butterfly steps and 16 waves, so at most 54 roundings, half of which
    reach 1/sqrt; the mean, eps, the reciprocal square root (one unit) and two products add 6."""
    return (1 + 27 + 6) * U24 * y.abs()


@pytest.mark.parametrize("tin,tout", [("f32", "f32"), ("f32", "bf16"), ("f32", "mx8"), ("bf16", "bf16"), ("bf16", "mx8"),
                                      ("bf16", "f32"), ("f16", "f16"), ("f16", "mx8"), ("f16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("rows,dim,pad,res,weight", [
    (1, 1, 0, False, False), (3, 7, 2, True, True), (33, 128, 0, True, False), (17, 200, 0, False, True), (5, 257, 8, True, True),
    (4, 513, 1, True, True), (1, 2048, 0, True, True), (3, 1999, 0, True, True), (2, 4096, 0, False, False),
    (3, 5001, 3, True, True), (2, 8192, 0, True, True), (2, 32768, 0, True, True), (1, 20001, 0, False, True)])
def test_norm(amlike_device, tin, tout, rows, dim, pad, res, weight):
    loud = torch.exp2(torch.arange(rows).double() % 9 - 4).unsqueeze(1)
    x = U.rounded(randn(rows, dim, 1) * loud, tin)
    r = U.rounded(randn(rows, dim, 2) * loud, tin) if res else None
    w = (1 + 0.3 * randn(1, dim, 3)[0]).float().double() if weight else None
    eps = 1e-5
    norm = dense.RmsNorm(dim, w.numpy() if weight else None, eps)
    eps = float(np.float32(eps))
    dx = U.DeviceMatrix(rows, dim, tin, pad, fill=x)
    dr = U.DeviceMatrix(rows, dim, tin, pad, fill=r) if res else None
    ds, out = U.DeviceMatrix(rows, dim, tin, pad), U.DeviceMatrix(rows, dim, tout, pad)
    norm.ApplyDevice(dx.m, rows, out.m, residual=dr.m if res else None, sum=ds.m)
    torch.cuda.synchronize()
    s, y = norm_reference(x, r, w, eps)
    U.check_output(out, y, norm_error(s, y))
    U.check_output(ds, s, U24 * s.abs())  # the sum in fp32, then the rounding to its type
    for m in (ds, out):
        m.assert_rest_untouched()
    # the sum is optional and does not change the output
    out2 = U.DeviceMatrix(rows, dim, tout, pad)
    norm.ApplyDevice(dx.m, rows, out2.m, residual=dr.m if res else None)
    torch.cuda.synchronize()
    assert torch.equal(out.values(), out2.values())


def test_norm_in_place(amlike_device):
    """The residual stream updated in place, and the output over its input."""
    for dim in (200, 2048, 9000):
        x, r = U.rounded(randn(9, dim, 4), "bf16"), U.rounded(randn(9, dim, 5), "bf16")
        norm = dense.RmsNorm(dim)
        dx, dr = U.DeviceMatrix(9, dim, "bf16", fill=x), U.DeviceMatrix(9, dim, "bf16", fill=r)
        ds, out = U.DeviceMatrix(9, dim, "bf16"), U.DeviceMatrix(9, dim, "bf16")
        norm.ApplyDevice(dx.m, 9, out.m, residual=dr.m, sum=ds.m)
        norm.ApplyDevice(dx.m, 9, dr.m, residual=dr.m, sum=dx.m)
        torch.cuda.synchronize()
        assert torch.equal(dx.values(), ds.values()) and torch.equal(dr.values(), out.values())


def test_norm_rows_that_leave_the_range(amlike_device):
    """Squares beyond fp32, rows of zeros, infinities and NaN; the other rows do not notice."""
    dim = 300
    x = randn(8, dim, 6)
    x[0] *= 1e30
    x[1] = 3.4e38
    x[2] = 0
    x[3, 7] = math.inf
    x[4, 250] = math.nan
    x[5] *= 1e-20
    x[6, 299] = -math.inf
    x = x.float().double()
    for tout in ("f32", "mx8"):
        out = U.DeviceMatrix(8, dim, tout)
        dense.RmsNorm(dim, None, 1e-6).ApplyDevice(U.DeviceMatrix(8, dim, "f32", fill=x).m, 8, out.m)
        torch.cuda.synchronize()
        s, y = norm_reference(x, None, None, float(np.float32(1e-6)))
        y[3], y[4], y[6] = 0, math.nan, 0
        y[3, 7] = y[6, 299] = math.nan
        U.check_output(out, y, norm_error(s, torch.nan_to_num(y)))


def test_norm_host(amlike_device):
    x, r = randn(37, 200, 7).float().numpy(), randn(37, 200, 8).float().numpy()
    w = (1 + 0.1 * randn(1, 200, 9)[0]).float().numpy()
    norm = dense.RmsNorm(200, w, 1e-5)
    assert norm.Dim() == 200
    t = lambda a: torch.from_numpy(a).double()  # noqa: E731
    s, y = norm_reference(t(x), t(r), t(w), float(np.float32(1e-5)))
    got, total = norm.Apply(x, residual=r, return_sum=True)
    U.assert_close(t(got), y, norm_error(s, y) + U24 * y.abs())
    U.assert_close(t(total), s, U24 * s.abs())
    s, y = norm_reference(t(x), None, t(w), float(np.float32(1e-5)))
    wide = np.full((37, 230), np.nan, np.float32)
    wide[:, :200] = x
    U.assert_close(t(norm.Apply(wide[:, :200])), y, norm_error(s, y) + U24 * y.abs())
    assert norm.Apply(x[:0]).shape == (0, 200)


# ---- linear --------------------------------------------------------------------------------------------

ACT = {"none": lambda v: v, "relu": lambda v: torch.where(v < 0, torch.zeros_like(v), v), "sigmoid": torch.sigmoid,
       "tanh": torch.tanh, "silu": lambda v: v * torch.sigmoid(v), "gelu": lambda v: v * 0.5 * torch.erfc(-v * math.sqrt(0.5))}  # 1 + erf would cancel


def linear_reference(x, w, b, act, r):
    pre = x @ w.t()
    mass = x.abs() @ w.abs().t()
    if b is not None:
        pre, mass = pre + b, mass + b.abs()
    y = ACT[act](pre)
    return pre, mass, y + r if r is not None else y, y


def linear_error(k, mass, pre, act_y, y, tout, act, type_="bf16"):
    """Before the output's rounding.  The products are exact in fp32; a sum of k of them and the bias
    in any order, each addition rounded or cut off (2^-23), is off by at most (k + 1) * 2^-23 * mass.
    An activation has slope at most 1.13.  Its own error: exp2's argument carries half a step of
    up to 1.45 |pre| and the result a few units, which a sigmoid passes on as at most
    (3 + |pre|) * 2^-23 of itself; gelu's polynomial is 1.5e-7 off for fp32 outputs, 3.5e-5 otherwise,
    on the normal tail, which is at most half of |pre|, its exponential's argument pre^2 / 2 carries
    4 roundings, and exp(-a) * a is below 1/2.  The residual's addition rounds once."""
    e = 1.13 * (k + 1) * 2.0 ** -23 * mass
    if type_ == "mx8" and tout != "f32":
        # the 8-bit instruction drops what lies over 13 places below the largest of (taken here) four
        # neighbouring products: at most 3 * 2^-13 of that one, and so of the mass
        e = e + 1.13 * 3 * 2.0 ** -13 * mass
    if act in ("sigmoid", "tanh", "silu"):
        e = e + (6 + 2 * pre.abs()) * 2.0 ** -23 * torch.clamp(act_y.abs(), min=1.0 if act == "tanh" else 0.0)
    if act == "gelu":
        e = e + pre.abs() * ((1.5e-7 if tout == "f32" else 3.5e-5) * 0.5 + 8 * 2.0 ** -23)
    return e + U24 * (y.abs() + act_y.abs())


SIZES = [(1, 1, 1), (1, 64, 64), (1, 2048, 200), (2, 33, 5), (3, 360, 129), (7, 129, 64), (16, 512, 320), (17, 250, 96), (31, 1000, 65),
         (33, 127, 257), (64, 128, 128), (65, 63, 191), (100, 360, 300), (129, 200, 70), (300, 96, 264), (257, 520, 513), (640, 136, 520),
         (2100, 80, 8200), (4099, 72, 4160), (9000, 65, 520),
         (256, 3328, 4096), (200, 1984, 1032)]


@pytest.mark.parametrize("type_", ["bf16", "f16", "mx8"])
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_linear_is_exact_on_small_integers(amlike_device, type_, rows, k, n):
    """Integers whose sums fp32 holds exactly: every product is there once, and nothing else."""
    for pad in (0, 3, 8) if rows < 2000 and n < 4000 else (8,) if rows > 2000 else (0,):
        x = torch.randint(-8, 9, (rows, k), generator=gen(k + pad)).double()
        w = torch.randint(-8, 9, (n, k), generator=gen(n + pad)).double()
        b = torch.randint(-99, 99, (n,), generator=gen(7)).double()
        r = torch.randint(-99, 99, (rows, n), generator=gen(8)).double()
        lin = dense.Linear(w.numpy(), b.numpy(), type_)
        assert (lin.InputDim(), lin.OutputDim()) == (k, n)
        dx = U.DeviceMatrix(rows, k, type_, pad, fill=x)
        dr = U.DeviceMatrix(rows, n, "f32", pad, fill=r)
        out = U.DeviceMatrix(rows, n, "f32", pad)
        lin.ApplyDevice(dx.m, rows, out.m, residual=dr.m)
        torch.cuda.synchronize()
        assert torch.equal(out.values(), x @ w.t() + b + r), (pad,)
        out.assert_rest_untouched()
        if type_ == "mx8":  # a 16-bit output: the 8-bit instruction (products below 2^7 lose nothing in it)
            out = U.DeviceMatrix(rows, n, "bf16", pad)
            lin.ApplyDevice(dx.m, rows, out.m, residual=dr.m)
            torch.cuda.synchronize()
            assert torch.equal(out.values(), (x @ w.t() + b + r).bfloat16().double()), (pad,)
            out.assert_rest_untouched()
        if rows > 1:  # the 8-bit scales of different groups: rows and weights at different powers of two
            p, q = torch.exp2(torch.arange(rows).double() % 5 - 2).unsqueeze(1), torch.exp2(torch.arange(n).double() % 7 - 3)
            c = torch.exp2((torch.arange(k) // 32).double() % 3)
            lin2 = dense.Linear((w * q.unsqueeze(1) * c).numpy(), None, type_)
            dx = U.DeviceMatrix(rows, k, type_, pad, fill=x * p / c)
            out = U.DeviceMatrix(rows, n, "f32", pad)
            lin2.ApplyDevice(dx.m, rows, out.m, activation="relu")
            torch.cuda.synchronize()
            assert torch.equal(out.values(), torch.relu((x @ w.t()) * p * q)), (pad,)
            if type_ == "mx8":
                out = U.DeviceMatrix(rows, n, "bf16", pad)
                lin2.ApplyDevice(dx.m, rows, out.m, activation="relu")
                torch.cuda.synchronize()
                assert torch.equal(out.values(), torch.relu((x @ w.t()) * p * q).bfloat16().double()), (pad,)


# Sizes that are large enough for every form of the tile kernel on 256 compute units (in 8 bits with twice
# the columns): k-tiles of one block and of two groups of waves, 64, 128 and 256 wide, one tile a
# block and several; the last is for rows that start anywhere.
FORMS = [(990, 200, 2000, 16), (60000, 200, 60, 16), (500, 1000, 2000, 16), (3990, 200, 1990, 16), (4090, 200, 4600, 16), (1990, 1000, 1990, 16),
         (90000, 504, 120, 16), (4090, 1000, 4090, 16), (8000, 200, 8000, 16), (500, 1017, 2000, 3)]


@pytest.mark.parametrize("type_", ["bf16", "f16", "mx8"])
@pytest.mark.parametrize("rows,k,n,pad", FORMS)
def test_linear_forms_are_exact_on_small_integers(amlike_device, type_, rows, k, n, pad):
    k *= 2 if type_ == "mx8" else 1
    x = torch.randint(-8, 9, (rows, k), generator=gen(61)).double()
    w = torch.randint(-8, 9, (n, k), generator=gen(62)).double()
    b = torch.randint(-99, 99, (n,), generator=gen(63)).double()
    lin = dense.Linear(w.numpy(), b.numpy(), type_)
    dx = U.DeviceMatrix(rows, k, type_, pad, fill=x)
    want = x @ w.t() + b
    for tout in ("f32", "bf16", "mx8") if rows < 5000 else ("f32", "bf16"):
        out = U.DeviceMatrix(rows, n, tout, pad)
        lin.ApplyDevice(dx.m, rows, out.m)
        torch.cuda.synchronize()
        U.check_output(out, want, torch.zeros_like(want)) if tout == "mx8" else U.assert_close(out.values(), U.rounded(want, tout), 0.0, tout)
        out.assert_rest_untouched()


@pytest.mark.parametrize("type_", ["bf16", "f16", "mx8"])
@pytest.mark.parametrize("tout,act,tres", [("f32", "none", None), ("f32", "gelu", "f32"), ("f32", "tanh", "bf16"), ("f32", "silu", None),
                                           ("f32", "sigmoid", "f16"), ("bf16", "gelu", "bf16"), ("bf16", "relu", None), ("f16", "silu", "f16"),
                                           ("f16", "none", "f32"), ("mx8", "gelu", None), ("mx8", "silu", "bf16"), ("mx8", "none", "f32"),
                                           ("bf16", "tanh", None), ("f16", "sigmoid", None)])
@pytest.mark.parametrize("rows,k,n,pad", [(1, 500, 200, 0), (5, 64, 33, 1), (16, 1024, 256, 0), (40, 300, 100, 8), (130, 256, 300, 0),
                                          (520, 200, 264, 8)])
def test_linear_epilogue(amlike_device, type_, tout, act, tres, rows, k, n, pad):
    x, w = U.rounded(2 * randn(rows, k, 11), type_), U.rounded(randn(n, k, 12) / math.sqrt(k), type_)
    b = randn(1, n, 13)[0].float().double()
    r = U.rounded(3 * randn(rows, n, 14), tres) if tres else None
    lin = dense.Linear(w.numpy(), b.numpy(), type_)
    dx = U.DeviceMatrix(rows, k, type_, pad, fill=x)
    dr = U.DeviceMatrix(rows, n, tres, pad, fill=r) if tres else None
    out = U.DeviceMatrix(rows, n, tout, pad)
    lin.ApplyDevice(dx.m, rows, out.m, activation=act, residual=dr.m if tres else None)
    torch.cuda.synchronize()
    pre, mass, y, act_y = linear_reference(x, w, b, act, r)
    U.check_output(out, y, linear_error(k, mass, pre, act_y, y, tout, act, type_))
    out.assert_rest_untouched()


@pytest.mark.parametrize("act", ["relu", "sigmoid", "tanh", "silu", "gelu"])
def test_linear_activations_over_their_range(amlike_device, act):
    """A layer that copies its input (f16): small, large and extreme arguments."""
    v = torch.cat([torch.linspace(-12, 12, 977), torch.tensor([0.0, -0.0, 1e-4, -1e-4, 6e-8, 60.0, -60.0, 300.0, -300.0, 6e4, -6e4]),
                   torch.logspace(-6, 1, 36)]).to(torch.float16).double()
    x = v.repeat(1, 1)
    n = x.shape[1]
    lin = dense.Linear(np.eye(n, dtype=np.float32), None, "f16")
    out = U.DeviceMatrix(1, n, "f32")
    lin.ApplyDevice(U.DeviceMatrix(1, n, "f16", fill=x).m, 1, out.m, activation=act)
    torch.cuda.synchronize()
    want, got = ACT[act](x), out.values()
    # (the product is exact here.)  gelu's factor is relatively exact, so its result is too, as the
    # exponent's 4 roundings of up to pre^2 / 2 allow
    tol = {"relu": 0 * x, "sigmoid": (6 + 2 * x.abs()) * 2.0 ** -23 * want, "silu": (6 + 2 * x.abs()) * 2.0 ** -23 * want.abs(),
           "tanh": 6 * 2.0 ** -23 * want.abs(), "gelu": (2e-7 + (8 + 2 * x * x) * 2.0 ** -23) * want.abs()}[act]
    U.assert_close(got, want, tol + 2.0 ** -125)  # (what is below fp32's normal range may be cut off)


def test_linear_rows_are_independent_and_nan_stays_in_its_row(amlike_device):
    """A row's bits depend neither on the other rows nor on how many there are of the same kernel."""
    rng_w = randn(200, 360, 21) / 19
    for type_ in ("bf16", "f16", "mx8"):
        x = U.rounded(randn(300, 360, 22), type_)
        lin = dense.Linear(rng_w.numpy(), None, type_)

        def run(a):
            out = U.DeviceMatrix(a.shape[0], 200, "f32")
            lin.ApplyDevice(U.DeviceMatrix(a.shape[0], 360, type_, fill=a).m, a.shape[0], out.m, activation="silu")
            torch.cuda.synchronize()
            return out.values()

        base = run(x)
        bad = x.clone()
        bad[17, 5] = math.nan
        bad[250, 359] = math.inf
        got = run(bad)
        assert torch.isnan(got[17]).all() and not torch.isfinite(got[250]).any()
        keep = torch.ones(300, dtype=torch.bool)
        keep[17] = keep[250] = False
        assert torch.equal(got[keep], base[keep])


def test_linear_extreme_scales(amlike_device):
    """8-bit groups at both ends of the scales' range."""
    k, n = 128, 64
    c = torch.exp2(torch.tensor([-100.0, 0, 100, 110]).double()).repeat_interleave(32)
    x, w = torch.randint(-8, 9, (20, k), generator=gen(1)).double(), torch.randint(-8, 9, (n, k), generator=gen(2)).double()
    x[:, 0::32], w[:, 0::32] = 8, 8
    lin = dense.Linear((w / c).numpy(), None, "mx8")
    for tout in ("f32", "bf16"):
        out = U.DeviceMatrix(20, n, tout)
        lin.ApplyDevice(U.DeviceMatrix(20, k, "mx8", fill=x * c).m, 20, out.m)
        torch.cuda.synchronize()
        assert torch.equal(out.values(), U.rounded(x @ w.t(), tout))
    # the smallest scale there is, 2^-127, under a large one
    x = torch.zeros(3, 64, dtype=torch.float64)
    x[:, :32] = torch.randint(1, 9, (3, 32), generator=gen(3)).double() * 2.0 ** -133
    wide = torch.full((n, 64), 2.0 ** 100, dtype=torch.float64)
    for tout in ("f32", "bf16"):
        out = U.DeviceMatrix(3, n, tout)
        dense.Linear(wide.numpy(), None, "mx8").ApplyDevice(U.DeviceMatrix(3, 64, "mx8", fill=x).m, 3, out.m)
        torch.cuda.synchronize()
        assert torch.equal(out.values(), U.rounded(x @ wide.t(), tout))


@pytest.mark.parametrize("rows,k,n", [(3, 96, 40), (20, 256, 64), (990, 400, 2000)])
def test_linear_scale_bytes_at_both_ends(amlike_device, rows, k, n):
    """Byte 0 stands for 2^-127, byte 255 for NaN: of its row alone."""
    x, w = torch.randint(-8, 9, (rows, k), generator=gen(71)).double(), torch.randint(-8, 9, (n, k), generator=gen(72)).double()
    w[:, ::3] = 8
    lin = dense.Linear(w.numpy(), None, "mx8")
    dx = U.DeviceMatrix(rows, k, "mx8", 16, fill=x)
    dx.scales[0, :(k + 31) // 32] = 0
    dx.scales[rows - 1, 1] = 255
    want = dx.values()[:rows - 1] @ w.t()
    for tout in ("f32", "bf16"):
        out = U.DeviceMatrix(rows, n, tout)
        lin.ApplyDevice(dx.m, rows, out.m)
        torch.cuda.synchronize()
        got = out.values()
        assert torch.isnan(got[rows - 1]).all()
        # (integers of at most 8 are held as multiples of 2^5 and more: no sum lies below 2^-122)
        assert torch.equal(got[:rows - 1], U.rounded(want, tout))


def test_linear_residual_in_place(amlike_device):
    x, r = U.rounded(randn(50, 96, 31), "bf16"), U.rounded(randn(50, 130, 32), "bf16")
    lin = dense.Linear((randn(130, 96, 33) / 10).numpy(), None, "bf16")
    dx, dr = U.DeviceMatrix(50, 96, "bf16", fill=x), U.DeviceMatrix(50, 130, "bf16", fill=r)
    out = U.DeviceMatrix(50, 130, "bf16")
    lin.ApplyDevice(dx.m, 50, out.m, residual=dr.m)
    lin.ApplyDevice(dx.m, 50, dr.m, residual=dr.m)
    torch.cuda.synchronize()
    assert torch.equal(out.values(), dr.values())


def test_linear_host(amlike_device):
    x, w = randn(70, 40, 41).float(), (randn(33, 40, 42) / 6).float()
    r = randn(70, 33, 43).float()
    for type_ in ("bf16", "f16", "mx8"):
        lin = dense.Linear(w.numpy(), None, type_)
        got = torch.from_numpy(lin.Apply(x.numpy(), "gelu", r.numpy())).double()
        pre, mass, y, act_y = linear_reference(U.rounded(x.double(), type_), U.rounded(w.double(), type_), None, "gelu", r.double())
        U.assert_close(got, y, linear_error(40, mass, pre, act_y, y, "f32", "gelu") + U24 * y.abs())
        assert lin.Apply(x.numpy()[:0]).shape == (0, 33)


@pytest.mark.parametrize("type_", ["bf16", "mx8"])
def test_offsets_beyond_32_bits(amlike_device, type_):
    """Rows 2^30 elements apart: byte offsets pass 32 bits for every operand."""
    rows, k, n, ld = 5, 160, 96, 1 << 30
    x, w = torch.randint(-4, 5, (rows, k), generator=gen(51)).double(), torch.randint(-4, 5, (n, k), generator=gen(52)).double()
    dt = torch.uint8 if type_ == "mx8" else torch.bfloat16
    bx = torch.empty(((rows - 1) * ld + k,), dtype=dt, device="cuda")
    bo = torch.empty(((rows - 1) * ld + n,), dtype=torch.bfloat16, device="cuda")
    small = U.DeviceMatrix(rows, k, type_, fill=x)
    for i in range(rows):
        bx[i * ld:i * ld + k] = small.buf[i]
    mx = dense.Matrix(bx.data_ptr(), type_, ld, small.scales.data_ptr() if type_ == "mx8" else 0, small.ld_scales if type_ == "mx8" else 0)
    lin = dense.Linear(w.numpy(), None, type_)
    mo = dense.Matrix(bo.data_ptr(), "bf16", ld)
    lin.ApplyDevice(mx, rows, mo)
    got = torch.stack([bo[i * ld:i * ld + n] for i in range(rows)]).cpu().double()
    assert torch.equal(got, (x @ w.t()).bfloat16().double())
    norm = dense.RmsNorm(n)
    y = U.DeviceMatrix(rows, n, "f32")
    norm.ApplyDevice(mo, rows, y.m, sum=mo)
    torch.cuda.synchronize()
    s, want = norm_reference(got, None, None, float(np.float32(1e-5)))
    U.check_output(y, want, norm_error(s, want))


# ---- the operators together ------------------------------------------------------------------------------

class Block:
    """x += W2 gelu(W1 norm(x + r)): the residual block they are made for, in 8 bits inside."""

    def __init__(self, rows, dim, wide, seed):
        self.rows, self.dim, self.wide = rows, dim, wide
        self.w1, self.w2 = U.rounded(randn(wide, dim, seed) / math.sqrt(dim), "mx8"), U.rounded(randn(dim, wide, seed + 1) / math.sqrt(wide), "mx8")
        self.b1, self.g = randn(1, wide, seed + 2)[0].float().double(), (1 + 0.1 * randn(1, dim, seed + 3)[0]).float().double()
        self.norm = dense.RmsNorm(dim, self.g.numpy(), 1e-5)
        self.l1, self.l2 = dense.Linear(self.w1.numpy(), self.b1.numpy(), "mx8"), dense.Linear(self.w2.numpy(), None, "mx8")
        self.x, self.r, self.s = (U.DeviceMatrix(rows, dim, "bf16") for _ in range(3))
        self.q, self.h, self.y = U.DeviceMatrix(rows, dim, "mx8"), U.DeviceMatrix(rows, wide, "mx8"), U.DeviceMatrix(rows, dim, "bf16")

    def fill(self, seed):
        for i, m in enumerate((self.x, self.r)):
            m.buf[:self.rows] = randn(self.rows, self.dim, seed + i).bfloat16().cuda()

    def run(self, stream=None):
        self.norm.ApplyDevice(self.x.m, self.rows, self.q.m, residual=self.r.m, sum=self.s.m, stream=stream)
        self.l1.ApplyDevice(self.q.m, self.rows, self.h.m, activation="gelu", stream=stream)
        self.l2.ApplyDevice(self.h.m, self.rows, self.y.m, residual=self.s.m, stream=stream)

    def check(self):
        """Each stage against what the stage before left in memory."""
        s, q = norm_reference(self.x.values(), self.r.values(), self.g, float(np.float32(1e-5)))
        U.check_output(self.s, s, U24 * s.abs())
        U.check_output(self.q, q, norm_error(s, q))
        pre, mass, y, act_y = linear_reference(self.q.values(), self.w1, self.b1, "gelu", None)
        U.check_output(self.h, y, linear_error(self.dim, mass, pre, act_y, y, "mx8", "gelu", "mx8"))
        pre, mass, y, act_y = linear_reference(self.h.values(), self.w2, None, "none", self.s.values())
        U.check_output(self.y, y, linear_error(self.wide, mass, pre, act_y, y, "bf16", "none", "mx8"))


@pytest.mark.parametrize("rows,dim,wide", [(1, 256, 1024), (16, 512, 2048), (77, 200, 808), (300, 384, 1536)])
def test_block(amlike_device, rows, dim, wide):
    b = Block(rows, dim, wide, 60)
    b.fill(70)
    torch.cuda.synchronize()
    b.run()
    torch.cuda.synchronize()
    b.check()
    # and as a whole against the same network in 64 bits: 8-bit roundings of 2^-4 in q, h and nothing
    # else of note give a relative error of about sqrt(2) * 2^-4 / sqrt(3) on the branch
    s, q = norm_reference(b.x.values(), b.r.values(), b.g, 1e-5)
    branch = ACT["gelu"](q @ b.w1.t() + b.b1) @ b.w2.t()
    off = b.y.values() - (s + branch)
    assert float(off.norm() / branch.norm()) < 2.0 ** -4


@pytest.mark.parametrize("rows", [1, 16, 300])
def test_block_in_a_graph(amlike_device, rows):
    """Recorded once, replayed with other inputs, eager work between the replays; two graphs of
    the same handles replayed on two streams at once."""
    blocks = [Block(rows, 256, 512, 80) for _ in range(2)]
    blocks[1].norm, blocks[1].l1, blocks[1].l2 = blocks[0].norm, blocks[0].l1, blocks[0].l2
    graphs = []
    for b in blocks:
        b.fill(1)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            b.run(torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(4):
        for i, b in enumerate(blocks):
            b.fill(100 + 10 * turn + i)
            b.y.buf.fill_(0)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        got = [b.y.buf[:rows].clone() for b in blocks]
        for b, y in zip(blocks, got):
            b.run()
            torch.cuda.synchronize()
            assert torch.equal(b.y.buf[:rows], y)
            b.check()


def test_two_threads_on_two_streams_of_one_handle(amlike_device):
    w = (randn(320, 200, 90) / 14).numpy()
    lin, norm = dense.Linear(w, None, "bf16"), dense.RmsNorm(320)
    results, errors = {}, []

    def work(i):
        try:
            st = torch.cuda.Stream()
            x = U.DeviceMatrix(90 + i, 200, "bf16", fill=randn(90 + i, 200, 91 + i))
            mid, out = U.DeviceMatrix(90 + i, 320, "bf16"), U.DeviceMatrix(90 + i, 320, "mx8")
            torch.cuda.synchronize()
            seen = []
            for _ in range(20):
                lin.ApplyDevice(x.m, 90 + i, mid.m, activation="silu", stream=st.cuda_stream)
                norm.ApplyDevice(mid.m, 90 + i, out.m, stream=st.cuda_stream)
                st.synchronize()
                seen.append((mid.values(), out.values()))
            assert all(torch.equal(a, seen[0][0]) and torch.equal(b, seen[0][1]) for a, b in seen)
            results[i] = (x.values(), seen[0][0])
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    wr = U.rounded(torch.from_numpy(w).float().double(), "bf16")
    for x, y in results.values():
        pre, mass, want, act_y = linear_reference(x, wr, None, "silu", None)
        e = linear_error(200, mass, pre, act_y, want, "bf16", "silu")
        U.assert_close(y, want, e + (want.abs() + e) * 2.0 ** -8)


# ---- refusals that need a handle ---------------------------------------------------------------------------

def refused(fn, code=_lib.EINVAL, text=None):
    with pytest.raises(_lib.AmlikeError) as e:
        fn()
    assert e.value.code == code and (text is None or text in str(e.value)), str(e.value)


def test_refusals(amlike_device):
    x, o = U.DeviceMatrix(4, 64, "bf16"), U.DeviceMatrix(4, 96, "bf16")
    lin, norm = dense.Linear(np.ones((96, 64), np.float32), None, "bf16"), dense.RmsNorm(64)
    M = dense.Matrix
    refused(lambda: lin.ApplyDevice(x.m, -1, o.m))
    refused(lambda: lin.ApplyDevice(M(x.buf.data_ptr(), "f16", 64), 4, o.m), text="type")
    refused(lambda: lin.ApplyDevice(M(x.buf.data_ptr(), "bf16", 63), 4, o.m), text="stride")
    refused(lambda: lin.ApplyDevice(M(x.buf.data_ptr() + 1, "bf16", 64), 4, o.m), text="aligned")
    refused(lambda: lin.ApplyDevice(M(0, "bf16", 64), 4, o.m))
    refused(lambda: lin.ApplyDevice(x.m, 4, M(o.buf.data_ptr(), "mx8", 96)), text="scales")
    refused(lambda: lin.ApplyDevice(x.m, 4, M(x.buf.data_ptr(), "bf16", 96)), text="overlap")
    refused(lambda: lin.ApplyDevice(x.m, 4, o.m, residual=M(o.buf.data_ptr() + 2, "bf16", 96)), text="overlap")
    refused(lambda: lin.ApplyDevice(x.m, 4, o.m, residual=M(x.buf.data_ptr(), "mx8", 96, x.buf.data_ptr(), 3)))
    assert _lib.lib().amlike_linear_apply_dev(lin._h, x.m.ref, 4, 6, None, o.m.ref, None) == _lib.EINVAL
    assert _lib.lib().amlike_linear_apply_dev(None, x.m.ref, 4, 0, None, o.m.ref, None) == _lib.EINVAL
    assert _lib.lib().amlike_norm_apply_dev(None, x.m.ref, None, 4, None, x.m.ref, None) == _lib.EINVAL
    y = U.DeviceMatrix(4, 64, "bf16")
    refused(lambda: norm.ApplyDevice(x.m, 4, y.m, residual=M(y.buf.data_ptr(), "f16", 64)), text="type")
    refused(lambda: norm.ApplyDevice(x.m, 4, y.m, sum=y.m), text="overlap")
    refused(lambda: norm.ApplyDevice(x.m, 4, M(x.buf.data_ptr(), "f32", 64)), text="overlap")
    refused(lambda: norm.ApplyDevice(M(x.buf.data_ptr(), "mx8", 64, x.buf.data_ptr(), 2), 4, y.m))
    lin.ApplyDevice(x.m, 0, o.m)
    norm.ApplyDevice(x.m, 0, y.m)
    dense.ConvertDevice(x.m, 0, 64, y.m)
    torch.cuda.synchronize()
    for m in (o, y):
        m.assert_rest_untouched()
        assert (m.buf.view(torch.uint8) == 0xFF).all()


def test_weights_that_do_not_fit(amlike_device):
    w = np.ones((3, 40), np.float32)
    for bad, types in ((np.nan, ("bf16", "f16", "mx8")), (np.inf, ("bf16", "f16", "mx8")), (7e4, ("f16",))):
        w[1, 39] = bad
        for t in types:
            refused(lambda t=t: dense.Linear(w, None, t), _lib.ENONFINITE, "not finite")
    w[1, 39] = 7e4
    dense.Linear(w, None, "bf16").close()
    refused(lambda: dense.Linear(w, np.array([0, np.nan, 0], np.float32), "bf16"), _lib.ENONFINITE, "bias")
