"""Digits of the feature operators: sums, intermediate values and activations
at the sizes and values where they could be lost.

Tolerances are bounds on roundings, counted as in test_features_gpu: u = 2^-23
for an fp32 operation (the tensor core truncates its sums), h = eps(dtype) / 2
for the one rounding to the output's type.
"""

import math

import pytest
import torch

from dsl_splat_b200 import features
from test_features_gpu import (ACTS, DTYPES, U, check, draws, half_step, smallest,
                               value_and_slope)

pytestmark = pytest.mark.gpu
HALF = (torch.bfloat16, torch.float16)


# ---- dz = dy act'(z) between the products of the backward ------------------------

# the one-pass kernels (16-byte rows, other rows), the products (16-byte rows,
# other rows of few and of many), on either side of 64 and 128 features
DZ_SIZES = [(300, 64, 64), (700, 128, 128), (5000, 32, 24), (300, 35, 64), (513, 33, 25),
            (700, 100, 72), (400, 127, 101), (520, 264, 200), (400, 300, 17), (300, 17, 300),
            (333, 301, 201), (17000, 301, 33), (16500, 136, 200), (9000, 512, 512)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid", "relu"])
@pytest.mark.parametrize("m, k, n", DZ_SIZES)
def test_gradients_round_once(m, k, n, act, dtype):
    """dx and dW of 16-bit types are off by their own rounding and little else:
    dz is kept as two values of the type, h^2 relative (and half the type's
    smallest value) off."""
    normal = draws(41)
    x, w, b = (normal(*s, dtype=dtype) for s in ((m, k), (n, k), (n,)))
    w = w / 16
    dy = normal(m, n, dtype=dtype)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = features.linear(*leaves, activation=act)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    xd, wd, dyd = (t.detach().double() for t in (x, w, dy))
    z = xd @ wd.t() + b.detach().double()
    e_z = (k + 8) * U * (xd.abs() @ wd.abs().t() + b.detach().double().abs())
    _, rate = value_and_slope(z, act)
    dz = dyd * rate
    # the slope: 16 u of its terms and its argument's error; for GELU 2^-15 more,
    # half (the largest tail) of the 2^-14 that the tails of 16-bit types may be off
    e_dz = dyd.abs() * (1.2 * e_z + 16 * U * (1 + z.abs()) + 2.0 ** -15 * (act == "gelu"))
    if act == "relu":
        e_dz = dyd.abs() * ((z.abs() <= e_z).double() + U)
    e_dz = e_dz + half_step(dtype) ** 2 * (dz.abs() + e_dz) + smallest(dtype)
    # a product's sums truncate at most once for 16 terms of each of two parts
    check(dx, dz @ wd, (n / 8 + 16) * U * (dz.abs() @ wd.abs()) + e_dz @ wd.abs(), "dx")
    check(dw, dz.t() @ xd, (min(m, 8192) / 8 + 16) * U * (dz.abs().t() @ xd.abs())
          + e_dz.t() @ xd.abs(), "dw")


def test_gradients_beyond_the_types_range():
    """act' is up to 1.13: a dz above fp16's largest value does not spoil what
    is formed from it."""
    for k, n in ((64, 64), (35, 20), (264, 200), (301, 37)):
        x = torch.zeros(256, k, device="cuda", dtype=torch.float16)
        x[:, 0] = 1.5
        w = torch.zeros(n, k, device="cuda", dtype=torch.float16)
        w[:, 0] = 1.0
        w[:, 1] = 2.0 ** -10
        dy = torch.zeros(256, n, device="cuda", dtype=torch.float16)
        dy[:, 3] = 65504.0
        x.requires_grad_()
        y = features.linear(x, w, activation="gelu")
        dx, = torch.autograd.grad(y, x, dy)
        _, rate = value_and_slope(torch.tensor(1.5, dtype=torch.float64), "gelu")
        want = 65504.0 * float(rate) * 2.0 ** -10
        assert float(rate) > 1.1
        # its own rounding, and that of the second part: 4 of 73857
        assert ((dx[:, 1].double() - want).abs() <= (2.0 ** -11 + 2.0 ** -13) * want).all()


@pytest.mark.parametrize("k, n", [(64, 64), (35, 20), (264, 200), (301, 37)])
@pytest.mark.parametrize("dtype", HALF)
def test_infinite_gradients_stay_infinite(k, n, dtype):
    """An infinite dy gives infinities, as the one value dz would, and spoils
    no other row."""
    normal = draws(42)
    x, w, dy = (normal(*s, dtype=dtype) for s in ((300, k), (n, k), (300, n)))
    w = w.abs() + 0.25
    x.requires_grad_()

    def run(dy):
        y = features.linear(x, w, activation="sigmoid")
        return torch.autograd.grad(y, x, dy)[0]

    clean = run(dy)
    dy = dy.clone()
    dy[130, 1] = float("inf")
    x.data[130] = 0.01
    spoilt = run(dy)
    keep = torch.arange(300, device="cuda") != 130
    assert torch.equal(spoilt[keep], clean[keep])
    assert (spoilt[130] == float("inf")).all()

# ---- group norm of samples whose first row is unlike the rest ---------------------

def norm_exact(x, groups):
    b, s, c = x.shape
    X = x.double().reshape(b, s, groups, -1)
    mean = X.mean((1, 3), keepdim=True)
    var = (X - mean).square().mean((1, 3), keepdim=True)
    return X, mean, var


NORM_FIRST = [(1, 40 * 50, 32, 8), (2, 67 * 101, 48, 4), (1, 300 * 300, 32, 8),
              (1, 301 * 211, 35, 5), (3, 250 * 260, 16, 16), (1, 500 * 400, 64, 16),
              (2, 90 * 90, 600, 1), (1, 800, 2050, 2), (64, 170 * 170, 32, 8), (1, 7, 3, 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("apart", [30.0, 300.0, 3000.0])
@pytest.mark.parametrize("b, s, c, groups", NORM_FIRST)
def test_group_norm_first_row_unlike_the_rest(b, s, c, groups, apart, dtype):
    """An empty corner of an image of far features.  The variance is joined
    from sums of squares of one sign about means that lie among the values:
    chains of at most 64 additions of them, each half of u, and four times
    that for the moving mean; y is off by half of its relative error."""
    normal = draws(45)
    x = normal(b, s, c, dtype=dtype, shift=apart)
    x[:, 0] = 0
    dy = normal(b, s, c, dtype=dtype)
    x.requires_grad_()
    y = features.group_norm(x, groups, spatial_dims=1)
    dx, = torch.autograd.grad(y, x, dy)
    X, mean, var = norm_exact(x.detach(), groups)
    rstd = (var + 1e-5).rsqrt()
    e_rstd = 128 * U * rstd  # relative: half of 256 u
    # the mean is kept as an fp32 value, and formed from fp32 differences to the
    # first row and to each other
    e_mean = U * mean.abs() + U * (X[:, :1] - mean).abs().mean(3, keepdim=True) \
        + 64 * U * var.sqrt()
    hat = (X - mean) * rstd
    e_hat = (e_mean + U * (X - mean).abs()) * rstd + (X - mean).abs() * e_rstd + 4 * U * hat.abs()
    check(y.detach(), hat.reshape(x.shape), e_hat.reshape(x.shape), "y")
    D = dy.double().reshape(X.shape)

    def avg(v):
        return v.mean((1, 3), keepdim=True)

    m1, m2 = avg(D), avg(D * hat)
    e_m2 = avg(D.abs() * e_hat) + 520 * U * avg((D * hat).abs())
    inner = D - m1 - hat * m2
    e_inner = (520 * U * avg(D.abs()) + e_hat * m2.abs() + hat.abs() * e_m2
               + 4 * U * (D.abs() + m1.abs() + (hat * m2).abs()))
    check(dx, (rstd * inner).reshape(x.shape),
          (rstd * e_inner + e_rstd * inner.abs()).reshape(x.shape), "dx")


def test_group_norm_halves_apart():
    """Values on two sides of a step: no row stands for all."""
    for s, c in ((5000, 8), (400_000, 32)):
        normal = draws(46)
        x = normal(1, s, c, dtype=torch.float32)
        x[:, s // 3:] += 1000.0
        y = features.group_norm(x, 2, spatial_dims=1)
        X, mean, var = norm_exact(x, 2)
        hat = (X - mean) * (var + 1e-5).rsqrt()
        check(y, hat.reshape(x.shape), (200 * U * (hat.abs() + 1)).reshape(x.shape), "y")

# ---- long sums -------------------------------------------------------------------

@pytest.mark.parametrize("rows, k, n, power", [(200_000_000, 8, 8, -13), (200_000_000, 9, 7, -13),
                                               (800_000, 2048, 2048, -5)])
def test_weight_gradient_over_many_rows(rows, k, n, power):
    """fp16: an accumulator of dW takes 1024 additions at most (u each), and
    what it holds is added up in fp32: 64 additions in a chain (u / 2 each).
    The sum lies just above a value of fp16 whose step is 2^-10 of it, so that
    a bias of half a step shows."""
    x = torch.full((rows, k), 1285 / 1024, device="cuda", dtype=torch.float16)
    dy = torch.full((rows, n), 2.0 ** power * 1105 / 1024, device="cuda", dtype=torch.float16)
    value = float(x[0, 0]) * float(dy[0, 0])
    used = math.ceil(32800 / value)
    assert used <= rows
    x, dy = x[:used], dy[:used]
    w = torch.zeros(n, k, device="cuda", dtype=torch.float16, requires_grad=True)
    y = features.linear(x, w)
    dw, = torch.autograd.grad(y, w, dy)
    want = torch.full((n, k), used * value, device="cuda", dtype=torch.float64)
    check(dw, want, (1024 + 32) * U * want, "dw")


# ---- whole numbers -----------------------------------------------------------------

EXACT_SIZES = [(120001, 64, 64), (70001, 35, 64), (50000, 128, 128), (40000, 100, 72),
               (30001, 96, 128), (60000, 33, 20), (50001, 40, 3), (4096, 256, 256),
               (17001, 300, 17), (20000, 129, 130), (18000, 520, 137), (200001, 8, 8),
               (9000, 16, 200), (1, 3, 5), (129, 64, 32)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["none", "relu"])
@pytest.mark.parametrize("m, k, n", EXACT_SIZES)
def test_linear_whole_numbers(m, k, n, act, dtype):
    """Small whole numbers: every sum is one of fp32's, so each result is the
    exact sum rounded once, to the bit; a tile that is lost, doubled or stale
    changes it."""
    g = torch.Generator().manual_seed(44)

    def whole(*shape, most):
        return torch.randint(-most, most + 1, shape, generator=g).to(dtype).cuda()

    x, w, b = whole(m, k, most=3), whole(n, k, most=1), whole(n, most=2)
    dy, r = whole(m, n, most=2), whole(m, n, most=3)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = features.linear(x, w, b, residual=r, activation=act)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    xd, wd, dyd = (t.detach().double() for t in (x, w, dy))
    z = xd @ wd.t() + b.detach().double()
    value, rate = value_and_slope(z, act)
    dz = dyd * rate
    for name, got, want in (("y", y, value + r.double()), ("dx", dx, dz @ wd),
                            ("dw", dw, dz.t() @ xd), ("db", db, dz.sum(0))):
        assert want.abs().max() < 2 ** 24, name
        assert torch.equal(got.detach(), want.to(dtype)), name

@pytest.mark.parametrize("m, k, n", [(130, 1100, 40), (130, 5003, 33), (64, 16384, 24),
                                     (40, 65535, 9), (20, 20001, 200),
                                     (16400, 1100, 140)])
@pytest.mark.parametrize("act", ["none", "sigmoid"])
def test_linear_long_rows_of_one_sign(m, k, n, act):
    """fp32: an accumulator sums 512 inputs in 32 truncating additions (48 u
    with those within a product), the rest is added in fp32 (u / 2 each)."""
    g = torch.Generator().manual_seed(43)
    x = (0.5 + torch.rand(m, k, generator=g)).cuda()
    w = ((0.5 + torch.rand(n, k, generator=g)) / k).cuda()
    r = torch.randn(m, n, generator=g).cuda()
    b = torch.randn(n, generator=g).cuda()
    z = x.double() @ w.double().t()
    e_z = (48 + k / 1024) * U * z + 2 * U * b.double().abs()
    z = z + b.double()
    value, rate = value_and_slope(z, act)
    x.requires_grad_()
    y = features.linear(x, w, b, residual=r, activation=act)
    want = value + r.double()
    check(y.detach(), want, e_z + 16 * U * value.abs() + U * want.abs(), "y")
    # dx = dy act'(z) w: z is formed again
    dy = torch.zeros(m, n, device="cuda")
    dy[:, 1] = 1.0
    dx, = torch.autograd.grad(y, x, dy)
    want = rate[:, 1:2] * w.double()[1]
    check(dx, want, (rate[:, 1:2] * 20 * U + e_z[:, 1:2]) * w.double()[1], "dx")

# ---- activations at large arguments ------------------------------------------------

def through(z, act, dtype):
    """act and its slope of the values z through a layer of weight 1, whose
    products and sums are exact."""
    x = z.to(dtype).cuda().reshape(-1, 1).requires_grad_()
    w = torch.ones(1, 1, device="cuda", dtype=dtype)
    y = features.linear(x, w, activation=act)
    slope, = torch.autograd.grad(y, x, torch.ones_like(y))
    return x.detach().double(), y.detach(), slope


def exact_activation(z, act):
    """Value and slope without cancellation, and the slope's terms."""
    if act == "gelu":
        c = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        d = z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * c, c + d, c + d.abs()
    s, t = torch.special.expit(z), torch.special.expit(-z)
    if act == "silu":
        return z * s, s + z * s * t, s + (z * s * t).abs()
    return s, s * t, s * t


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
def test_activations_keep_their_digits(act):
    """fp32: 16 u of the value itself, however small (and the smallest normal
    value's step)."""
    most = 13.0 if act == "gelu" else 86.0
    z = torch.cat([torch.linspace(-most, most, 20001), torch.linspace(-1, 1, 4001),
                   torch.tensor([0.0, -0.0, 1e-20, -1e-20, 200.0, 1e30])])
    z, y, slope = through(z, act, torch.float32)
    value, rate, terms = exact_activation(z, act)
    rate = torch.where(z > 100, rate.nan_to_num(), rate)
    check(y, value, 16 * U * value.abs() + 2.0 ** -126, "y")
    check(slope, rate, 16 * U * terms.nan_to_num() + 2.0 ** -126, "slope")


@pytest.mark.parametrize("act", ["silu", "sigmoid"])
def test_activations_below_the_normal_range(act):
    """e^z below 2^-126 is not taken for 0."""
    z, y, _ = through(torch.linspace(-95, -86, 901), act, torch.float32)
    value, _, _ = exact_activation(z, act)
    check(y, value, 16 * U * value.abs() + 16 * 2.0 ** -149 * (1 + z.abs()), "y")


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
def test_activations_of_short_types(act, dtype):
    """2^-13 relative where the type's own step is 2^-8 or 2^-11."""
    most = 12.0 if act == "gelu" else 80.0
    z, y, slope = through(torch.linspace(-most, most, 60001), act, dtype)
    value, rate, terms = exact_activation(z, act)
    check(y, value, 2.0 ** -13 * value.abs(), "y")
    check(slope, rate, 2.0 ** -13 * terms, "slope")


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
def test_group_norm_activations_keep_their_digits(act):
    """The same through group norm: one group of -1 and 1, scaled by the
    weights."""
    c = 512
    x = torch.ones(1, 2, 2, c, device="cuda")
    x[:, :, 1] = -1.0
    w = torch.linspace(0.0, 12.0, c, device="cuda")
    y = features.group_norm(x, 1, w, eps=2.0 ** -40, activation=act)
    # hat is +-1 to 2^-40; z = hat w, 4 u
    z = (x.double() * w.double())
    value, _, terms = exact_activation(z, act)
    # an argument off by 4 u |z| changes the tails by 4 u z^2 of themselves
    check(y, value, (16 + 4 * z.abs() + 4 * z * z) * U * value.abs() + 2.0 ** -126, "y")


@pytest.mark.parametrize("k", [16384, 20000, 40008, 65535])
@pytest.mark.parametrize("n", [1, 33, 200])
def test_short_types_over_long_rows(k, n):
    """fp16: the tensor core cuts what an addition leaves below the step of its
    accumulator.  One large product first and then sums of 1.9 steps each lose
    nine tenths of a step an addition; 1024 additions (u each) at most lie in
    one accumulator, the rest is added in fp32."""
    x = torch.full((130, k), 2.0 ** -13, device="cuda", dtype=torch.float16)
    w = torch.full((n, k), 1.9 * 2.0 ** -14, device="cuda", dtype=torch.float16)
    x[:, 0] = 1.0
    w[:, 0] = 1.0
    want = x.double() @ w.double().t()
    tolerance = (1024 + 16) * U * want
    check(features.linear(x, w), want, tolerance, "y")
    residual = torch.ones_like(want, dtype=torch.float16)
    check(features.linear(x, w, residual=residual), want + 1, tolerance + U * (want + 1),
          "y + residual")
    # dx of a layer with so many outputs, and z in its gradient, are such sums too
    leaf = w[:, :1].new_zeros(130, n).requires_grad_()
    dx, = torch.autograd.grad(features.linear(leaf, w.t()), leaf, x)
    check(dx, want, tolerance, "dx")
    x.requires_grad_()
    y = features.linear(x, w, activation="sigmoid")
    dy = torch.zeros_like(y)
    dy[:, 0] = 1.0
    dx, = torch.autograd.grad(y, x, dy)
    s = torch.sigmoid(want)
    check(y.detach(), s, tolerance + 16 * U, "sigmoid")
    rate = (s * (1 - s))[:, :1]
    check(dx, rate * w.double()[0], (tolerance[:, :1] + 2.0 ** -13 * rate) * w.double()[0], "dx")


def test_short_types_over_long_rows_of_two_parts():
    """The same for dx where dz is two values: 512 additions of each."""
    n = 65535
    dy = torch.full((64, n), 2.0 ** -13, device="cuda", dtype=torch.bfloat16)
    x = torch.zeros(64, 40, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.rand(n, 40, generator=torch.Generator().manual_seed(47)).to(torch.bfloat16).cuda()
    dx, = torch.autograd.grad(features.linear(x, w, activation="sigmoid"), x, dy)
    want = dy.double() @ w.double() / 4  # the slope at 0
    check(dx, want, (1024 + 16 + 16) * U * want, "dx")


# ---- the ends of fp32's range ------------------------------------------------------

@pytest.mark.parametrize("m, k, n", [(70, 35, 20), (200, 64, 64), (300, 300, 200),
                                     (17000, 300, 140)])
def test_largest_and_infinite_fp32_values(m, k, n):
    """Values that round to more than bf16's largest are split like others, and
    an infinity gives what IEEE arithmetic gives."""
    normal = draws(48)
    x, w = normal(m, k, dtype=torch.float32), normal(n, k, dtype=torch.float32)
    dy = normal(m, n, dtype=torch.float32)
    most = torch.finfo(torch.float32).max
    w = w * 2.0 ** -12
    x[3] = 0.0
    x[3, 5] = most
    x[4, 1] = float("inf")
    x[5, 2] = -float("inf")
    x[6, 3], x[6, 4] = float("inf"), -float("inf")
    x.requires_grad_()
    y = features.linear(x, w)
    want = x.double() @ w.double().t()
    fine = want.isfinite()
    check(y[fine].detach(), want[fine].detach(),
          (k + 8) * U * (x.detach().nan_to_num(0, 0, 0).double().abs() @ w.double().abs().t())[fine],
          "y")
    for row in (4, 5, 6):
        assert torch.equal(y[row].isnan(), want[row].float().isnan())
        assert torch.equal(y[row].nan_to_num(0.0), want[row].float().nan_to_num(0.0))
    # dy: its products with w, and (by way of dW) with x
    dy[3] = 0.0
    dy[3, 7] = most
    dy[9, 2] = float("inf")
    dx, = torch.autograd.grad(y, x, dy)
    want = dy.double() @ w.double()
    fine = want.isfinite()
    check(dx[fine], want[fine], (n + 8) * U * (dy.nan_to_num(0, 0, 0).double().abs()
                                               @ w.double().abs())[fine], "dx")
    assert torch.equal(dx[9], want[9].float())


def test_training_over_more_rows_than_an_int():
    """2^31 + 2^20 rows of one value, in many more blocks than are resident: sums
    of powers of two are exact until they are rounded."""
    rows = (1 << 31) + (1 << 20)
    x = torch.ones(rows, 1, device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(1, 1, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    b = torch.zeros(1, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = features.linear(x, w, b, activation="sigmoid")
    dw, db = torch.autograd.grad(y, (w, b), torch.full_like(y, 2.0 ** -20))
    want = torch.tensor(rows * 2.0 ** -22, dtype=torch.float64).to(torch.bfloat16)
    assert float(dw) == float(want) and float(db) == float(want)
