"""Feature operators on the GPU against their definitions in 64 bits.

Tolerances are bounds on the rounding of each value, not measured figures.
With u = 2^-23 for each fp32 operation (sums may truncate, hence twice half a
step) and h = eps(dtype) / 2 for the one rounding to the output's type:

* a sum of n products is off by at most (n + 8) u times the sum of the
  products' magnitudes;
* an activation and its slope, 16 u relative, and what their argument is off
  by times their Lipschitz constants (both at most 1.2);
* 16-bit types take dz = dy act'(z) in their own type: half a step relative
  (and half their smallest value) of each dz, besides the above, in dx and dW;
  db is summed from dz before that.
"""

import math

import pytest
import torch

from dsl_splat_b200 import features

pytestmark = pytest.mark.gpu

U = 2.0 ** -23
ACTS = ("none", "relu", "silu", "gelu", "sigmoid")
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    # values below the type's normal range round to multiples of its smallest
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def value_and_slope(z, act):
    if act == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        c = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "sigmoid":
        s = torch.sigmoid(z)
        return s, s * (1 - s)
    return z, torch.ones_like(z)


def check(got, want, tolerance, name):
    assert got.shape == want.shape, name
    rounded = half_step(got.dtype) * (want.abs() + tolerance) + smallest(got.dtype)
    off = (got.double() - want).abs()
    bad = ~(off <= tolerance + rounded)
    if bad.any():
        i = int(bad.flatten().nonzero()[0])
        pytest.fail(f"{name}: {int(bad.sum())} of {bad.numel()} values; value {i}: "
                    f"{float(got.flatten()[i])} against {float(want.flatten()[i])}")


def draws(seed):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape, dtype, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=g) * scale + shift).to(dtype).cuda()

    return normal


# ---- linear ------------------------------------------------------------------

def check_linear(x, w, b, r, act, y, grads=None, dy=None):
    """y and (dx, dw, db) of rows x against the formulas."""
    xd, wd = x.double(), w.double()
    bd = torch.zeros(len(w), dtype=torch.float64, device=x.device) if b is None else b.double()
    k, n, m = x.shape[1], len(w), len(x)
    z = xd @ wd.t() + bd
    e_z = (k + 8) * U * (xd.abs() @ wd.abs().t() + bd.abs())
    value, rate = value_and_slope(z, act)
    e_value = 1.2 * e_z + 16 * U * value.abs() + 1e-30
    if r is not None:
        value = value + r.double()
        e_value = e_value + U * value.abs()
    check(y, value, e_value, "y")
    if grads is None:
        return
    dyd = dy.double()
    dz = dyd * rate
    e_dz = dyd.abs() * (1.2 * e_z + 16 * U * (1 + z.abs()))
    if act == "none":
        e_dz = dyd.abs() * U
    if act == "relu":  # the slope jumps where z is within its own error of 0
        e_dz = dyd.abs() * ((z.abs() <= e_z).double() + U)
    e_sum = e_dz  # db is summed from dz before its rounding
    if x.dtype != torch.float32:
        e_dz = e_dz + half_step(x.dtype) * (dz.abs() + e_dz) + smallest(x.dtype)
    dx, dw, db = grads
    if dx is not None:
        check(dx, dz @ wd, (n + 8) * U * (dz.abs() @ wd.abs()) + e_dz @ wd.abs(), "dx")
    if dw is not None:
        check(dw, dz.t() @ xd, (m + 8) * U * (dz.abs().t() @ xd.abs()) + e_dz.t() @ xd.abs(),
              "dw")
    if db is not None:
        check(db, dz.sum(0), (m + 8) * U * dz.abs().sum(0) + e_sum.sum(0), "db")


def linear_case(m, k, n, dtype, act, bias=True, residual=False, seed=0):
    normal = draws(seed)
    x = normal(m, k, dtype=dtype)
    w = normal(n, k, dtype=dtype, scale=1 / math.sqrt(k))
    b = normal(n, dtype=dtype) if bias else None
    r = normal(m, n, dtype=dtype) if residual else None
    leaves = [t.requires_grad_() for t in (x, w, b, r) if t is not None]
    y = features.linear(x, w, b, residual=r, activation=act)
    dy = normal(m, n, dtype=dtype)
    grads = iter(torch.autograd.grad(y, leaves, dy))
    dx, dw = next(grads), next(grads)
    db = next(grads) if bias else None
    if residual:
        assert torch.equal(next(grads), dy)
    check_linear(x.detach(), w.detach(), b if b is None else b.detach(),
                 r if r is None else r.detach(), act, y.detach(), (dx, dw, db), dy)


SIZES = [(1, 1, 1), (1, 32, 3), (2, 3, 5), (7, 35, 64), (127, 64, 64), (128, 64, 64),
         (129, 32, 16), (300, 48, 72), (513, 100, 31), (257, 129, 130), (140, 256, 256),
         (200, 300, 17), (65, 17, 300), (33, 520, 264), (5000, 64, 32), (1000, 8, 512)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, k, n", SIZES)
def test_linear_sizes(m, k, n, dtype):
    linear_case(m, k, n, dtype, "silu", residual=True)


# rows enough for several tiles of a block, and for operands laid out before
# the products (16384): aligned and odd widths on either side of 64, 128 and 256
MANY_ROWS = [(1024, 300, 17), (1500, 35, 300), (2001, 129, 130), (1300, 520, 264),
             (1100, 264, 520), (50001, 40, 3), (60000, 33, 20), (120001, 64, 64),
             (70001, 35, 64), (70000, 64, 35), (50000, 128, 128), (40000, 100, 72),
             (30001, 96, 128), (4096, 256, 256), (9000, 16, 200), (17001, 300, 17),
             (16384, 35, 300), (20000, 129, 130), (16500, 264, 200), (18000, 520, 137)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, k, n", MANY_ROWS)
def test_linear_many_rows(m, k, n, dtype):
    linear_case(m, k, n, dtype, "gelu", residual=True, seed=20)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, k, n", [(3000, 300, 200), (3000, 301, 37), (70000, 48, 32),
                                     (20000, 300, 200), (20000, 301, 37)])
def test_linear_many_rows_without_activation(m, k, n, dtype):
    linear_case(m, k, n, dtype, "none", seed=21)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k, n", [(68, 17), (128, 32), (100, 64), (185, 24), (35, 24)])
def test_linear_very_many_tiles(k, n, dtype):
    """Ten tiles and more to every block, of one chunk of inputs and of several."""
    normal = draws(26)
    x, w, b = (normal(*s, dtype=dtype) for s in ((400001, k), (n, k), (n,)))
    for _ in range(3):
        y = features.linear(x, w, b, activation="sigmoid")
        check_linear(x, w, b, None, "sigmoid", y)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_very_wide(dtype):
    """A bias of more values than a block keeps, and thousands of inputs."""
    linear_case(40, 24, 5003, dtype, "silu", seed=22)
    linear_case(40, 5003, 24, dtype, "silu", seed=23)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias, residual", [(True, False), (False, True), (False, False)])
def test_linear_activations(act, bias, residual, dtype):
    linear_case(333, 40, 24, dtype, act, bias, residual, seed=1)
    linear_case(70, 33, 25, dtype, act, bias, residual, seed=2)
    linear_case(150, 264, 200, dtype, act, bias, residual, seed=3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_single_gradients(dtype):
    normal = draws(4)
    x, w, b = (normal(*s, dtype=dtype) for s in ((200, 24), (40, 24), (40,)))
    dy = normal(200, 40, dtype=dtype)
    for which in range(3):
        leaves = [t.detach().clone() for t in (x, w, b)]
        leaves[which].requires_grad_()
        y = features.linear(*leaves, activation="gelu")
        grads = [None] * 3
        grads[which], = torch.autograd.grad(y, leaves[which], dy)
        check_linear(x, w, b, None, "gelu", y.detach(), grads, dy)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, k, n", [(1200, 24, 40), (1200, 300, 200), (1200, 301, 33),
                                     (17000, 301, 33)])
def test_linear_any_subset_of_gradients(m, k, n, dtype):
    """Each subset's gradients are those of the whole set."""
    normal = draws(24)
    tensors = [normal(*s, dtype=dtype) for s in ((m, k), (n, k), (n,), (m, n))]
    dy = normal(m, n, dtype=dtype)

    def grads(which):
        leaves = [t.detach().clone().requires_grad_(i in which) for i, t in enumerate(tensors)]
        y = features.linear(leaves[0], leaves[1], leaves[2], residual=leaves[3],
                            activation="silu")
        return dict(zip(which, torch.autograd.grad(y, [leaves[i] for i in which], dy)))

    whole = grads((0, 1, 2, 3))
    for which in ((0,), (1,), (2,), (3,), (0, 1), (1, 2), (0, 3)):
        for i, g in grads(which).items():
            assert torch.equal(g, whole[i])


def test_no_second_derivative():
    x = torch.ones(4, 8, device="cuda", requires_grad=True)
    w = torch.ones(8, 8, device="cuda", requires_grad=True)
    for y in (features.linear(x, w, activation="gelu"),
              features.group_norm(x, 2, spatial_dims=1)):
        g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_residual_is_the_input(dtype):
    normal = draws(25)
    x, w = normal(130, 32, dtype=dtype), normal(32, 32, dtype=dtype)
    dy = normal(130, 32, dtype=dtype)
    leaf = x.clone().requires_grad_()
    y = features.linear(leaf, w, residual=leaf, activation="silu")
    both, = torch.autograd.grad(y, leaf, dy)
    apart = [x.clone().requires_grad_() for _ in range(2)]
    y = features.linear(apart[0], w, residual=apart[1], activation="silu")
    dx, dr = torch.autograd.grad(y, apart, dy)
    assert torch.equal(both, dx + dr)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_layouts(dtype):
    """Batch dimensions, slices of wider rows, offsets, a transposed weight and
    an expanded upstream."""
    normal = draws(5)
    wide = normal(3, 5, 7, 40, dtype=dtype)
    x = wide[..., 3:38]
    w = normal(35, 12, dtype=dtype).t()
    r = normal(3, 5, 12, 7, dtype=dtype).transpose(2, 3)
    y = features.linear(x, w, residual=r, activation="silu")
    assert y.shape == (3, 5, 7, 12)
    check_linear(x.reshape(-1, 35), w, None, r.reshape(-1, 12), "silu", y.reshape(-1, 12))
    flat = normal(1 + 64 * 16, dtype=dtype)[1:].view(64, 16)  # off a 16-byte boundary
    w = normal(16, 16, dtype=dtype).requires_grad_()
    y = features.linear(flat, w)
    dw, = torch.autograd.grad(y.sum(), w)
    check_linear(flat, w.detach(), None, None, "none", y.detach(), (None, dw, None),
                 torch.ones_like(y))
    vector = features.linear(flat[0], w.detach())
    assert torch.equal(vector, features.linear(flat[:1], w.detach())[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_without_rows(dtype):
    x = torch.zeros(0, 4, 6, device="cuda", dtype=dtype, requires_grad=True)
    w = torch.ones(5, 6, device="cuda", dtype=dtype, requires_grad=True)
    b = torch.ones(5, device="cuda", dtype=dtype, requires_grad=True)
    y = features.linear(x, w, b, activation="relu")
    assert y.shape == (0, 4, 5)
    y.sum().backward()
    assert x.grad.shape == x.shape
    assert not w.grad.any() and not b.grad.any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k, n", [(32, 24), (300, 200)])
def test_linear_not_finite_rows_stay_apart(k, n, dtype):
    """A row of NaN or infinities spoils its own outputs and no others."""
    normal = draws(6)
    x, w = normal(260, k, dtype=dtype), normal(n, k, dtype=dtype)
    clean = features.linear(x, w, activation="silu")
    spoilt = x.clone()
    spoilt[17, 2] = float("nan")
    spoilt[130, 0] = float("inf")
    y = features.linear(spoilt, w, activation="silu")
    keep = torch.ones(260, dtype=torch.bool, device="cuda")
    keep[[17, 130]] = False
    assert torch.equal(y[keep], clean[keep])
    assert y[17].isnan().all() and not y[130].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_same_bits_again(dtype):
    normal = draws(7)
    x = normal(40000, 48, dtype=dtype).requires_grad_()
    w = normal(64, 48, dtype=dtype).requires_grad_()
    b = normal(64, dtype=dtype).requires_grad_()
    dy = normal(40000, 64, dtype=dtype)
    runs = []
    for _ in range(2):
        y = features.linear(x, w, b, activation="gelu")
        runs.append((y, *torch.autograd.grad(y, (x, w, b), dy)))
    assert all(torch.equal(a, c) for a, c in zip(*runs))


def test_linear_gradient_is_the_differences():
    """Central differences of a loss in the fp32 operator: a step s is off by
    s^2 times a third derivative (bounded by 2 a term here) and by the values'
    rounding over s."""
    normal = draws(8)
    x, w, b, c = (normal(*s, dtype=torch.float32) for s in ((6, 5), (4, 5), (4,), (6, 4)))

    def loss(x, w, b):
        return (features.linear(x, w, b, activation="gelu").double() * c.double()).sum()

    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    step = 2.0 ** -7
    for which, leaf in enumerate(leaves):
        at = [t.detach().clone() for t in leaves]
        for i in range(leaf.numel()):
            flat = at[which].view(-1)
            old = float(flat[i])
            flat[i] = old + step
            up = float(loss(*at))
            flat[i] = old - step
            down = float(loss(*at))
            flat[i] = old
            magnitude = float(c.abs().sum() * (1 + x.detach().abs().max() ** 3
                                               + w.detach().abs().max() ** 3))
            bound = 2 * step ** 2 * magnitude + 64 * U * magnitude / step
            assert abs((up - down) / (2 * step) - float(grads[which].view(-1)[i])) <= bound


def test_linear_long_rows():
    """Offsets past 2^31 values: the last rows of a long bf16 input."""
    rows, k, n = 34_000_000, 64, 8
    x = torch.zeros(rows, k, device="cuda", dtype=torch.bfloat16)
    normal = draws(9)
    x[-5:] = normal(5, k, dtype=torch.bfloat16)
    w = normal(n, k, dtype=torch.bfloat16)
    y = features.linear(x, w)
    check_linear(x[-5:], w, None, None, "none", y[-5:])
    assert not y[:-5].any()


def test_linear_more_rows_than_an_int():
    """2^31 + 300 rows of one value."""
    rows = (1 << 31) + 300
    x = torch.zeros(rows, 1, device="cuda", dtype=torch.bfloat16)
    x[-3:, 0] = torch.tensor([1.0, -2.0, 3.0])
    w = torch.full((1, 1), 2.0, device="cuda", dtype=torch.bfloat16)
    y = features.linear(x, w)
    assert y[-3:, 0].tolist() == [2.0, -4.0, 6.0]
    assert not y[:-3].any()


# ---- group norm ----------------------------------------------------------------

def norm_case(shape, groups, dtype, act, affine=True, spatial_dims=2, shift=0.0, seed=0):
    normal = draws(seed)
    c = shape[-1]
    x = normal(*shape, dtype=dtype, shift=shift).requires_grad_()
    w = normal(c, dtype=dtype, scale=0.3, shift=1.0).requires_grad_() if affine else None
    b = normal(c, dtype=dtype, scale=0.3).requires_grad_() if affine else None
    y = features.group_norm(x, groups, w, b, activation=act, spatial_dims=spatial_dims)
    dy = normal(*shape, dtype=dtype)
    leaves = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    check_norm(x.detach(), groups, w, b, act, spatial_dims, y.detach(), grads, dy)


def check_norm(x, groups, w, b, act, spatial_dims, y, grads=None, dy=None):
    """Every value against the formulas.  The moments are joined in doubles
    from fp32 sums of at most 2^9 terms of x - pivot: (2^9 + 8) u relative to
    the mean magnitude (of the square, for the variance)."""
    c = x.shape[-1]
    s = math.prod(x.shape[-1 - spatial_dims:-1])
    X = x.double().reshape(-1, s, groups, c // groups)
    one = torch.ones(c, device=x.device, dtype=torch.float64)
    W = (one if w is None else w.detach().double()).reshape(groups, -1)
    B = (0 * one if b is None else b.detach().double()).reshape(groups, -1)
    mean = X.mean((1, 3), keepdim=True)
    var = (X - mean).square().mean((1, 3), keepdim=True)
    rstd = (var + 1e-5).rsqrt()
    hat = (X - mean) * rstd
    U_ = hat * W + B
    n = 520 * U
    apart = (X - X[:, :1]).abs().mean((1, 3), keepdim=True)
    spread = (X - X[:, :1]).square().mean((1, 3), keepdim=True)
    e_mean = n * apart + U * mean.abs()
    e_rstd = rstd * (n * spread * rstd.square() + 4 * U)  # relative: half of d var / var
    e_hat = (e_mean + U * (X.abs() + mean.abs())) * rstd + (X - mean).abs() * e_rstd \
        + 4 * U * hat.abs()
    e_u = e_hat * W.abs() + 4 * U * (U_.abs() + B.abs())
    value, rate = value_and_slope(U_, act)
    check(y, value.reshape(x.shape), (1.2 * e_u + 16 * U * value.abs() + 1e-30).reshape(x.shape),
          "y")
    if grads is None:
        return
    D = dy.double().reshape(X.shape)
    du = D * rate
    e_du = D.abs() * (1.2 * e_u + 16 * U * (1 + U_.abs()))
    if act == "none":
        e_du = D.abs() * U
    if act == "relu":
        e_du = D.abs() * ((U_.abs() <= e_u).double() + U)
    if len(grads) == 3:
        e_db = n * du.abs().sum((0, 1)) + e_du.sum((0, 1))
        e_dw = n * (du * hat).abs().sum((0, 1)) + (e_du * hat.abs() + du.abs() * e_hat).sum((0, 1))
        check(grads[1], (du * hat).sum((0, 1)).reshape(-1), e_dw.reshape(-1), "dw")
        check(grads[2], du.sum((0, 1)).reshape(-1), e_db.reshape(-1), "db")
    dh = du * W
    e_dh = e_du * W.abs() + U * dh.abs()

    def avg(v):
        return v.mean((1, 3), keepdim=True)

    m1, m2 = avg(dh), avg(dh * hat)
    e_m1 = avg(e_dh) + n * avg(dh.abs())
    e_m2 = avg(e_dh * hat.abs() + dh.abs() * e_hat) + n * avg((dh * hat).abs())
    inner = dh - m1 - hat * m2
    e_inner = (e_dh + e_m1 + e_hat * m2.abs() + hat.abs() * e_m2
               + 4 * U * (dh.abs() + m1.abs() + (hat * m2).abs()))
    check(grads[0], (rstd * inner).reshape(x.shape),
          (rstd * e_inner + e_rstd * inner.abs()).reshape(x.shape), "dx")


NORM_SHAPES = [((1, 1, 1, 4), 2), ((1, 1, 1, 1), 1), ((2, 3, 5, 8), 8), ((1, 37, 53, 35), 5),
               ((3, 17, 19, 35), 7), ((2, 16, 16, 32), 4), ((1, 100, 90, 64), 1),
               ((2, 31, 33, 48), 4), ((5, 8, 9, 6), 3), ((1, 9, 9, 1031), 1),
               ((1, 5, 7, 2050), 2), ((4, 2, 2, 512), 32), ((300, 2, 1, 8), 2),
               ((2, 120, 160, 24), 8), ((1, 200, 300, 3), 1), ((1, 301, 211, 35), 5),
               ((2, 300, 200, 35), 7), ((1, 150, 130, 149), 1), ((1, 40, 60, 600), 1),
               ((3, 90, 110, 66), 2), ((2, 80, 80, 32), 8), ((1, 150, 160, 40), 8)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape, groups", NORM_SHAPES)
def test_group_norm_shapes(shape, groups, dtype):
    norm_case(shape, groups, dtype, "silu")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("affine", [True, False])
def test_group_norm_activations(act, affine, dtype):
    norm_case((2, 20, 30, 40), 5, dtype, act, affine, seed=1)
    norm_case((1, 150, 130, 16), 4, dtype, act, affine, seed=2)


def test_group_norm_far_from_zero():
    """A mean of 1000 deviations does not cost the variance its digits."""
    norm_case((2, 64, 64, 32), 8, torch.float32, "none", shift=1000.0, seed=3)
    norm_case((1, 300, 300, 32), 8, torch.float32, "none", shift=1000.0, seed=3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_group_norm_constant_group(dtype):
    x = torch.full((1, 20, 20, 8), 3.0, device="cuda", dtype=dtype)
    y = features.group_norm(x, 2)
    assert not y.any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_group_norm_sets_and_strides(dtype):
    norm_case((2, 700, 24), 3, dtype, "gelu", spatial_dims=1, seed=4)
    norm_case((2, 3, 9, 7, 5, 12), 3, dtype, "gelu", spatial_dims=3, seed=4)
    normal = draws(5)
    x = normal(2, 21, 23, 20, dtype=dtype)[..., 2:18]
    y = features.group_norm(x, 4, activation="silu")
    check_norm(x, 4, None, None, "silu", 2, y)
    nchw = normal(2, 16, 21, 23, dtype=dtype).permute(0, 2, 3, 1)
    y = features.group_norm(nchw, 4)
    check_norm(nchw, 4, None, None, "none", 2, y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(0, 4, 4, 8), (2, 0, 4, 8)])
def test_group_norm_without_values(shape, dtype):
    x = torch.zeros(shape, device="cuda", dtype=dtype, requires_grad=True)
    w = torch.ones(8, device="cuda", dtype=dtype, requires_grad=True)
    y = features.group_norm(x, 2, w)
    assert y.shape == shape
    y.sum().backward()
    assert x.grad.shape == shape and not w.grad.any()


@pytest.mark.parametrize("side", [20, 300])
@pytest.mark.parametrize("dtype", DTYPES)
def test_group_norm_not_finite_stays_in_its_group(side, dtype):
    normal = draws(6)
    x = normal(2, side, side, 16, dtype=dtype)
    clean = features.group_norm(x, 4)
    x[1, 3, 2, 5] = float("nan")
    y = features.group_norm(x, 4)
    assert y[1, ..., 4:8].isnan().all()
    assert torch.equal(y[0], clean[0])
    assert torch.equal(y[1, ..., :4], clean[1, ..., :4])
    assert torch.equal(y[1, ..., 8:], clean[1, ..., 8:])


@pytest.mark.parametrize("dtype", DTYPES)
def test_group_norm_same_bits_again(dtype):
    normal = draws(7)
    x = normal(2, 200, 150, 32, dtype=dtype).requires_grad_()
    w, b = (normal(32, dtype=dtype).requires_grad_() for _ in range(2))
    dy = normal(2, 200, 150, 32, dtype=dtype)
    runs = []
    for _ in range(2):
        y = features.group_norm(x, 8, w, b, activation="silu")
        runs.append((y, *torch.autograd.grad(y, (x, w, b), dy)))
    assert all(torch.equal(a, c) for a, c in zip(*runs))


def test_group_norm_single_gradients():
    normal = draws(8)
    x = normal(2, 30, 20, 16, dtype=torch.float32)
    w, b = (normal(16, dtype=torch.float32) for _ in range(2))
    dy = normal(2, 30, 20, 16, dtype=torch.float32)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = features.group_norm(leaves[0], 4, leaves[1], leaves[2], activation="silu")
    whole = torch.autograd.grad(y, leaves, dy)
    for which in range(3):
        one = [t.clone() for t in (x, w, b)]
        one[which].requires_grad_()
        y = features.group_norm(one[0], 4, one[1], one[2], activation="silu")
        assert torch.equal(torch.autograd.grad(y, one[which], dy)[0], whole[which])


# ---- together --------------------------------------------------------------------

def decoder(dtype, normal, grad=True, channels=35):
    def leaf(*shape, scale=1.0, shift=0.0):
        return normal(*shape, dtype=dtype, scale=scale, shift=shift).requires_grad_(grad)

    F = features
    return F.FeatureDecoder(
        F.Linear(leaf(32, channels, scale=channels ** -0.5), leaf(32), "silu"),
        F.GroupNorm(8, leaf(32, shift=1.0), leaf(32), activation="gelu"),
        F.Linear(leaf(32, 32, scale=32 ** -0.5), leaf(32), "silu", residual=True),
        F.Linear(leaf(3, 32, scale=32 ** -0.5), leaf(3), "sigmoid"))


def plain_decoder(layers, image):
    for v in layers:
        if isinstance(v, features.Linear):
            y = value_and_slope(image @ v.weight.double().t() + v.bias.double(), v.activation)[0]
            image = y + image if v.residual else y
        else:
            b, h, w, c = image.shape
            g = image.reshape(b, h * w, v.groups, -1)
            m = g.mean((1, 3), keepdim=True)
            var = (g - m).square().mean((1, 3), keepdim=True)
            g = ((g - m) * (var + v.eps).rsqrt()).reshape(image.shape)
            image = value_and_slope(g * v.weight.double() + v.bias.double(), v.activation)[0]
    return image


@pytest.mark.parametrize("dtype", DTYPES)
def test_decoder_run(dtype):
    """Four layers and their gradients.  Each layer rounds once (h), each
    gradient once more, and the layers' norms amplify by a factor of a few:
    64 h relative in the 2-norm covers eight roundings amplified eightfold."""
    normal = draws(10)
    d = decoder(dtype, normal)
    image = normal(2, 40, 50, 35, dtype=dtype).requires_grad_()
    dy = normal(2, 40, 50, 3, dtype=dtype)
    out = d(image)
    leaves = [image, *d.parameters()]
    grads = torch.autograd.grad(out, leaves, dy)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    params = iter(wide[1:])
    layers = []
    for v in d.layers:
        w, b = next(params), next(params)
        layers.append(features.Linear(w, b, v.activation, v.residual)
                      if isinstance(v, features.Linear)
                      else features.GroupNorm(v.groups, w, b, v.eps, v.activation))
    want = plain_decoder(layers, wide[0])
    want_grads = torch.autograd.grad(want, wide, dy.double())
    bound = 64 * max(half_step(dtype), U)
    for a, c in zip((out, *grads), (want, *want_grads)):
        assert (a.detach().double() - c.detach()).norm() <= bound * c.detach().norm()


@pytest.mark.parametrize("which", ["gs3d", "rade", "aaa"])
def test_rasterize_with_decoder(which):
    """The decoded image is the decoder's answer for the extras' image, and its
    gradients reach the Gaussians' features and the decoder."""
    import dsl_splat_b200
    from dsl_splat_b200.scenes import make_scene

    rasterize = getattr(dsl_splat_b200, which).rasterize
    s = make_scene(1, n=3000, width=96, height=64)
    dev = torch.device("cuda", 0)
    normal = draws(11)
    d = decoder(torch.bfloat16, normal, channels=20)  # gs3d blends at most 32 channels
    extra = normal(3000, 20, dtype=torch.float32).requires_grad_()
    args = [t.to(dev) for t in (s.means, s.quats, s.scales, s.opacities, s.viewmats, s.Ks)]
    res = rasterize(*args, s.width, s.height, sh_coeffs=s.sh_coeffs.to(dev), extra_features=extra,
                    feature_decoder=d)
    assert res.decoded_features.shape == res.features.shape[:-1] + (3,)
    assert torch.equal(res.decoded_features, d(res.extra_features))
    res.decoded_features.float().square().sum().backward()
    for t in (extra, *d.parameters()):
        assert t.grad is not None and t.grad.isfinite().all() and t.grad.any()
    plain = rasterize(*args, s.width, s.height, sh_coeffs=s.sh_coeffs.to(dev),
                      extra_features=extra)
    assert plain.decoded_features is None
    assert torch.equal(plain.features, res.features)


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_and_replayed(dtype):
    """Forward and backward in a CUDA graph, replayed on new inputs, against
    the same calls outside it; two graphs of one pool do not disturb each other."""
    normal = draws(12)
    d = decoder(dtype, normal)
    first, second = (normal(1, 64, 70, 35, dtype=dtype) for _ in range(2))
    dy = normal(1, 64, 70, 3, dtype=dtype)

    def step(image):
        leaf = image.detach().requires_grad_()
        out = d(leaf)
        grads = torch.autograd.grad(out, [leaf, *d.parameters()], dy)
        # no eager graph of the parameters may live on into the capture
        return (out.detach(), *grads)

    want = [[t.clone() for t in step(v)] for v in (first, second)]
    static = first.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    pool = torch.cuda.graph_pool_handle()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(step(static))
        graphs.append(g)
    for image, expected in zip((first, second), want):
        for g, out in zip(graphs, outs):
            static.copy_(image)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, expected))


def test_two_streams_at_once():
    """Calls in flight on two streams share nothing."""
    normal = draws(13)
    d = decoder(torch.bfloat16, normal, grad=False)
    images = [normal(1, 200, 300, 35, dtype=torch.bfloat16) for _ in range(2)]
    want = [d(v) for v in images]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = d(images[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", DTYPES)
def test_torch_ops_forms(dtype):
    normal = draws(14)
    x, w, b, r = (normal(*s, dtype=dtype).requires_grad_()
                  for s in ((90, 24), (40, 24), (40,), (90, 40)))
    dy = normal(90, 40, dtype=dtype)
    y = torch.ops.splat200.feature_linear(x, w, b, r, "silu")
    own = features.linear(x, w, b, residual=r, activation="silu")
    assert torch.equal(y, own)
    for a, c in zip(torch.autograd.grad(y, (x, w, b, r), dy),
                    torch.autograd.grad(own, (x, w, b, r), dy)):
        assert torch.equal(a, c)
    v = normal(2, 45, 40, dtype=dtype).requires_grad_()
    y = torch.ops.splat200.feature_norm(v, 4, b, None, 1e-5, "gelu")[0]
    own = features.group_norm(v, 4, b, activation="gelu", spatial_dims=1)
    assert torch.equal(y, own)
    dy = normal(2, 45, 40, dtype=dtype)
    for a, c in zip(torch.autograd.grad(y, (v, b), dy), torch.autograd.grad(own, (v, b), dy)):
        assert torch.equal(a, c)
