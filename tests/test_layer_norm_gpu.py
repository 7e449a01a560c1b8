"""features.layer_norm on the GPU against its definition in 64 bits.

Tolerances bound each value's rounding, with u = 2^-23 for an fp32 operation and half a
step of the type for the one rounding to it.  A row's sums are trees: a lane adds
at most 32 values (of long rows a 256th of them), 16 steps join lanes and warps, so a sum is
off by at most `depth` u times its terms' magnitudes.  Activations and slopes: 16 u
relative, and what their argument is off by times 1.2.
"""

import pytest
import torch

from dsl_splat_b200 import features
from test_features_gpu import ACTS, DTYPES, U, check, draws, value_and_slope

pytestmark = pytest.mark.gpu


def reference(x, w, b, eps, act, dy=None):
    """Values and bounds of y (and dx, dw, db)."""
    C, M = x.shape[-1], x.numel() // x.shape[-1]
    depth = 48 + C // 256
    xd = x.double().reshape(M, C)
    wd = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.double()
    bd = torch.zeros_like(wd) if b is None else b.double()
    d = xd - xd.mean(1, keepdim=True)
    var = d.square().mean(1, keepdim=True)
    rstd = (var + eps).rsqrt()
    h = d * rstd
    # the second mean is taken of the deviations: they are off by the rounding of x - mean
    # and by their own sum's; the variance by that and its sum's, twice
    size = d.abs().mean(1, keepdim=True)
    e_d0 = (depth + 4) * U * (d.abs() + size)
    e_h = e_d0 * rstd + (2 * depth + 12) * U * h.abs()
    u = h * wd + bd
    e_u = e_h * wd.abs() + 2 * U * ((h * wd).abs() + bd.abs())
    value, rate = value_and_slope(u, act)
    out = [(value, 1.2 * e_u + 16 * U * value.abs() + 1e-30)]
    if dy is None:
        return out
    g0 = dy.double().reshape(M, C)
    du = g0 * rate
    e_du = g0.abs() * (1.2 * e_u + 16 * U * (1 + u.abs()))
    if act == "none":
        e_du = du.abs() * U
    if act == "relu":  # the slope jumps where u is within its own error of 0
        e_du = g0.abs() * ((u.abs() <= e_u).double() + U)
    g = du * wd
    e_g = e_du * wd.abs() + U * g.abs()
    m1, m2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    e_m1 = e_g.mean(1, keepdim=True) + depth * U * g.abs().mean(1, keepdim=True)
    e_m2 = ((e_g * h.abs() + g.abs() * e_h).mean(1, keepdim=True)
            + (depth + 2) * U * (g * h).abs().mean(1, keepdim=True))
    dx = rstd * (g - m1 - h * m2)
    e_dx = rstd * (e_g + e_m1 + e_h * m2.abs() + h.abs() * e_m2
                   + 4 * U * (g.abs() + m1.abs() + (h * m2).abs())) \
        + (2 * depth + 12) * U * dx.abs()
    out.append((dx, e_dx + 1e-30))
    out.append(((du * h).sum(0), (e_du * h.abs() + du.abs() * e_h).sum(0)
                + (M + 8) * U * (du * h).abs().sum(0) + 1e-30))
    out.append((du.sum(0), e_du.sum(0) + (M + 8) * U * du.abs().sum(0) + 1e-30))
    return out


def run(x, w, b, act, dy, eps=1e-5):
    tensors = [t for t in (x, w, b) if t is not None]
    leaves = [t.detach().requires_grad_() for t in tensors]
    given = iter(leaves)
    args = [None if t is None else next(given) for t in (x, w, b)]
    y = features.layer_norm(*args, eps=eps, activation=act)
    grads = iter(torch.autograd.grad(y, leaves, dy))
    want = reference(x, w, b, eps, act, dy)
    check(y.detach().reshape(want[0][0].shape), *want[0], "y")
    for t, (value, tolerance), name in zip((x, w, b), want[1:], ("dx", "dw", "db")):
        if t is not None:
            check(next(grads).reshape(value.shape), value, tolerance, name)
    with torch.no_grad():
        assert torch.equal(features.layer_norm(x, w, b, eps=eps, activation=act), y)


def make(m, c, dtype, seed, shift=0.0, affine=True):
    normal = draws(seed)
    x = normal(m, c, dtype=dtype, scale=1.5, shift=shift)
    w = normal(c, dtype=dtype, scale=0.3, shift=1.0) if affine else None
    b = normal(c, dtype=dtype, scale=0.3) if affine else None
    return x, w, b, normal(m, c, dtype=dtype)


SIZES = [(1, 1), (3, 2), (1, 8), (7, 3), (33, 16), (129, 32), (1000, 35), (500, 48), (257, 64),
         (64, 100), (40, 128), (300, 129), (31, 255), (17, 256), (9, 300), (70, 511), (33, 512),
         (12, 777), (11, 1023), (8, 1024), (5, 1025), (6, 2048), (3, 5000), (2, 8191), (3, 8192),
         (2, 8193), (5, 20000), (1, 65535)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, c", SIZES)
def test_sizes(m, c, dtype):
    x, w, b, dy = make(m, c, dtype, 1)
    run(x, w, b, "silu", dy)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, c", [(100001, 35), (70000, 64), (60001, 8), (3000, 1000),
                                  (20000, 3), (900, 9000)])
def test_many_rows(m, c, dtype):
    x, w, b, dy = make(m, c, dtype, 2)
    run(x, w, b, "gelu", dy)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("affine", [True, False])
def test_activations(act, affine, dtype):
    for c in (24, 25, 1500):
        x, w, b, dy = make(130, c, dtype, 3, affine=affine)
        run(x, w, b, act, dy)


@pytest.mark.parametrize("dtype", DTYPES)
def test_far_means(dtype):
    """A mean of many deviations costs the variance no digits."""
    for c in (64, 33, 1200, 9001):
        x, w, b, dy = make(50, c, dtype, 4, shift=200.0)
        run(x, w, b, "none", dy)


@pytest.mark.parametrize("dtype", DTYPES)
def test_constant_rows_and_eps(dtype):
    x = torch.full((5, 40), 3.0, dtype=dtype, device="cuda")
    b = draws(5)(40, dtype=dtype)
    y = features.layer_norm(x, None, b)
    assert torch.equal(y, b.expand(5, 40))
    x, w, b, dy = make(40, 48, dtype, 6)
    run(x, w, b, "none", dy, eps=0.5)


def test_rows_do_not_meet():
    """A row that is not finite leaves the others as they are."""
    for c in (32, 35, 1100, 9000):
        x, w, b, _ = make(21, c, torch.float32, 7)
        want = features.layer_norm(x, w, b)
        x[4, 1], x[9, 0] = float("nan"), float("inf")
        got = features.layer_norm(x, w, b)
        rest = torch.ones(21, dtype=torch.bool)
        rest[[4, 9]] = False
        assert torch.equal(got[rest], want[rest])
        assert got[4].isnan().all() and not got[9].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_shapes_and_strides(dtype):
    normal = draws(8)
    base = normal(6, 5, 80, dtype=dtype)
    w = normal(80, dtype=dtype)[::2]
    for x in (base[..., :40], base[:, 1:4, 1:41], base.transpose(0, 1)[..., 3:43]):
        want = features.layer_norm(x.contiguous(), w.contiguous())
        assert torch.equal(features.layer_norm(x, w), want)
    assert features.layer_norm(normal(0, 12, dtype=dtype)).shape == (0, 12)
    x = normal(0, 12, dtype=dtype).requires_grad_()
    w = normal(12, dtype=dtype).requires_grad_()
    dx, dw = torch.autograd.grad(features.layer_norm(x, w), (x, w), torch.empty_like(x))
    assert dx.shape == (0, 12) and not dw.any()


@pytest.mark.parametrize("which", [(0,), (1,), (2,), (0, 2), (1, 2)])
def test_any_subset_of_gradients(which):
    for c in (48, 35, 3000, 9001):
        x, w, b, dy = make(77, c, torch.bfloat16, 9)

        def grads(some):
            leaves = [t.detach().clone().requires_grad_(i in some)
                      for i, t in enumerate((x, w, b))]
            y = features.layer_norm(*leaves, activation="silu")
            return dict(zip(some, torch.autograd.grad(y, [leaves[i] for i in some], dy)))

        whole = grads((0, 1, 2))
        for i, g in grads(which).items():
            assert torch.equal(g, whole[i])


def test_against_differences():
    x, w, b, dy = make(9, 12, torch.float32, 10)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(features.layer_norm(*leaves, activation="gelu"), leaves, dy)
    for leaf, grad in zip(leaves, grads):
        direction = torch.randn_like(leaf)
        ends = []
        with torch.no_grad():
            for sign in (1, -1):
                moved = [t + sign * 2 ** -7 * direction if t is leaf else t for t in leaves]
                ends.append((features.layer_norm(*moved, activation="gelu").double()
                             * dy.double()).sum())
        slope = float(ends[0] - ends[1]) * 2 ** 6
        # third derivatives (of order one, times 100 values) and 2^-24 relative of the ends
        assert abs(slope - float((grad.double() * direction.double()).sum())) < 0.05


def test_streams_and_graphs():
    x, w, b, dy = make(3000, 64, torch.float32, 11)
    want = features.layer_norm(x, w, b, activation="silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        graph = torch.cuda.CUDAGraph()
        y = features.layer_norm(*leaves, activation="silu")
        first = torch.autograd.grad(y, leaves, dy)
        del y
        with torch.cuda.graph(graph, stream=side):
            y = features.layer_norm(*leaves, activation="silu")
            grads = torch.autograd.grad(y, leaves, dy)
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
    for g, f in zip(grads, first):
        assert torch.equal(g, f)


@pytest.mark.parametrize("dtype", DTYPES)
def test_weight_or_bias_alone(dtype):
    for c in (24, 25, 1500, 9000):
        x, w, b, dy = make(90, c, dtype, 12)
        run(x, w, None, "silu", dy)
        run(x, None, b, "gelu", dy)
