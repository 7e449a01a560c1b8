"""features.linear_cross_entropy on the GPU against its definition in 64 bits.

Bounds, with u = 2^-23 for an fp32 operation (sums may truncate): a logit is off by
e_z = (K + 8) u sum |x w| + |b|; a log sum by the largest of its logits' errors that
matter (their mean under the softmax, and second orders), 8 u of its exponentials, and of the
sum itself (V + 8) u at most; p = exp(z - lse) relatively by both and u of the argument.
dz = u_i (p - [target]) is held in the operands' type, half a step relative and, of
float16, half of 2^-24 / 2^15 of the largest |u|; the products then add (n + 8) u."""

import math

import pytest
import torch

from dsl_splat_b200 import _native, features
from test_features_gpu import DTYPES, U, check, draws, half_step

pytestmark = pytest.mark.gpu


def reference(x, w, b, target, ignore, reduction, up=None):
    """Values and bounds of the loss (and dx, dw, db), for x (M,K)."""
    xd, wd = x.double(), w.double()
    M, K = xd.shape
    V = len(wd)
    bd = torch.zeros(V, dtype=torch.float64, device=x.device) if b is None else b.double()
    z = xd @ wd.t() + bd
    e_z = (K + 8) * U * (xd.abs() @ wd.abs().t()) + 2 * U * torch.where(bd.isinf(), 0, bd).abs()
    lse = torch.logsumexp(z, 1)
    p = torch.exp(z - lse[:, None])
    e_lse = ((p * e_z).sum(1) + torch.where(p > 0, e_z, 0).max(1).values ** 2
             + (min(V, 64 + V // 64) + 24) * U + 4 * U * lse.abs()
             + U * (p * torch.where(p > 0, z - lse[:, None], 0).abs()).sum(1))
    used = (target != ignore) & (target >= 0) & (target < V)
    at = torch.where(used, target.long(), 0)[:, None]
    rows = torch.where(used, lse - z.gather(1, at)[:, 0], 0.0)
    e_rows = torch.where(used, e_lse + e_z.gather(1, at)[:, 0] + U * rows.abs(), 0.0)
    count = max(1, int(used.sum()))
    if reduction == "none":
        out = [(rows, e_rows)]
    else:
        share = count if reduction == "mean" else 1
        out = [(rows.sum() / share, e_rows.sum() / share + 4 * U * rows.sum().abs() / share)]
    if up is None:
        return out
    ud = (up.double() * used) / (count if reduction == "mean" else 1)
    ud = ud.expand(M) if ud.ndim == 0 else ud
    hit = torch.zeros_like(z).scatter_(1, at, 1.0)
    dz = ud[:, None] * (p - hit)
    exponent = torch.where(p > 0, z - lse[:, None], 0).abs()
    e_p = p * (e_z + e_lse[:, None] + U * (exponent + 8) + 2 * U * torch.where(
        z.isinf(), 0, z).abs())
    e_dz = ud[:, None].abs() * (e_p + 2 * U * (p - hit).abs()) + 1e-36 * ud.abs().max()
    e_sum = e_dz
    if x.dtype != torch.float32:
        e_dz = e_dz + half_step(x.dtype) * (dz.abs() + e_dz)
        if x.dtype == torch.float16:
            e_dz = e_dz + 2.0 ** -39 * ud.abs().max() * used[:, None]
    out.append((dz @ wd, (V + 8) * U * (dz.abs() @ wd.abs()) + e_dz @ wd.abs()))
    out.append((dz.t() @ xd, (M + 8) * U * (dz.abs().t() @ xd.abs()) + e_dz.t() @ xd.abs()))
    out.append((dz.sum(0), (M + 8) * U * dz.abs().sum(0) + e_sum.sum(0)))
    return out


def make(m, k, v, dtype, seed, bias=True, ignored=0.2, ids=torch.int64, scale=2.0):
    normal = draws(seed)
    g = torch.Generator().manual_seed(seed + 1)
    target = torch.randint(0, v, (m,), generator=g)
    target[torch.rand(m, generator=g) < ignored] = -100
    return (normal(m, k, dtype=dtype), normal(v, k, dtype=dtype, scale=scale / math.sqrt(k)),
            normal(v, dtype=dtype) if bias else None, target.to(ids).cuda())


def run(x, w, b, target, reduction="mean", ignore=-100, up=None):
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    args = leaves + [None] * (3 - len(leaves))
    loss = features.linear_cross_entropy(args[0], args[1], target, args[2], ignore_index=ignore,
                                         reduction=reduction)
    assert loss.dtype == torch.float32
    if up is None:
        up = draws(99)(*loss.shape, dtype=torch.float32, shift=1.0)
    grads = torch.autograd.grad(loss, leaves, up)
    want = reference(x, w, b, target, ignore, reduction, up)
    check(loss.detach(), *want[0], "loss")
    for got, (value, tolerance), name in zip(grads, want[1:], ("dx", "dw", "db")):
        check(got, value, tolerance, name)
    with torch.no_grad():
        again = features.linear_cross_entropy(x, w, target, b, ignore_index=ignore,
                                              reduction=reduction)
    assert torch.equal(again, loss.detach())
    return loss.detach(), grads


SIZES = [(1, 1, 1), (1, 8, 2), (1, 64, 5000), (3, 5, 7), (50, 35, 150), (128, 64, 128),
         (129, 64, 129), (200, 72, 256), (255, 16, 257), (333, 100, 1203), (400, 64, 2049),
         (64, 128, 4096), (130, 512, 700), (257, 520, 515), (40, 1000, 300), (1000, 24, 20),
         (5000, 32, 33), (3000, 300, 1000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, k, v", SIZES)
def test_sizes(m, k, v, dtype):
    run(*make(m, k, v, dtype, 1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("bias, ids", [(True, torch.int32), (False, torch.int64)])
def test_reductions(reduction, bias, ids, dtype):
    for m, k, v in ((300, 40, 130), (700, 33, 2100), (260, 256, 600)):
        run(*make(m, k, v, dtype, 2, bias=bias, ids=ids), reduction=reduction)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, k, v", [(40000, 64, 2000), (70000, 16, 1000), (1000, 64, 70000),
                                     (20000, 40, 5003), (300, 24, 300007)])
def test_several_pieces(m, k, v, dtype):
    run(*make(m, k, v, dtype, 3), reduction="none")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_pieces_of_a_large_vocabulary(reduction, dtype):
    """dz takes 1.2 GB at least: two to four pieces, the last one short."""
    run(*make(4500, 24, 1 << 17, dtype, 27), reduction=reduction)


@pytest.mark.parametrize("dtype", DTYPES)
def test_wide_features(dtype):
    """More inputs than one accumulator takes."""
    run(*make(70, 5000, 90, dtype, 4))
    run(*make(20, 20008, 200, dtype, 5, bias=False))


@pytest.mark.parametrize("dtype", DTYPES)
def test_any_subset_of_gradients(dtype):
    for shape in ((500, 48, 700), (300, 35, 4100)):
        x, w, b, target = make(*shape, dtype, 6)

        def grads(which):
            leaves = [t.detach().clone().requires_grad_(i in which)
                      for i, t in enumerate((x, w, b))]
            loss = features.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2])
            return dict(zip(which, torch.autograd.grad(loss, [leaves[i] for i in which])))

        whole = grads((0, 1, 2))
        for which in ((0,), (1,), (2,), (0, 1), (1, 2)):
            for i, g in grads(which).items():
                assert torch.equal(g, whole[i])


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_do_not_count(dtype):
    x, w, b, target = make(300, 64, 500, dtype, 7)
    target[:] = -100
    for reduction in ("none", "sum", "mean"):
        loss, grads = run(x, w, b, target, reduction)
        assert not loss.any() and not any(g.any() for g in grads)
    target[17] = 3
    run(x, w, b, target, "mean")
    # another index, which is one of the words
    run(x, w, b, target.fill_(9), "mean", ignore=9)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [200, 3000])
def test_words_taken_out(dtype, v):
    """A bias of minus infinity, of the type's lowest value, and a single word left."""
    x, w, b, target = make(200, 40, v, dtype, 8, ignored=0.0)
    out = torch.rand(v, generator=torch.Generator().manual_seed(9)).cuda() < 0.5
    out[target.unique()] = False
    for low in (-math.inf, torch.finfo(dtype).min):
        loss, grads = run(x, w, torch.where(out, torch.full_like(b, low), b), target, "none")
        assert loss.isfinite().all() and not grads[1][out].any() and not grads[2][out].any()
    # whole tiles of nothing, before and behind the only word
    for word in (0, v // 2, v - 1):
        alone = torch.full_like(b, -math.inf)
        alone[word] = 1.0
        loss, grads = run(x, w, alone, torch.full_like(target, word), "none")
        # log2 of the exponential of r, less r: r is what the rounding of the largest logit to
        # units of log 2 leaves.  The exponential is off by 2 units of 2^-23 and rounded by half
        # a one, its logarithm and the difference (both below 2^-20) add less than one
        assert float(loss.abs().max()) <= 2.0 ** -21
    # a target that is out has an infinite loss; nothing left is not a number
    b[int(target[5])] = -math.inf
    loss = features.linear_cross_entropy(x, w, target, b, reduction="none")
    assert bool((loss.isinf() == (target == target[5])).all())
    loss = features.linear_cross_entropy(x, w, target, torch.full_like(b, -math.inf),
                                         reduction="none")
    assert loss.isnan().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_logits(dtype):
    """Logits of some hundred: exponentials that only exist relative to the largest."""
    run(*make(300, 64, 700, dtype, 10, scale=60.0), reduction="none")


@pytest.mark.parametrize("dtype", DTYPES)
def test_small_and_unlike_upstreams(dtype):
    x, w, b, target = make(400, 64, 900, dtype, 11)
    for exponent in (-90, -24, 0, 30):
        up = draws(12)(400, dtype=torch.float32) * 2.0 ** exponent
        if dtype == torch.float16:
            up = up * 2.0 ** 8 if exponent == -24 else up
        if dtype != torch.float16 or -24 <= exponent <= 0:
            run(x, w, b, target, "none", up=up)
    up = draws(13)(400, dtype=torch.float32)
    up[::2] *= 2.0 ** -20
    run(x, w, b, target, "none", up=up)
    loss, grads = run(x, w, b, target, "none", up=torch.zeros(400, device="cuda"))
    assert not any(g.any() for g in grads)


def test_rows_do_not_meet():
    """A row that is not finite leaves the others' losses and gradients as they are."""
    for dtype, v in ((torch.float32, 300), (torch.bfloat16, 300), (torch.bfloat16, 5000)):
        x, w, b, target = make(300, 64, v, dtype, 14, ignored=0.0)

        def both():
            leaf = x.detach().clone().requires_grad_()
            loss = features.linear_cross_entropy(leaf, w, target, b, reduction="none")
            return loss.detach(), torch.autograd.grad(loss.sum(), leaf)[0]

        want = both()
        x[7, 3], x[130, 0] = float("nan"), float("inf")
        got = both()
        rest = torch.ones(300, dtype=torch.bool)
        rest[[7, 130]] = False
        for a, c in zip(got, want):
            assert torch.equal(a[rest], c[rest])
            assert not a[7].isfinite().any()
        assert not got[0][130].isfinite()


@pytest.mark.parametrize("dtype", DTYPES)
def test_upstreams_that_are_not_finite(dtype):
    """They reach their rows' dx, and no other's."""
    x, w, b, target = make(300, 64, 300, dtype, 28, ignored=0.1)
    target[5], target[9] = -100, 3
    up = draws(29)(300, dtype=torch.float32)

    def dx():
        leaf = x.detach().clone().requires_grad_()
        loss = features.linear_cross_entropy(leaf, w, target, b, reduction="none")
        return torch.autograd.grad(loss, leaf, up)[0]

    want = dx()
    up[[5, 9, 200]] = torch.tensor([math.nan, math.inf, math.nan], device="cuda")
    target[200] = 4
    got = dx()
    rest = torch.ones(300, dtype=torch.bool)
    rest[[9, 200]] = False
    assert torch.equal(got[rest], want[rest]) and not got[5].any()
    assert not got[9].isfinite().any() and not got[200].isfinite().any()


def test_targets_outside_the_vocabulary():
    device = torch.device("cuda", torch.cuda.current_device())
    x, w, b, target = make(600, 64, 300, torch.bfloat16, 15)
    assert _native.device_error(device) == 0
    bad = target.clone()
    bad[::3] = torch.tensor([-1, 300, 1 << 40, -(1 << 40)], device="cuda").repeat(50)
    run(x, w, b, bad, "mean")
    assert _native.device_error(device) == -6 and _native.device_error(device) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_shapes_and_strides(dtype):
    x, w, b, target = make(120, 80, 90, dtype, 16)
    wide = x.reshape(5, 4, 6, 80)
    labels = target.reshape(5, 4, 6)
    want = features.linear_cross_entropy(x[:, ::2].contiguous(), w[:, ::2].contiguous(), target,
                                         b, reduction="none").reshape(5, 4, 6)
    got = features.linear_cross_entropy(wide[..., ::2], w[:, ::2], labels, b, reduction="none")
    assert torch.equal(got, want)
    got = features.linear_cross_entropy(wide.transpose(0, 2)[..., ::2], w[:, ::2],
                                        labels.transpose(0, 2), b, reduction="none")
    assert torch.equal(got, want.transpose(0, 2))
    one = features.linear_cross_entropy(x[3], w, target[3], b, reduction="none")
    assert one.shape == () and abs(float(one - features.linear_cross_entropy(
        x, w, target, b, reduction="none")[3])) <= 1e-5 * (1 + abs(float(one)))
    # a broadcast upstream
    leaf = x.detach().requires_grad_()
    loss = features.linear_cross_entropy(leaf, w, target, b, reduction="none")
    a, = torch.autograd.grad(loss.sum(), leaf)
    c, = torch.autograd.grad(features.linear_cross_entropy(leaf, w, target, b, reduction="none"),
                             leaf, torch.ones(120, device="cuda"))
    assert torch.equal(a, c)


def test_no_rows():
    w = torch.ones(7, 4, device="cuda", requires_grad=True)
    x = torch.empty(0, 4, device="cuda", requires_grad=True)
    target = torch.empty(0, dtype=torch.int64, device="cuda")
    for reduction in ("none", "sum", "mean"):
        loss = features.linear_cross_entropy(x, w, target, reduction=reduction)
        assert not loss.any() and loss.shape == ((0,) if reduction == "none" else ())
        dx, dw = torch.autograd.grad(loss, (x, w), torch.ones_like(loss))
        assert dx.shape == (0, 4) and not dw.any()


def test_against_differences():
    x, w, b, target = make(60, 24, 40, torch.float32, 17)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    loss = features.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2])
    grads = torch.autograd.grad(loss, leaves)
    for i, grad in enumerate(grads):
        direction = torch.randn_like(grad)
        ends = []
        with torch.no_grad():
            for sign in (1, -1):
                moved = [t + sign * 2 ** -8 * direction if j == i else t
                         for j, t in enumerate(leaves)]
                ends.append(float(features.linear_cross_entropy(moved[0], moved[1], target,
                                                                moved[2]).double()))
        # third derivatives of order |d z|^3 (some 10^3) times 2^-16 / 6, and 2^-22 of the loss
        # over the step
        slope = (ends[0] - ends[1]) * 2 ** 7
        assert abs(slope - float((grad.double() * direction.double()).sum())) < 0.02


@pytest.mark.parametrize("dtype, v", [(torch.float32, 300), (torch.bfloat16, 300),
                                      (torch.bfloat16, 5000)])
def test_captured_and_replayed(dtype, v):
    """Two captured training steps replayed in turn, on another stream."""
    side = torch.cuda.Stream()
    runs = []
    for seed in (18, 19):
        x, w, b, target = make(700, 64, v, dtype, seed)
        want = run(x, w, b, target, up=torch.ones((), device="cuda"))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            leaves = [t.detach().requires_grad_() for t in (x, w, b)]
            up = torch.ones((), device="cuda")
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                loss = features.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2])
                grads = torch.autograd.grad(loss, leaves, up)
        # a graph reads its inputs where they were: they are kept
        runs.append((graph, loss, grads, want, leaves, target, up))
    with torch.cuda.stream(side):
        for _ in range(2):
            for graph, *_ in runs:
                graph.replay()
    torch.cuda.synchronize()
    for _, loss, grads, want, *_ in runs:
        assert torch.equal(loss, want[0])
        for a, c in zip(grads, want[1]):
            assert torch.equal(a, c)


def test_decoder():
    x, w, b, target = make(600, 64, 300, torch.float32, 20)
    g, h = draws(21)(64, dtype=torch.float32), draws(22)(64, dtype=torch.float32)
    decoder = features.FeatureDecoder(features.LayerNorm(g, h, activation="silu"),
                                      features.Linear(w, b))
    image, labels = x.reshape(20, 30, 64), target.reshape(20, 30)
    got = decoder.cross_entropy(image, labels, reduction="none")
    want = torch.nn.functional.cross_entropy(decoder(image).reshape(600, 300).double(), target,
                                             reduction="none").reshape(20, 30)
    # both take the same logits but for their rounding: 64 products of about one
    assert float((got - want).abs().max()) < 100 * U * 20


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("rows", [3, 2048])
def test_upstreams_cost_no_digits(rows, reduction, dtype):
    """Labels' dz, which is nearly -u, is what most of dx and dW is made of.  The gradients'
    own rounding leaves a relative 2-norm error of up to half a step / sqrt(3).  dz with u of
    its own has two values; with a shared u, which is left to the results, it is p - 1 or p,
    whose rounding is small (1 - p beside 1, p of some 2^-8, an eighth of a step here).  So the
    whole stays below 1.2 times the rounding; a u that dz had taken in as one value would
    add up to half a step."""
    x, w, _, target = make(rows, 64, 512, dtype, 23, bias=False, scale=1.0, ignored=0.0)
    up = torch.full((rows,) if reduction == "none" else (), 1.0 + 2.0 ** -9, device="cuda")
    if reduction == "none":
        up = up + draws(24)(rows, dtype=torch.float32).abs()
    leaves = [t.detach().requires_grad_() for t in (x, w)]
    loss = features.linear_cross_entropy(*leaves, target, reduction=reduction)
    grads = torch.autograd.grad(loss, leaves, up)
    for got, (want, _) in zip(grads, reference(x, w, None, target, -100, reduction, up)[1:3]):
        off = float((got.double() - want).norm() / want.norm())
        assert off < 1.2 * half_step(dtype) / math.sqrt(3)


def gradients(x, w, b, target, reduction, up):
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    loss = features.linear_cross_entropy(*leaves[:2], target, leaves[2], reduction=reduction)
    return loss.detach(), torch.autograd.grad(loss, leaves, up)


# on the chip of whole 16-byte rows and of odd ones, and rows of several accumulators
WIDTHS = [(700, 64, 300), (700, 35, 300), (300, 520, 260), (70, 16392, 40)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("m, k, v", WIDTHS)
def test_rows_that_do_not_count_may_hold_anything(m, k, v, reduction, dtype):
    """Infinities and NaN of padded rows reach no loss and no gradient."""
    x, w, b, target = make(m, k, v, dtype, 30, ignored=0.3)
    target[5], target[6], target[-1] = -100, v, -100
    up = draws(31)(*([m] if reduction == "none" else []), dtype=torch.float32, shift=1.0)
    want = gradients(x, w, b, target, reduction, up)
    out = (target < 0) | (target >= v)
    x[out] = torch.tensor([math.nan, math.inf, -math.inf], device="cuda").to(dtype).repeat(m)[
        :int(out.sum())][:, None]
    got = gradients(x, w, b, target, reduction, up)
    assert torch.equal(got[0], want[0])
    for a, c in zip(got[1], want[1]):
        assert torch.equal(a, c)
    assert not got[1][0][out].any()
    assert _native.device_error(torch.device("cuda", torch.cuda.current_device())) == -6


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, k, v", WIDTHS)
def test_weights_that_are_not_finite_leave_rows_that_do_not_count(m, k, v, dtype):
    x, w, b, target = make(m, k, v, dtype, 32, ignored=0.3)
    w[3], w[7, 2] = math.nan, math.inf
    _, (dx, _, _) = gradients(x, w, b, target, "mean", torch.ones((), device="cuda"))
    assert not dx[target < 0].any() and not dx[target >= 0].isfinite().any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["sum", "mean"])
@pytest.mark.parametrize("up", [math.nan, math.inf])
def test_a_shared_upstream_that_is_not_finite(up, reduction, dtype):
    """It reaches the rows that count, and nothing where none does."""
    up = torch.tensor(up, device="cuda")
    for m, k, v in WIDTHS:
        x, w, b, target = make(m, k, v, dtype, 33, ignored=0.3)
        _, (dx, dw, db) = gradients(x, w, b, target, reduction, up)
        assert not dx[target < 0].any() and not dx[target >= 0].isfinite().any()
        assert not dw[target[target >= 0]].isfinite().any()
        assert not db[target[target >= 0]].isfinite().any()
        _, grads = gradients(x, w, b, target.fill_(-100), reduction, up)
        assert not any(g.any() for g in grads)


def labels_of(kind, x, w, seed):
    """Those of a head that has learnt nothing, of one whose softmax they follow, and of one
    that is always right."""
    z = (x.double() @ w.double().t()).cpu()
    g = torch.Generator().manual_seed(seed)
    return {"random": lambda: torch.randint(0, z.shape[1], (len(z),), generator=g),
            "drawn": lambda: torch.multinomial(torch.softmax(z, 1), 1, generator=g)[:, 0],
            "largest": lambda: z.argmax(1)}[kind]().to(x.device)


def digits(x, w, target, reduction, up, got):
    """The relative 2-norms of dx's and dW's errors, over those of their own rounding."""
    for have, (want, _) in zip(got, reference(x, w, None, target, -100, reduction, up)[1:3]):
        own = (want.to(have.dtype).double() - want).norm()
        yield float((have.double() - want).norm() / own)


# dz as two values is off by 2^-17 (bf16), and the logits by four additions of 2^-23 of some
# 2^4: 2^-17 relative of the exponentials.  Over fp16's own rounding (2^-11 / sqrt 6) that
# is 0.04, and as much again for the other sums.
TWO_VALUES = 1.1
# one value's rounding is of the size of the results' own: sqrt 2 where all of dz has it and
# rows of W are unlike, and that of the largest of 2048 such sums
ONE_VALUE = 1.55


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("kind", ["random", "drawn", "largest"])
def test_digits_of_gradients(kind, reduction, dtype):
    x, w, _, _ = make(2048, 64, 512, dtype, 34, bias=False, scale=4.0)
    target = labels_of(kind, x, w, 35)
    up = torch.full((2048,) if reduction == "none" else (), 1.0 + 2.0 ** -9, device="cuda")
    if reduction == "none":
        up = up + draws(36)(2048, dtype=torch.float32).abs()
    _, got = gradients(x, w, torch.zeros_like(w[:, 0]), target, reduction, up)
    for off in digits(x, w, target, reduction, up, got[:2]):
        assert off <= (TWO_VALUES if reduction == "none" else ONE_VALUE)


def pieces_of(m, k, v, dtype, reduction):
    """How many pieces the backward takes, and the last one's rows.  Its workspace holds what
    a piece needs, and so stops growing with the rows where they are one."""
    def size(rows):
        return _native.lib.splat_feature_entropy_workspace_bytes(
            {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype], rows, k, v,
            2 if reduction == "none" else 1)

    low, high = 1, 1 << 29  # size(high) is that of a whole piece
    while low < high:
        middle = (low + high) // 2
        if size(middle) == size(1 << 29):
            high = middle
        else:
            low = middle + 1
    return -(-m // low), m - (m - 1) // low * low


@pytest.mark.parametrize("m, k, v, dtype, reduction, pieces", [
    # on the chip, dW in several ranges of rows, of which the last piece has fewer
    (300000, 64, 2000, torch.float32, "mean", 4), (300000, 64, 2000, torch.bfloat16, "none", 3),
    (300000, 64, 2000, torch.float16, "mean", 2),
    # logits in memory: a range, and several
    (4500, 520, 1 << 17, torch.float32, "none", 3), (4500, 520, 1 << 17, torch.float32, "mean", 3),
    (200000, 520, 2000, torch.float32, "none", 2), (200000, 520, 2000, torch.float32, "mean", 2),
    (20000, 16392, 100, torch.bfloat16, "none", 2), (20000, 16392, 100, torch.bfloat16, "mean", 2),
    (20000, 16392, 100, torch.float16, "mean", 2)])
def test_pieces_with_a_short_last_one(m, k, v, dtype, reduction, pieces):
    count, last = pieces_of(m, k, v, dtype, reduction)
    assert count == pieces and last < m // count
    run(*make(m, k, v, dtype, 40), reduction=reduction)
    torch.cuda.empty_cache()
