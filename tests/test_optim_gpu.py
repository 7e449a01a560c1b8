"""optim on the GPU: AdamW steps against the formula in 64 bits, 8-bit codes against
their definition bit by bit."""

import copy
import io
import math

import pytest
import torch

from dsl_splat_b200 import optim
from test_features_gpu import DTYPES, half_step, smallest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32
RUN = 256


def draw(seed, *shape, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).cuda()


def wide(t):
    return t.double()


def reference(p, g, m, v, step, lr, betas, eps, decay):
    """p', m', v' in 64 bits and what fp32 arithmetic may be off them."""
    b1, b2 = betas
    m1 = b1 * wide(m) + (1 - b1) * wide(g)
    v1 = b2 * wide(v) + (1 - b2) * wide(g) ** 2
    # two products and a sum, factors rounded to fp32
    e_m = 4 * U * (b1 * wide(m).abs() + (1 - b1) * wide(g).abs()) + 2.0 ** -148
    e_v = 5 * U * v1 + 2.0 ** -148
    rate = lr / (1 - b1 ** step)
    denominator = (v1 / (1 - b2 ** step)).sqrt() + eps
    move = rate * m1 / denominator
    p1 = wide(p) * (1 - lr * decay) - move
    # the root is off by half of v's error and its own rounding, then a product, a sum, a
    # quotient and a product
    e_p = (rate * e_m / denominator + move.abs() * 12 * U + wide(p).abs() * 3 * U + 3 * U
           * (p1.abs() + move.abs()))
    return (p1, m1, v1), (e_p, e_m, e_v)


def close(got, want, tolerance, name):
    rounded = (0 if got.dtype == torch.float32 else half_step(got.dtype)) * want.abs() \
        + smallest(got.dtype)
    off = (got.double() - want).abs()
    assert bool((off <= tolerance + rounded).all()), f"{name}: {float((off - tolerance).max())}"


SHAPES = [(1,), (3,), (255,), (256,), (257,), (4096,), (4097,), (1000, 3), (77, 15, 3), (20001,)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("maximize", [False, True])
def test_steps_in_32_bits(dtype, maximize):
    params = [draw(i, *s).to(dtype) for i, s in enumerate(SHAPES)]
    moments = [[torch.zeros(s, device="cuda") for s in SHAPES] for _ in range(2)]
    lrs = [10.0 ** -(1 + i % 4) for i in range(len(SHAPES))]
    decays = [0.1 * (i % 3) for i in range(len(SHAPES))]
    for step in (1, 2, 3, 1000):
        grads = [draw(100 * step + i, *s, scale=2.0 ** -i).to(dtype)
                 for i, s in enumerate(SHAPES)]
        before = [[t.clone() for t in group] for group in (params, *moments)]
        optim.adamw(params, grads, *moments, step=step, lr=lrs, betas=(0.9, 0.99), eps=1e-10,
                    weight_decay=decays, maximize=maximize)
        for i in range(len(SHAPES)):
            p, m, v = (group[i] for group in before)
            g = -grads[i] if maximize else grads[i]
            want, tolerance = reference(p, g, m, v, step, lrs[i], (0.9, 0.99), 1e-10, decays[i])
            for got, w, t, name in zip((params[i], moments[0][i], moments[1][i]), want,
                                       tolerance, "pmv"):
                close(got, w, t, f"{name} of {SHAPES[i]} at step {step}")


def test_unaligned_views_and_many_tensors():
    base = draw(1, 40000)
    cuts = [base[1 + 130 * i:1 + 130 * i + 129 - i % 3] for i in range(250)]
    grads = [draw(2 + i, len(c)) for i, c in enumerate(cuts)]
    grads[7] = torch.cat([grads[7], grads[7]]).reshape(2, -1).t()[:, 0]  # not contiguous
    moments = [[torch.zeros_like(c) for c in cuts] for _ in range(2)]
    before, whole = [c.clone() for c in cuts], base.clone()
    optim.adamw(cuts, grads, *moments, step=1, lr=0.01)
    touched = torch.zeros(40000, dtype=torch.bool, device="cuda")
    for i, c in enumerate(cuts):
        zero = torch.zeros_like(c)
        want, tolerance = reference(before[i], grads[i], zero, zero, 1, 0.01, (0.9, 0.999), 1e-8,
                                    0.01)
        close(c, want[0], tolerance[0], f"p {i}")
        touched[1 + 130 * i:1 + 130 * i + len(c)] = True
    assert torch.equal(base[~touched], whole[~touched])


# ---- 8 bits ------------------------------------------------------------------------------

def decoded(codes, exponents, mantissa, signed):
    """From a code's sign, exponent and mantissa, in 64 bits."""
    c = codes.reshape(-1).long()
    negative = signed & (c >= 128)
    c = torch.where(negative, c - 128, c)
    e, f = c // mantissa, c % mantissa
    size = torch.where(e == 0, f.double() / mantissa * 2.0 ** -14,
                       (1 + f.double() / mantissa) * 2.0 ** (e - 15).double())
    run = torch.arange(len(c), device=c.device) // RUN
    value = size * 2.0 ** exponents.double()[run]
    return torch.where(negative, -value, value).reshape(codes.shape)


def test_every_code():
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").repeat(5)
    exponents = torch.tensor([-126, -20, 0, 15, 100], dtype=torch.int8, device="cuda")
    for squared, mantissa in ((False, 8), (True, 16)):
        got = optim.Moment8(codes, exponents, squared).values()
        want = decoded(codes, exponents, mantissa, torch.tensor(not squared, device="cuda"))
        # exact but below fp32's normal range
        want = want.float().square() if squared else want.float()
        assert torch.equal(got, want)
        # and back, to the same codes' values (a run of less than half of its range moves
        # its exponent; its values stay)
        again = optim.Moment8.of(got[RUN:4 * RUN], squared).values()
        assert torch.equal(again, got[RUN:4 * RUN])


@pytest.mark.parametrize("n", [1, 31, 256, 1000, 70001])
def test_nearest_codes(n):
    x = draw(n, n) * 2.0 ** (20 * draw(n + 1, n)).clamp(-30, 30)
    for squared, mantissa in ((False, 8), (True, 16)):
        values = x.square() if squared else x
        moment = optim.Moment8.of(values, squared)
        held = decoded(moment.codes, moment.exponents, mantissa,
                       torch.tensor(not squared, device="cuda"))
        want = values.double().sqrt() if squared else values.double()
        run = torch.arange(n, device="cuda") // RUN
        least = 2.0 ** (moment.exponents.double()[run] - 14) / mantissa
        # half a step: relative of normal codes, of the least one below; a root's least code
        # stands for all below it; the root's own rounding comes first
        allowed = torch.maximum(want.abs() / mantissa / 2, least * (1.0 if squared else 0.5))
        assert bool(((held - want).abs() <= allowed * (1 + 2.0 ** -20)).all())
        if squared:
            assert bool(((values > 0) == (held > 0)).all())


def noise(n, step):
    low = 0xffffffff
    h = torch.arange(n, device="cuda")
    h = (h * 0x9e3779b9 + (step & low) * 0x6a09e667 + (h >> 32) * 0xbb67ae85) & low
    h = ((h ^ (h >> 16)) * 0x3c6ef373) & low
    h = ((h ^ (h >> 15)) * 0x510e527f) & low
    h = h ^ (h >> 16)
    return h & 0xffff, h >> 16


def rounded_down(x, mantissa, dither):
    """Codes and exponents of fp32 values: the definition, by exact steps in 64 bits."""
    n = len(x)
    size = x.double().abs()
    runs = torch.nn.functional.pad(size, (0, -n % RUN)).reshape(-1, RUN).amax(1)
    # the least exponent whose largest code reaches the largest magnitude
    e = torch.full_like(runs, -126)
    for k in range(-126, 128):
        e = torch.where(runs > (2 - 1 / mantissa) * 2.0 ** (e), torch.full_like(e, k), e)
    run = torch.arange(n, device="cuda") // RUN
    y = size * 2.0 ** -e[run]
    binade = torch.floor(torch.log2(y.clamp(min=2.0 ** -14)))
    binade = torch.where(2.0 ** binade > y.clamp(min=2.0 ** -14), binade - 1, binade)
    binade = torch.where(2.0 ** (binade + 1) <= y, binade + 1, binade).clamp(min=-14)
    step = 2.0 ** binade / mantissa
    k = torch.floor(y / step + dither.double() / 65536)
    code = torch.where(y < 2.0 ** -14, k, (binade + 14) * mantissa + k)
    return code.long(), e.to(torch.int8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 255, 256, 4097, 100001])
def test_steps_in_8_bits(n, dtype):
    p, m, v = (draw(n, n).to(dtype), draw(n + 1, n) * 0.1, draw(n + 2, n).square() * 0.01)
    first, second = optim.Moment8.of(m), optim.Moment8.of(v, squared=True)
    betas = (0.9, 0.999)
    for step in (1, 2, 50000):
        g = (draw(n + 3 + step, n) * 0.1).to(dtype)
        m, v, before = first.values(), second.values(), p.clone()
        optim.adamw([p], [g], [first], [second], step=step, lr=0.01, betas=betas, eps=1e-15,
                    weight_decay=0.0)
        want, tolerance = reference(before, g, m, v, step, 0.01, betas, 1e-15, 0.0)
        close(p, want[0], tolerance[0], "p")
        # single fp32 operations, in the order that the codes are defined by
        m1 = m * betas[0] + g.float() * (1 - betas[0])
        v1 = v * betas[1] + (g.float() * (1 - betas[1])) * g.float()
        low, high = noise(n, step)
        c, e = rounded_down(m1, 8, low)
        assert torch.equal(first.exponents, e)
        assert torch.equal(first.codes.long() & 127, c)
        assert torch.equal(first.codes >= 128, m1 < 0)
        c, e = rounded_down(v1.sqrt(), 16, high)
        assert torch.equal(second.exponents, e)
        assert torch.equal(second.codes.long(), torch.where(v1 > 0, c.clamp(min=1), c))


def behind(t, offset):
    """The same values from `offset` elements behind an aligned address on."""
    flat = torch.empty(t.numel() + offset, dtype=t.dtype, device=t.device)[offset:]
    return flat.copy_(t.reshape(-1)).view(t.shape)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["all", "p", "g", "m", "v"])
def test_8_bit_steps_of_unaligned_tensors(which, dtype):
    """More tensors than a launch takes, of which any may lie off 16 bytes: the same bits as
    those that lie on them."""
    sizes = [1, 3, 255, 256, 257, 1000, 16384, 16385, 40000] + [130 + i for i in range(100)]
    p = [draw(i, n).to(dtype) for i, n in enumerate(sizes)]
    g = [draw(1000 + i, n).to(dtype) for i, n in enumerate(sizes)]
    first = [optim.Moment8.of(0.1 * draw(2000 + i, n)) for i, n in enumerate(sizes)]
    second = [optim.Moment8.of(draw(3000 + i, n).square(), squared=True)
              for i, n in enumerate(sizes)]

    def moved(name, t, i):
        return behind(t, 1 + i % 7 if which in ("all", name) else 0)

    twins = [moved("p", t, i) for i, t in enumerate(p)], [moved("g", t, i) for i, t in enumerate(g)]
    moments = [[optim.Moment8(moved(name, t.codes, i), moved(name, t.exponents, i), t.squared)
                for i, t in enumerate(group)] for name, group in (("m", first), ("v", second))]
    for step in (1, 9):
        optim.adamw(p, g, first, second, step=step, lr=0.01)
        optim.adamw(*twins, *moments, step=step, lr=0.01)
    for a, c in zip(p, twins[0]):
        assert torch.equal(a, c)
    for group, others in zip((first, second), moments):
        for a, c in zip(group, others):
            assert torch.equal(a.codes, c.codes) and torch.equal(a.exponents, c.exponents)
            assert torch.equal(a.values(), c.values())
    # and encoding and decoding
    for t in (0.1 * draw(1, 1001), draw(2, 1001).square()):
        for squared in (False, True):
            a, c = optim.Moment8.of(t.abs(), squared), optim.Moment8.of(behind(t.abs(), 3), squared)
            assert torch.equal(a.codes, c.codes) and torch.equal(a.exponents, c.exponents)


def test_8_bit_averages_follow_small_steps():
    """A constant gradient: v' moves by a thousandth of what it lacks, less than any
    code's step; over 3000 steps it has to come within a twentieth of its limit."""
    n = 4096
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 3.0, device="cuda")
    first = optim.Moment8.zeros_like(p)
    second = optim.Moment8.of(torch.full((n,), 1.0, device="cuda"), squared=True)
    for step in range(1, 3001):
        optim.adamw([p], [g], [first], [second], step=step, lr=1e-3, weight_decay=0.0)
    # the mean of n independent codes, each within a step (2^-3 of v)
    limit = 9.0 + (1.0 - 9.0) * 0.999 ** 3000
    assert abs(float(second.values().mean()) / limit - 1) < 0.05
    assert abs(float(first.values().mean()) / 3.0 - 1) < 0.05


def test_8_bit_zero_gradients():
    """Values that no gradient ever reached stay, as do those whose gradient stopped."""
    p = draw(1, 3000)
    g = draw(2, 3000) * 2.0 ** (12 * draw(3, 3000))
    g[::3] = 0.0
    first, second = optim.Moment8.zeros_like(p), optim.Moment8.zeros_like(p, squared=True)
    before = p.clone()
    optim.adamw([p], [g], [first], [second], step=1, lr=0.1, eps=1e-15, weight_decay=0.0)
    assert torch.equal(p[::3], before[::3])
    for step in range(2, 60):
        was = p.clone()
        optim.adamw([p], [torch.zeros_like(g)], [first], [second], step=step, lr=0.1, eps=1e-15,
                    weight_decay=0.0)
        # |m'| / root' of decaying averages: never above that of a single gradient, 10 at
        # most, by what a step of either code may add (9 / 8 and a vanished root's two)
        assert float((p - was).abs().max()) <= 0.1 * 10 * 2.5
    assert p.isfinite().all()


def test_8_bit_non_finite_gradients():
    p = torch.zeros(1000, device="cuda")
    first, second = optim.Moment8.zeros_like(p), optim.Moment8.zeros_like(p, squared=True)
    g = torch.ones(1000, device="cuda")
    g[300] = float("nan")
    optim.adamw([p], [g], [first], [second], step=1, lr=0.1)
    assert p.isnan().nonzero().flatten().tolist() == [300]
    run = torch.arange(1000, device="cuda") // RUN == 1
    assert first.values().isnan()[run].all() and second.values().isnan()[run].all()
    assert first.values()[~run].isfinite().all()


# ---- the optimizer -----------------------------------------------------------------------

def scene(seed, n=500, dtype=torch.float32):
    return [draw(seed + i, n, *s).to(dtype).requires_grad_()
            for i, s in enumerate([(3,), (4,), (3,), (), (1, 3), (15, 3)])]


def set_grads(params, seed):
    for i, p in enumerate(params):
        p.grad = draw(seed + i, *p.shape).to(p.dtype)


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_makes_the_functional_steps(bits):
    params = scene(1)
    twins = [p.detach().clone() for p in params]
    lrs = [1e-2, 2e-3, 5e-3, 5e-2, 2.5e-3, 1e-4]
    optimizer = optim.AdamW([{"params": [p], "lr": lr} for p, lr in zip(params, lrs)],
                            eps=1e-15, weight_decay=0.01, state_bits=bits)
    if bits == 8:
        moments = [[optim.Moment8.zeros_like(p, squared) for p in twins]
                   for squared in (False, True)]
    else:
        moments = [[torch.zeros_like(p) for p in twins] for _ in range(2)]
    for step in range(1, 4):
        set_grads(params, 50 * step)
        versions = [p._version for p in params]
        optimizer.step()
        assert all(p._version > v for p, v in zip(params, versions))
        optim.adamw(twins, [p.grad for p in params], *moments, step=step, lr=lrs, eps=1e-15,
                    weight_decay=0.01)
        for p, t in zip(params, twins):
            assert torch.equal(p, t)
    for i, p in enumerate(params):
        m, v = optimizer.moments(p)
        want = [group[i].values() if bits == 8 else group[i] for group in moments]
        assert torch.equal(m, want[0]) and torch.equal(v, want[1])


def test_optimizer_against_torch():
    """Over ten steps of the same gradients; each step's update is off by some 2^-20 of
    itself, ten of at most lr 1.5 each."""
    params = scene(2)
    twins = [p.detach().clone().requires_grad_() for p in params]
    ours = optim.AdamW(params, lr=0.01, weight_decay=0.1)
    theirs = torch.optim.AdamW(twins, lr=0.01, weight_decay=0.1)
    for step in range(10):
        set_grads(params, 70 * step)
        for p, t in zip(params, twins):
            t.grad = p.grad.clone()
        ours.step()
        theirs.step()
    for p, t in zip(params, twins):
        assert float((p - t).abs().max()) <= 10 * (0.015 * 2.0 ** -19
                                                   + float(t.abs().max()) * 4 * U)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_state_dict(bits, dtype):
    params = scene(3, dtype=dtype)
    optimizer = optim.AdamW(params, lr=0.01, state_bits=bits)
    for step in range(2):
        set_grads(params, 30 * step)
        optimizer.step()
    twins = [p.detach().clone().requires_grad_() for p in params]
    twin = optim.AdamW(twins, lr=0.5, state_bits=bits)
    twin.load_state_dict(copy.deepcopy(optimizer.state_dict()))
    set_grads(params, 90)
    set_grads(twins, 90)
    optimizer.step()
    twin.step()
    for p, t in zip(params, twins):
        assert torch.equal(p, t)
        for a, b in zip(optimizer.moments(p), twin.moments(t)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["host", "capturable", "fused"])
def test_state_of_torch(kind, dtype, bits):
    """A checkpoint of torch.optim.AdamW is followed by the step that its formula asks for."""
    params = scene(9, dtype=dtype)
    theirs = torch.optim.AdamW([{"params": params[:3], "lr": 0.01},
                                {"params": params[3:], "lr": 0.002}], weight_decay=0.1,
                               **({kind: True} if kind != "host" else {}))
    for step in range(5):
        set_grads(params, 40 * step)
        theirs.step()
    saved = copy.deepcopy(theirs.state_dict())
    ours = optim.AdamW([{"params": params[:3]}, {"params": params[3:]}], lr=0.5, state_bits=bits)
    ours.load_state_dict(saved)
    for i, group in enumerate(ours.param_groups):
        assert group["lr"] == (0.01, 0.002)[i] and group["state_bits"] == bits
    moments = [tuple(t.clone() for t in ours.moments(p)) for p in params]
    for i, (p, (m, v)) in enumerate(zip(params, moments)):
        state = saved["state"][i]
        if bits == 32:
            assert torch.equal(m, state["exp_avg"].float())
            assert torch.equal(v, state["exp_avg_sq"].float())
        step = ours.state[p]["step"]
        assert int(step) == 5 and isinstance(step, torch.Tensor) == (kind == "capturable")
    before = [p.detach().clone() for p in params]
    set_grads(params, 900)
    ours.step()
    for p, b, (m, v), lr in zip(params, before, moments, [0.01] * 3 + [0.002] * 3):
        want, tolerance = reference(b, p.grad, m, v, 6, lr, (0.9, 0.999), 1e-8, 0.1)
        close(p.detach(), want[0], tolerance[0], "p")
        assert int(ours.state[p]["step"]) == 6
    # a state of its own that has been through torch.optim's again
    twin = optim.AdamW([{"params": params[:3]}, {"params": params[3:]}])
    twin.load_state_dict(copy.deepcopy(ours.state_dict()))
    for p in params:
        for a, c in zip(ours.moments(p), twin.moments(p)):
            assert torch.equal(a, c)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_read_on_the_host(bits):
    """What torch.load(map_location="cpu") gives, a learning rate on the device with it."""
    params = scene(15)
    optimizer = optim.AdamW(params, lr=torch.tensor(0.01, device="cuda"), state_bits=bits,
                            capturable=True)
    set_grads(params, 1)
    optimizer.step()
    file = io.BytesIO()
    torch.save(optimizer.state_dict(), file)
    file.seek(0)
    twins = [p.detach().clone().requires_grad_() for p in params]
    twin = optim.AdamW(twins, state_bits=bits)
    twin.load_state_dict(torch.load(file, map_location="cpu"))
    set_grads(params, 2)
    set_grads(twins, 2)
    optimizer.step()
    twin.step()
    assert twin.param_groups[0]["lr"].is_cuda and twin.param_groups[0]["capturable"]
    for p, t in zip(params, twins):
        assert torch.equal(p, t) and int(twin.state[t]["step"]) == 2
        for a, c in zip(optimizer.moments(p), twin.moments(t)):
            assert torch.equal(a, c)


def test_states_that_are_refused_change_nothing():
    params = scene(10)
    twins = [p.detach().clone().requires_grad_() for p in params]
    theirs = torch.optim.AdamW(twins, amsgrad=True)
    ours = optim.AdamW(params, lr=0.03)
    for p in (*params, *twins):
        p.grad = torch.ones_like(p)
    theirs.step()
    ours.step()
    before = [tuple(t.clone() for t in ours.moments(p)) for p in params]
    with pytest.raises(ValueError, match="amsgrad"):
        ours.load_state_dict(theirs.state_dict())
    assert ours.param_groups[0]["lr"] == 0.03
    for p, was in zip(params, before):
        assert all(torch.equal(a, c) for a, c in zip(ours.moments(p), was))


def test_hooks_of_a_loaded_state():
    """A hook that changes what is loaded is heard, one behind it sees the result."""
    p, q = draw(1, 40).requires_grad_(), draw(2, 40).requires_grad_()
    ours, twin = optim.AdamW([p]), optim.AdamW([q])
    p.grad = torch.ones_like(p)
    ours.step()
    seen = []
    twin.register_load_state_dict_pre_hook(
        lambda _, s: {**s, "state": {0: {**s["state"][0], "step": 41}}})
    twin.register_load_state_dict_post_hook(lambda o: seen.append(o.state[q]["step"]))
    twin.load_state_dict(ours.state_dict())
    assert seen == [41] and twin.state[q]["step"] == 41
    assert torch.equal(twin.moments(q)[0], ours.moments(p)[0])


@pytest.mark.parametrize("bits", [32, 8])
def test_fewer_and_more_gaussians(bits):
    """What a densification does: new tensors take over rows of the moments."""
    p = draw(4, 300, 3).requires_grad_()
    optimizer = optim.AdamW([p], lr=0.01, state_bits=bits)
    p.grad = draw(5, 300, 3)
    optimizer.step()
    m, v = optimizer.moments(p)
    keep = torch.arange(0, 300, 2, device="cuda")
    q = torch.cat([p.detach()[keep], p.detach()[:7]]).requires_grad_()
    state = optimizer.state.pop(p)
    optimizer.param_groups[0]["params"] = [q]
    optimizer.state[q] = {"step": state["step"]}
    optimizer.set_moments(q, *(torch.cat([t[keep], torch.zeros(7, 3, device="cuda")])
                               for t in (m, v)))
    got = optimizer.moments(q)
    for a, t, mantissa in ((got[0], m, 8), (got[1], v, 16)):
        want = torch.cat([t[keep], torch.zeros(7, 3, device="cuda")])
        assert bool(((a - want).abs() <= (0 if bits == 32 else 2 * want.abs() / mantissa
                                          + float(want.abs().max()) * 2.0 ** -17)).all())
    q.grad = draw(6, 157, 3)
    optimizer.step()
    assert optimizer.state[q]["step"] == 2 and q.isfinite().all()


def test_parameters_without_gradients_stay():
    params = scene(5)
    optimizer = optim.AdamW(params, lr=0.1)
    set_grads(params, 1)
    params[2].grad = None
    before = params[2].detach().clone()
    optimizer.step()
    assert torch.equal(params[2], before) and params[2] not in optimizer.state
    optimizer.zero_grad()
    was = [p.detach().clone() for p in params]
    optimizer.step()
    assert all(torch.equal(p, w) for p, w in zip(params, was))


def test_empty_parameters():
    p, q = torch.zeros(0, 3, device="cuda", requires_grad=True), draw(1, 5).requires_grad_()
    for bits in (8, 32):
        optimizer = optim.AdamW([p, q], state_bits=bits)
        p.grad, q.grad = torch.zeros_like(p), torch.ones_like(q)
        optimizer.step()
        assert optimizer.moments(p)[0].shape == (0, 3)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps(bits):
    """Two captured optimizers replayed in turn make the steps of eager ones; a learning
    rate on the device is followed."""
    lr = torch.tensor(0.01, device="cuda")
    runs = []
    for seed in (6, 7):
        params = scene(seed)
        twins = [p.detach().clone().requires_grad_() for p in params]
        ours = optim.AdamW(params, lr=lr, state_bits=bits, capturable=True)
        eager = optim.AdamW(twins, lr=float(lr), state_bits=bits)
        set_grads(params, 10 * seed)
        ours.step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ours.step()
        runs.append((graph, params, twins, ours, eager, seed))
    for graph, params, twins, ours, eager, seed in runs:
        for p, t in zip(params, twins):
            t.grad = p.grad
        eager.step()  # the step before the capture
    for step in range(3):
        lr.fill_(0.01 * (step + 1))
        for graph, params, twins, ours, eager, seed in runs:
            for i, p in enumerate(params):
                p.grad.copy_(draw(1000 * step + seed + i, *p.shape))
            graph.replay()
            # of the tensor's value, which is the nearest fp32 number
            eager.param_groups[0]["lr"] = float(lr)
            eager.step()
    for graph, params, twins, ours, eager, seed in runs:
        for p, t in zip(params, twins):
            assert torch.equal(p, t)
            assert int(ours.state[p]["step"]) == 4
            for a, b in zip(ours.moments(p), eager.moments(t)):
                assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [32, 8])
def test_moments_set_between_replays(bits):
    """A captured step holds the state's tensors: what is set later is what it goes on from."""
    p = draw(11, 700, 3).requires_grad_()
    p.grad = draw(12, 700, 3)
    optimizer = optim.AdamW([p], lr=0.01, state_bits=bits, capturable=True)
    optimizer.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        optimizer.step()
    graph.replay()
    m, v = (t.clone() for t in optimizer.moments(p))
    optimizer.set_moments(p, 0.5 * m, 2.0 * v)
    m, v = (t.clone() for t in optimizer.moments(p))
    before = p.detach().clone()
    graph.replay()
    want, tolerance = reference(before, p.grad, m, v, 3, 0.01, (0.9, 0.999), 1e-8, 0.01)
    close(p.detach(), want[0], tolerance[0], "p")
    if bits == 32:
        for got, w, t in zip(optimizer.moments(p), want[1:], tolerance[1:]):
            close(got, w, t, "moment")
    else:  # one step of a code below, at most
        for got, w, mantissa in zip(optimizer.moments(p), want[1:], (8, 8)):
            assert bool(((got - w).abs() <= 2.0 * w.abs() / mantissa
                         + float(w.abs().max()) * 2.0 ** -14).all())
            assert not torch.equal(got, m)
    # its own tensors, one in the other's place
    first, second = optimizer.moments(p)
    swapped = second.clone(), first.abs()
    optimizer.set_moments(p, second, first.abs())
    got = optimizer.moments(p)
    if bits == 32:
        assert torch.equal(got[0], swapped[0]) and torch.equal(got[1], swapped[1])


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_that_becomes_capturable(bits):
    """A state that counted on the host, in a group that has been made capturable."""
    p, q = draw(13, 300).requires_grad_(), draw(13, 300).requires_grad_()
    p.grad, q.grad = draw(14, 300), draw(14, 300)
    ours = optim.AdamW([p], lr=0.01, state_bits=bits)
    eager = optim.AdamW([q], lr=0.01, state_bits=bits)
    ours.step()
    ours.param_groups[0]["capturable"] = True
    with pytest.raises(RuntimeError, match="before a step is captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ours.step()
    ours.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ours.step()
    for _ in range(3):
        graph.replay()
    for _ in range(5):
        eager.step()
    assert torch.equal(p, q) and int(ours.state[p]["step"]) == 5


def test_capture_refusals():
    p = draw(1, 8).requires_grad_()
    p.grad = torch.ones_like(p)
    for capturable, message in ((False, "capturable=True"), (True, "before a step is captured")):
        optimizer = optim.AdamW([p], capturable=capturable)
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match=message):
            with torch.cuda.graph(graph):
                optimizer.step()


def test_another_stream():
    params = scene(8, n=20000)
    twins = [p.detach().clone() for p in params]
    grads = [draw(i, *p.shape) for i, p in enumerate(twins)]
    zeros = [[torch.zeros_like(p) for p in twins] for _ in range(4)]
    optim.adamw([p.detach() for p in params], grads, *zeros[:2], step=1, lr=0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        optim.adamw(twins, grads, *zeros[2:], step=1, lr=0.1)
    torch.cuda.synchronize()
    for p, t in zip(params, twins):
        assert torch.equal(p.detach(), t)


def test_refusals():
    p, g = draw(1, 10), draw(2, 10)
    m, v = torch.zeros(10, device="cuda"), torch.zeros(10, device="cuda")

    def refused(message, *args, **options):
        before = p.clone()
        with pytest.raises(ValueError, match=message):
            optim.adamw(*args, **{"step": 1, "lr": 0.1, **options})
        assert torch.equal(p, before)

    refused("same length", [p], [g], [m], [])
    refused("listed twice", [p, p], [g, g], [m, m], [v, v])
    refused("listed twice", [p, p.clone()], [g, g], [m, m], [v, v.clone()])
    refused("listed twice", [p], [g], [m], [m])
    first, second = optim.Moment8.zeros_like(p), optim.Moment8.zeros_like(p, squared=True)
    refused("listed twice", [p], [g], [first],
            [optim.Moment8(second.codes, first.exponents, squared=True)])
    refused("contiguous", [draw(3, 4, 5).t()], [draw(4, 5, 4)], [m], [v])
    refused("gradients must have", [p], [g.half()], [m], [v])
    refused("gradients must have", [p], [g[:9]], [m], [v])
    refused("moments must be", [p], [g], [m.half()], [v])
    refused("moments must be", [p], [g], [m[:9]], [v])
    refused("same number of bits", [p], [g], [m], [optim.Moment8.zeros_like(p, squared=True)])
    refused("squared", [p], [g], [optim.Moment8.zeros_like(p)], [optim.Moment8.zeros_like(p)])
    refused("CUDA", [p.cpu()], [g.cpu()], [m.cpu()], [v.cpu()])
    refused("step must be", [p], [g], [m], [v], step=0)
    refused("step must be", [p], [g], [m], [v], step=torch.ones((), device="cuda"))
    refused("lr must be", [p], [g], [m], [v], lr=math.nan)
    refused("lr must be", [p], [g], [m], [v], lr=torch.ones((), device="cuda").double())
    refused("one for each", [p], [g], [m], [v], lr=[0.1, 0.2])
    refused("dense", [p], [g.to_sparse()], [m], [v])


def test_gradients_that_are_written():
    """Other blocks of the same launch would read them while they change."""
    p, q, g = draw(1, 10), draw(2, 10), draw(3, 10)
    moments = [torch.zeros(10, device="cuda") for _ in range(4)]
    before = p.clone(), q.clone()
    for grads in ([q, g], [g, p], [g, moments[2]]):
        with pytest.raises(ValueError, match="a gradient is"):
            optim.adamw([p, q], grads, moments[:2], moments[2:], step=1, lr=0.1)
    assert torch.equal(p, before[0]) and torch.equal(q, before[1])
    optim.adamw([p, q], [g, g], moments[:2], moments[2:], step=1, lr=0.1)
    assert not torch.equal(p, before[0]) and not torch.equal(q, before[1])
