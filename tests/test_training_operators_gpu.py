"""The operators that train features, together and as they are used: a scene whose
Gaussians share a codebook of features, rendered, normalised and classified per pixel,
and stepped with AdamW."""

import pytest
import torch
import torch.nn.functional as F

from dsl_splat_b200 import aaa, features, gs3d, optim, rade
from dsl_splat_b200.scenes import make_scene
from test_features_gpu import draws

pytestmark = pytest.mark.gpu

WORDS = 300


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


class Scene:
    def __init__(self, channels=16, n=3000, codes=200):
        normal = draws(1)
        s = make_scene(1, n=n, width=96, height=64)
        self.size = s.width, s.height
        self.sh = s.sh_coeffs.cuda()
        self.geometry = [t.cuda() for t in (s.means, s.quats, s.scales, s.opacities)]
        self.cameras = [t.cuda() for t in (s.viewmats, s.Ks)]
        g = torch.Generator().manual_seed(2)
        self.ids = torch.randint(0, codes, (n,), generator=g).cuda()
        self.labels = torch.randint(0, WORDS, (1, s.height, s.width), generator=g).cuda()
        self.labels[:, ::7] = -100
        f32 = torch.float32
        self.table = normal(codes, channels, dtype=f32)
        self.norm = [normal(channels, dtype=f32, scale=0.2, shift=1.0),
                     normal(channels, dtype=f32, scale=0.2)]
        self.hidden = [normal(64, channels, dtype=f32, scale=0.25), normal(64, dtype=f32)]
        self.head = [normal(WORDS, 64, dtype=f32, scale=0.25), normal(WORDS, dtype=f32)]
        self.leaves = [t.requires_grad_()
                       for t in (self.table, *self.norm, *self.hidden, *self.head)]

    def render(self, rasterize, extra):
        return rasterize(*self.geometry, *self.cameras, *self.size, sh_coeffs=self.sh,
                         extra_features=extra).extra_features

    def decoder(self):
        return features.FeatureDecoder(features.LayerNorm(*self.norm, activation="silu"),
                                       features.Linear(*self.hidden, "gelu"),
                                       features.Linear(*self.head))

    def loss(self, rasterize):
        extra = features.embedding(self.ids, self.table, scale=0.5)
        return self.decoder().cross_entropy(self.render(rasterize, extra), self.labels)


@pytest.mark.parametrize("rasterize", [gs3d.rasterize, rade.rasterize, aaa.rasterize])
def test_a_labelled_scene(rasterize):
    """Loss and gradients against the same in 64 bits around the rasteriser.

    Every stage is off by a few 2^-23 of sums of at most 64 values, relative 2^-17 of its
    2-norm; four of them, and the rasteriser's own backward (1e-3 where its atomics'
    order shows, 1e-5 else) stay below 1e-4 but for the codebook's, 1e-3."""
    s = Scene()
    loss = s.loss(rasterize)
    grads = torch.autograd.grad(loss, s.leaves)
    wide = [t.detach().double().requires_grad_() for t in s.leaves]
    table, nw, nb, hw, hb, vw, vb = wide
    extra = (0.5 * table[s.ids]).float()
    image = s.render(rasterize, extra)
    held = image.detach().double().requires_grad_()
    x = F.silu(F.layer_norm(held, (16,), nw, nb, 1e-5))
    z = F.gelu(x @ hw.t() + hb) @ vw.t() + vb
    want = F.cross_entropy(z.reshape(-1, WORDS), s.labels.reshape(-1), ignore_index=-100)
    assert abs(float(loss.detach()) / float(want.detach()) - 1) < 1e-5
    want.backward()
    image.backward(held.grad.float())
    for got, t, most in zip(grads, wide, (1e-3, *[1e-4] * 6)):
        assert rel(got, t.grad) < most


@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps(bits):
    """Three steps: parameters follow the formula for the gradients that they were given
    (12 operations of 2^-24, of a step of at most lr times 10 in three steps), eager and
    captured alike."""
    s = Scene()
    lrs = [1e-2, 1e-3, 1e-3, 1e-3, 1e-3, 1e-3, 1e-3]
    optimizer = optim.AdamW([{"params": [p], "lr": lr} for p, lr in zip(s.leaves, lrs)],
                            weight_decay=0.01, state_bits=bits)
    for step in range(1, 4):
        before = [p.detach().double() for p in s.leaves]
        moments = ([tuple(t.double() for t in optimizer.moments(p)) for p in s.leaves]
                   if step > 1 else [(0.0, 0.0)] * len(s.leaves))
        optimizer.zero_grad()
        s.loss(gs3d.rasterize).backward()
        optimizer.step()
        for p, b, (m, v), lr in zip(s.leaves, before, moments, lrs):
            g = p.grad.double()
            m, v = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g * g
            want = b * (1 - lr * 0.01) - lr * (m / (1 - 0.9 ** step)) / (
                (v / (1 - 0.999 ** step)).sqrt() + 1e-8)
            assert float((p.detach() - want).abs().max()) <= 2.0 ** -20 * (
                10 * lr + float(b.abs().max()))


def test_captured_training_step():
    """The decoder's part of a step in a CUDA graph, replayed, against eager steps."""
    def make():
        s = Scene()
        image = s.render(gs3d.rasterize, s.table.detach()[s.ids])
        leaves = [t.detach().clone().requires_grad_() for t in s.leaves[1:]]
        norm, hidden, head = leaves[:2], leaves[2:4], leaves[4:]
        decoder = features.FeatureDecoder(features.LayerNorm(*norm, activation="silu"),
                                          features.Linear(*hidden, "gelu"),
                                          features.Linear(*head))
        optimizer = optim.AdamW(leaves, lr=1e-2, capturable=True)

        def step():
            loss = decoder.cross_entropy(image, s.labels)
            for p, g in zip(leaves, torch.autograd.grad(loss, leaves)):
                if p.grad is None:
                    p.grad = g
                else:
                    p.grad.copy_(g)
            optimizer.step()
            return loss.detach()

        return leaves, step, (s, image, decoder, optimizer)

    eager, step, _keep = make()
    want = [float(step()) for _ in range(4)]
    captured, step, _kept = make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [float(step())]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            loss = step()
        for _ in range(3):
            graph.replay()
            got.append(float(loss))
    torch.cuda.synchronize()
    assert got == want
    for p, q in zip(captured, eager):
        assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_compiled_programs(dtype):
    """What torch.compile records of the operators gives what the calls give."""
    normal = draws(5)
    ids = torch.arange(500, device="cuda") % 37
    table, w, b = (normal(*s, dtype=dtype) for s in ((37, 24), (24,), (24,)))
    words, bias = normal(90, 24, dtype=dtype), normal(90, dtype=dtype)
    target = torch.arange(500, device="cuda") % 90

    def run(table, w, b, words, bias):
        x = features.layer_norm(features.embedding(ids, table, scale=0.5), w, b,
                                activation="silu")
        return features.linear_cross_entropy(x, words, target, bias)

    results = []
    for call in (run, torch.compile(run, backend="aot_eager", fullgraph=True)):
        leaves = [t.detach().clone().requires_grad_() for t in (table, w, b, words, bias)]
        loss = call(*leaves)
        loss.backward()
        results.append([loss.detach(), *[t.grad for t in leaves]])
    for got, want in zip(*results):
        assert torch.equal(got, want)


def test_operators_by_name():
    """torch.ops.splat200 gives what the functions give."""
    ops = torch.ops.splat200
    normal = draws(6)
    x, w, b, dy = (normal(*s, dtype=torch.float32) for s in ((50, 24), (24,), (24,), (50, 24)))
    assert torch.equal(ops.feature_layer_norm(x, w, b, 1e-5, "silu"),
                       features.layer_norm(x, w, b, activation="silu"))
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(features.layer_norm(*leaves, activation="silu"), leaves, dy)
    for g, h in zip(grads, ops.feature_layer_norm_backward(x, w, b, 1e-5, "silu", dy)):
        assert torch.equal(g, h)
    ids = torch.arange(50, device="cuda") % 7
    leaf = x[:7].detach().requires_grad_()
    y = features.embedding(ids, leaf, scale=0.3)
    assert torch.equal(ops.feature_embedding(ids, x[:7], 0.3), y)
    assert torch.equal(ops.feature_embedding_backward(ids, 7, 0.3, dy),
                       torch.autograd.grad(y, leaf, dy)[0])
    words, bias, target = normal(90, 24, dtype=torch.float32), normal(90, dtype=torch.float32), ids
    loss, moments, counted = ops.feature_entropy(x, words, target, bias, -100, "mean")
    leaves = [t.detach().requires_grad_() for t in (x, words, bias)]
    want = features.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2])
    assert torch.equal(loss, want) and float(counted) == 50
    up = torch.tensor(2.0, device="cuda")
    for g, h in zip(torch.autograd.grad(want, leaves, up),
                    ops.feature_entropy_backward(x, words, target, bias, -100, "mean", moments,
                                                 counted, up)):
        assert torch.equal(g, h)


def test_offsets_beyond_32_bits():
    """The last rows of more than 2^31 values are those that they are on their own."""
    rows, tail = (1 << 25) + 1001, 700
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.empty(rows, 64, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    end = x[-tail:].clone()
    w, b = x[0].clone(), x[1].clone()

    def norm(t, dy):
        t = t.detach().requires_grad_()
        y = features.layer_norm(t, w, b, activation="silu")
        return y.detach(), torch.autograd.grad(y, t, dy)[0]

    for whole, alone in zip(norm(x, x), norm(end, end)):
        assert torch.equal(whole[-tail:], alone)

    words = x[:40].clone()
    target = torch.randint(0, 40, (rows,), device="cuda", generator=g, dtype=torch.int32)

    def entropy(t, target):
        t = t.detach().requires_grad_()
        loss = features.linear_cross_entropy(t, words, target, reduction="none")
        return loss.detach(), torch.autograd.grad(loss.sum(), t)[0]

    for whole, alone in zip(entropy(x, target), entropy(end, target[-tail:].clone())):
        assert torch.equal(whole[-tail:], alone)

    table = x[:40].clone().requires_grad_()
    y = features.embedding(target, table)
    assert torch.equal(y.detach()[-tail:], table.detach()[target[-tail:]])
    # whole numbers below 2^24, whose sums in fp32 are exact
    got, = torch.autograd.grad(y, table, torch.ones_like(y))
    count = torch.bincount(target.long(), minlength=40)
    assert torch.equal(got, count.to(got.dtype)[:, None].expand_as(got))
    del y

    def step(p, g):
        m, v = torch.zeros_like(p, dtype=torch.float32), torch.ones_like(p, dtype=torch.float32)
        optim.adamw([p], [g], [m], [v], step=3, lr=0.1)
        return p[-tail:], m[-tail:], v[-tail:]

    gradient = x.flip(0)
    alone = step(end.clone(), gradient[-tail:].clone())
    assert all(torch.equal(a, c) for a, c in zip(step(x, gradient), alone))
