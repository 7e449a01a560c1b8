"""Feature operators on the GPU in recorded programs: torch.compile, torch.jit.trace,
make_fx and CUDA graphs hold them and give what the calls themselves give."""

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from dsl_splat_b200 import features
from test_features_gpu import DTYPES, draws

pytestmark = pytest.mark.gpu


def layers(x, w, b, g):
    y = features.linear(x, w, b, activation="silu")
    y = features.group_norm(y, 4, g, activation="gelu")
    return features.linear(y, w[:, :24], residual=y, activation="none")


def tensors(dtype, grad):
    normal = draws(51)
    return [normal(*s, dtype=dtype).requires_grad_(grad)
            for s in ((2, 9, 11, 35), (24, 35), (24,), (24,))]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled(backend, dtype):
    torch._dynamo.reset()
    run = torch.compile(layers, backend=backend, fullgraph=True)
    for grad in (False, True):
        args = tensors(dtype, grad)
        want, got = layers(*args), run(*args)
        assert torch.equal(got, want)
        if grad:
            dy = torch.ones_like(want)
            for a, c in zip(torch.autograd.grad(got, args, dy),
                            torch.autograd.grad(want, args, dy)):
                assert torch.equal(a, c)


def test_traced():
    args = tensors(torch.bfloat16, False)
    other = [t * 0.5 for t in args]
    for run in (torch.jit.trace(layers, args, check_trace=False), make_fx(layers)(*args)):
        for inputs in (args, other):
            assert torch.equal(run(*inputs), layers(*inputs))


def test_under_torch_func():
    """torch.func's transforms are refused, not answered without the operator."""
    x, w, b, _ = tensors(torch.float32, False)
    for run in (lambda: torch.func.jvp(lambda v: features.linear(v, w, b), (x,), (x,)),
                lambda: torch.func.vmap(lambda v: features.linear(v, w, b))(x),
                lambda: torch.func.grad(lambda v: features.linear(v, w, b).sum())(x),
                lambda: torch.func.vmap(lambda v: features.group_norm(v, 5))(x)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            run()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, k, n, act", [(700, 512, 264, "gelu"), (700, 301, 200, "silu"),
                                          (17000, 301, 33, "sigmoid"), (900, 64, 48, "silu"),
                                          (40, 20001, 9, "silu"), (900, 35, 48, "relu")])
def test_captured_layers(m, k, n, act, dtype):
    """One training step of a layer, captured and replayed on other inputs
    beside an eager one on another stream."""
    normal = draws(52)
    w, b, dy = (normal(*s, dtype=dtype) for s in ((n, k), (n,), (m, n)))
    inputs = [normal(m, k, dtype=dtype) for _ in range(3)]

    def step(x):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = features.linear(*leaves, activation=act)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    want = [[t.clone() for t in step(x)] for x in inputs]
    static = inputs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for i, x in enumerate(inputs):
        static.copy_(x)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            beside = step(inputs[i - 1])
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want[i]))
        assert all(torch.equal(a, c) for a, c in zip(beside, want[i - 1]))
