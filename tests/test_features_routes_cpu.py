"""Feature operators without a GPU: the calls that reach them by torch.ops, under
forward-mode differentiation and while a program is traced."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from dsl_splat_b200 import features

ops = torch.ops.splat200


def fake(*shape, dtype=torch.float32, device="cuda"):
    return torch.empty(shape, device=device, dtype=dtype)


LINEAR = dict(x=(6, 3), weight=(4, 3), bias=(4,), residual=(6, 4))


def linear_tensors(change):
    dtypes = {m: change.get(m + "_dtype", torch.float32) for m in LINEAR}
    return [fake(*change.get(m, LINEAR[m]), dtype=dtypes[m],
                 device=change.get(m + "_device", "cuda")) for m in LINEAR]


LINEAR_CHANGES = [
    (dict(x=(8, 6), weight=(4, 3)), "weight must have shape"),
    (dict(weight=(4, 5)), "weight must have shape"),
    (dict(weight=(4,)), r"weight must be \(N,K\)"),
    (dict(bias=(1,)), "bias must have shape"),
    (dict(residual=(3, 4)), "residual must have shape"),
    (dict(weight_dtype=torch.bfloat16), "weight must have x's dtype"),
    (dict(bias_dtype=torch.float16), "bias must have x's dtype"),
    (dict(residual_dtype=torch.float64), "residual must have x's dtype"),
    (dict(weight_device="cpu"), "weight must have x's dtype and device"),
    (dict(x_device="cpu"), "x must be a CUDA"),
    (dict(x_dtype=torch.float64), "x must be a CUDA"),
    (dict(x=(1, 70000), weight=(4, 70000), residual=(1, 4)), "65535"),
]


@pytest.mark.parametrize("change, message", LINEAR_CHANGES)
def test_linear_op_refusals(change, message):
    with FakeTensorMode():
        with pytest.raises(ValueError, match=message):
            ops.feature_linear(*linear_tensors(change), "silu")


def test_linear_op_refuses_unknown_activations():
    with FakeTensorMode():
        with pytest.raises(ValueError, match="activation"):
            ops.feature_linear(*linear_tensors({}), "tanh")


@pytest.mark.parametrize("change, message", [
    (dict(x=(8, 6), weight=(4, 3)), "weight must have shape"),
    (dict(bias=(1,)), "bias must have shape"),
    (dict(weight_dtype=torch.bfloat16), "weight must have x's dtype"),
    (dict(upstream=(5, 4)), "upstream must have shape"),
    (dict(upstream_dtype=torch.float16), "upstream must have x's dtype"),
    (dict(activation="tanh"), "activation"),
])
def test_linear_backward_op_refusals(change, message):
    with FakeTensorMode():
        x, weight, bias, _ = linear_tensors(change)
        upstream = fake(*change.get("upstream", (6, 4)),
                        dtype=change.get("upstream_dtype", torch.float32))
        with pytest.raises(ValueError, match=message):
            ops.feature_linear_backward(x, weight, bias, change.get("activation", "silu"), upstream)


NORM_CHANGES = [
    (dict(groups=3), "groups must divide"),
    (dict(groups=0), "groups must be a positive"),
    (dict(eps=-1.0), "eps must be finite"),
    (dict(eps=float("inf")), "eps must be finite"),
    (dict(activation="swish"), "activation"),
    (dict(weight=(7,)), "weight must have shape"),
    (dict(bias=(9,)), "bias must have shape"),
    (dict(weight_dtype=torch.bfloat16), "weight must have x's dtype"),
    (dict(x=(8,)), "x must have"),
    (dict(x_device="cpu"), "x must be a CUDA"),
]


@pytest.mark.parametrize("change, message", NORM_CHANGES)
def test_norm_op_refusals(change, message):
    with FakeTensorMode():
        x = fake(*change.get("x", (2, 5, 8)), device=change.get("x_device", "cuda"))
        weight = fake(*change.get("weight", (8,)), dtype=change.get("weight_dtype", torch.float32))
        bias = fake(*change.get("bias", (8,)))
        with pytest.raises(ValueError, match=message):
            ops.feature_norm(x, change.get("groups", 2), weight, bias, change.get("eps", 1e-5),
                             change.get("activation", "silu"))


@pytest.mark.parametrize("change, message", [
    (dict(groups=3), "groups must divide"),
    (dict(upstream=(2, 4, 8)), "upstream must have shape"),
    (dict(upstream_dtype=torch.float16), "upstream must have x's dtype"),
    (dict(moments=(2, 2, 4)), "moments must be"),
    (dict(moments_dtype=torch.float64), "moments must be"),
    (dict(weight=(7,)), "weight must have shape"),
])
def test_norm_backward_op_refusals(change, message):
    with FakeTensorMode():
        moments = fake(*change.get("moments", (2, 2, 2)),
                       dtype=change.get("moments_dtype", torch.float32))
        upstream = fake(*change.get("upstream", (2, 5, 8)),
                        dtype=change.get("upstream_dtype", torch.float32))
        with pytest.raises(ValueError, match=message):
            ops.feature_norm_backward(fake(2, 5, 8), change.get("groups", 2),
                                      fake(*change.get("weight", (8,))), None, moments, "silu",
                                      upstream)


def test_forward_mode_is_refused():
    with FakeTensorMode(), fwAD.dual_level():
        x, w = fake(6, 3), fake(4, 3)
        dual = fwAD.make_dual(x, torch.ones_like(x))
        for call in (lambda: features.linear(dual, w),
                     lambda: features.linear(x, fwAD.make_dual(w, torch.ones_like(w))),
                     lambda: features.linear(x, w, residual=fwAD.make_dual(fake(6, 4),
                                                                           fake(6, 4))),
                     lambda: features.group_norm(dual[None], 3, spatial_dims=1)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_forward_mode_operators_are_refused():
    with FakeTensorMode(), fwAD.dual_level():
        x, w = fake(6, 3), fake(4, 3)
        dual = fwAD.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.feature_linear(dual, w, None, None, "silu")
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.feature_norm(dual[None], 3, None, None, 1e-5, "silu")


@pytest.mark.parametrize("grad", [False, True])
def test_traced_programs_hold_the_operators(grad):
    def run(x, w, b):
        y = features.linear(x, w, b, activation="silu")
        return features.group_norm(y[None], 2, spatial_dims=1)

    with FakeTensorMode():
        tensors = [fake(*s).requires_grad_(grad) for s in ((6, 3), (4, 3), (4,))]
        graph = make_fx(run)(*tensors)
    called = [n.target for n in graph.graph.nodes if n.op == "call_function"]
    assert ops.feature_linear.default in called
    assert ops.feature_norm.default in called


def test_traced_shapes():
    with FakeTensorMode():
        assert features.linear(fake(2, 5, 3), fake(4, 3)).shape == (2, 5, 4)
        assert features.linear(fake(3), fake(4, 3)).shape == (4,)
        assert features.group_norm(fake(3, 2, 5, 7, 8), 4).shape == (3, 2, 5, 7, 8)
        assert features.group_norm(fake(5, 8), 4, spatial_dims=1).shape == (5, 8)
        assert features.group_norm(fake(0, 4, 4, 8), 4).shape == (0, 4, 4, 8)


def test_norm_refuses_an_eps_that_float32_has_not():
    with FakeTensorMode():
        for eps in (1e-60, 1e60):
            with pytest.raises(ValueError, match="eps must be finite"):
                features.group_norm(fake(1, 3, 4, 8), 2, eps=eps)
