"""Feature operators without a GPU: what they refuse, the shapes of their
torch.ops forms and the C entry points' status codes."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from dsl_splat_b200 import features
from dsl_splat_b200._native import lib


def test_linear_refuses_host_tensors():
    with pytest.raises(ValueError, match="x must be a CUDA"):
        features.linear(torch.zeros(2, 3), torch.zeros(4, 3))


def test_group_norm_refuses_host_tensors():
    with pytest.raises(ValueError, match="x must be a CUDA"):
        features.group_norm(torch.zeros(2, 3, 4, 8), 2)


@pytest.mark.parametrize("change, message", [
    (dict(activation="tanh"), "activation"),
    (dict(weight=(4, 5)), "weight must have shape"),
    (dict(weight=(4,)), r"weight must be \(N,K\)"),
    (dict(weight=(0, 3)), r"weight must be \(N,K\)"),
    (dict(bias=(3,)), "bias must have shape"),
    (dict(residual=(2, 3)), "residual must have shape"),
    (dict(weight_dtype=torch.bfloat16), "weight must have x's dtype"),
    (dict(dtype=torch.float64), "x must be a CUDA"),
    (dict(x=()), "x must have a last dimension"),
    (dict(x=(2, 0), weight=(4, 0)), "x must have a last dimension"),
    (dict(x=(1, 70000), weight=(4, 70000)), "65535"),
])
def test_linear_refusals(change, message):
    with FakeTensorMode():
        dtype = change.get("dtype", torch.float32)
        x = torch.empty(change.get("x", (2, 3)), device="cuda", dtype=dtype)
        w = torch.empty(change.get("weight", (4, 3)), device="cuda",
                        dtype=change.get("weight_dtype", dtype))
        extra = {m: torch.empty(change[m], device="cuda", dtype=dtype)
                 for m in ("bias", "residual") if m in change}
        with pytest.raises(ValueError, match=message):
            features.linear(x, w, activation=change.get("activation", "relu"), **extra)


@pytest.mark.parametrize("change, message", [
    (dict(activation="swish"), "activation"),
    (dict(groups=3), "groups must divide"),
    (dict(groups=0), "groups must be a positive"),
    (dict(groups=True), "groups must be a positive"),
    (dict(eps=0.0), "eps must be finite"),
    (dict(eps=float("nan")), "eps must be finite"),
    (dict(spatial_dims=0), "spatial_dims"),
    (dict(spatial_dims=4), "spatial_dims"),
    (dict(weight=(7,)), "weight must have shape"),
    (dict(bias=(1, 8)), "bias must have shape"),
])
def test_group_norm_refusals(change, message):
    with FakeTensorMode():
        x = torch.empty(1, 3, 4, 8, device="cuda")
        extra = {m: torch.empty(change[m], device="cuda") for m in ("weight", "bias")
                 if m in change}
        options = {m: change[m] for m in ("eps", "activation", "spatial_dims") if m in change}
        with pytest.raises(ValueError, match=message):
            features.group_norm(x, change.get("groups", 2), **extra, **options)


def test_decoder_refuses_other_layers():
    with pytest.raises(ValueError, match="Linear and GroupNorm"):
        features.FeatureDecoder(torch.nn.Identity())
    with pytest.raises(ValueError, match="Linear and GroupNorm"):
        features.FeatureDecoder()


def test_fake_shapes():
    with FakeTensorMode():
        x = torch.empty(10, 35, device="cuda", dtype=torch.bfloat16)
        w = torch.empty(6, 35, device="cuda", dtype=torch.bfloat16)
        y = torch.ops.splat200.feature_linear(x, w, None, None, "silu")
        assert y.shape == (10, 6) and y.dtype == torch.bfloat16
        dx, dw, db = torch.ops.splat200.feature_linear_backward(x, w, None, "silu", y)
        assert dx.shape == x.shape and dw.shape == w.shape and db.shape == (6,)
        v = torch.empty(2, 50, 12, device="cuda", dtype=torch.float16)
        y, moments = torch.ops.splat200.feature_norm(v, 3, None, None, 1e-5, "none")
        assert y.shape == v.shape and moments.shape == (2, 2, 3)
        assert moments.dtype == torch.float32
        dx, dw, db = torch.ops.splat200.feature_norm_backward(v, 3, None, None, moments, "none",
                                                              y)
        assert dx.shape == v.shape and dw.shape == db.shape == (12,)


def test_entry_points_refuse_before_any_launch():
    before = lib.splat_launch_count()
    P = 256  # an aligned address that is never read
    assert lib.splat_feature_linear(3, 1, 1, 1, P, P, None, None, 0, P, None, 0, None) == -1
    assert lib.splat_feature_linear(0, 1, 1, 1, P, P, None, None, 5, P, None, 0, None) == -1
    assert lib.splat_feature_linear(0, 0, 1, 1, P, P, None, None, 0, P, None, 0, None) == -1
    assert lib.splat_feature_linear(0, 1, 1 << 20, 1, P, P, None, None, 0, P, None, 0, None) == -4
    assert lib.splat_feature_linear(0, 1, 1, 1, None, P, None, None, 0, P, None, 0, None) == -1
    assert lib.splat_feature_linear(0, 50000, 300, 9, P, P, None, None, 0, P, None, 0, None) == -5
    assert lib.splat_feature_linear_workspace_bytes(0, 50000, 300, 9) > 50000 * 300 * 6
    assert lib.splat_feature_linear_workspace_bytes(1, 50000, 304, 9) == 16
    assert lib.splat_feature_linear_backward(0, 8, 4, 4, P, P, None, 0, P, P, P, P, P, 0,
                                             None) == -5
    assert lib.splat_feature_linear_backward_workspace_bytes(7, 8, 4, 4, 0) == 0
    assert lib.splat_feature_norm(0, 1, 4, 8, 3, P, None, None, 1e-5, 0, P, P, P, P, 1 << 20,
                                  None) == -1
    assert lib.splat_feature_norm(0, 1, 4, 8, 2, P + 4, None, None, 1e-5, 0, P, P, P, P, 1 << 20,
                                  None) == -1
    assert lib.splat_feature_norm(0, 1, 4, 8, 2, P, None, None, 1e-5, 0, P, P, None, P, 1 << 20,
                                  None) == -1
    assert lib.splat_feature_norm(0, 1, 1 << 20, 8, 2, P, None, None, 1e-5, 0, P, P, P, P, 0,
                                  None) == -5
    assert lib.splat_feature_norm(0, 1, 1 << 32, 8, 2, P, None, None, 1e-5, 0, P, P, P, P, 0,
                                  None) == -4
    assert lib.splat_feature_norm_backward(0, 1, 4, 8, 2, P, None, None, P, P, 0, None, P, P, P,
                                           P, 1 << 20, None) == -1
    assert lib.splat_launch_count() == before
