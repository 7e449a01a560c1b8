"""Operators over learned features: what decodes the channel-last feature
images that the rasterisers blend (`extra_features`, arbitrary channels) and
the per-Gaussian features that they blend from.

* `linear`: act(x W^T + b) + residual over the last dimension;
* `group_norm`: group norm with an activation over channel-last images;
* `FeatureDecoder`: a run of them, called on an image, or passed to
  gs3d.rasterize / rade.rasterize / aaa.rasterize as `feature_decoder`.

Tensors are CUDA float32, bfloat16 or float16, all of one type per call (no
autocast).  Sums are held in fp32 or more and rounded once to that type, and
no result depends on the order in which blocks run.  The backward of a 16-bit
`linear` keeps dy act'(z) as two values of that type (2^-16 relative for
bfloat16, 2^-22 for float16, whose smallest value is 2^-24: float16 losses want
their usual scale).  Any strides are taken; what is not contiguous is copied
first.  First-order reverse-mode gradients only; forward-mode ones and
torch.func's transforms are refused.  float32 operands are split into three parts
of 8 digits, of which those below 2^-133 are lost (values below 2^-110 keep
fewer than 24).

A device-side wait that gives up (a defect, not a user's error) sets the
library's error word, which the next binning, or _native.device_error, reads.

Calls can be captured into CUDA graphs.  As with any torch operator, a
backward is captured only while no eager graph of the same leaves is alive
(drop or detach earlier results first): torch ties a leaf's gradient node to
the stream of its first use.

The reference has no counterpart; its users decode features in their own
training code.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from numbers import Integral
from typing import Any, Iterator

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import stages

ACTIVATIONS = stages.ACTIVATIONS


def _once(backward):
    """once_differentiable, whose cost only a backward that is recorded pays."""
    recorded = once_differentiable(backward)

    def run(ctx, *upstream):
        return (recorded if torch.is_grad_enabled() else backward)(ctx, *upstream)

    return run


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x: Tensor, weight: Tensor, bias: Tensor | None,
                residual: Tensor | None, activation: str) -> Tensor:
        ctx.save_for_backward(x, weight, bias)
        ctx.activation = activation
        ctx.set_materialize_grads(False)
        return stages.feature_linear(x, weight, bias, residual, activation)

    @staticmethod
    @_once
    def backward(ctx: Any, upstream: Tensor | None):
        if upstream is None:
            return (None,) * 5
        x, weight, bias = ctx.saved_tensors
        needs = ctx.needs_input_grad
        dx, dweight, dbias = stages.feature_linear_backward(
            x, weight, bias, ctx.activation, upstream, needs[:3])
        return dx, dweight, dbias, upstream if needs[3] else None, None


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x: Tensor, weight: Tensor | None, bias: Tensor | None, samples: int,
                groups: int, eps: float, activation: str) -> Tensor:
        y, moments = stages.feature_norm(x, samples, groups, weight, bias, eps, activation)
        ctx.save_for_backward(x, weight, bias, moments)
        ctx.settings = samples, groups, activation
        ctx.set_materialize_grads(False)
        return y

    @staticmethod
    @_once
    def backward(ctx: Any, upstream: Tensor | None):
        if upstream is None:
            return (None,) * 7
        x, weight, bias, moments = ctx.saved_tensors
        samples, groups, activation = ctx.settings
        dx, dweight, dbias = stages.feature_norm_backward(
            x, samples, groups, weight, bias, moments, activation, upstream,
            ctx.needs_input_grad[:3])
        return dx, dweight, dbias, None, None, None, None


def _check_activation(activation: str) -> None:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {ACTIVATIONS}")


def _check_input(x: Tensor) -> None:
    if not isinstance(x, Tensor) or not x.is_cuda or x.dtype not in stages.FEATURE_DTYPES:
        raise ValueError("x must be a CUDA float32, bfloat16 or float16 tensor")


def _check_like(t: Tensor | None, x: Tensor, shape: tuple, name: str) -> None:
    if t is None:
        return
    if not isinstance(t, Tensor) or t.dtype is not x.dtype or t.device != x.device:
        raise ValueError(f"{name} must have x's dtype and device")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _check_forward_mode(*tensors: Tensor | None) -> None:
    """Refuses dual tensors: a result without a tangent would pass for a
    derivative of zero."""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("forward-mode derivatives of the feature operators")


def _traced() -> bool:
    """Whether a program is being recorded: then the calls go through
    torch.ops.splat200, which it can hold (a launch through the C ABI leaves
    only the allocation of its result in it)."""
    return (torch.compiler.is_compiling() or torch._C._len_torch_dispatch_stack() > 0
            or torch._C._is_tracing())


def _recorded(*tensors: Tensor | None) -> bool:
    """Whether autograd has to know of a call."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def check_linear(x: Tensor, weight: Tensor, bias: Tensor | None, activation: str,
                 output: Tensor | None, name: str) -> None:
    """Refuses what `linear` does not take; output: of the result's shape."""
    _check_activation(activation)
    _check_input(x)
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError("x must have a last dimension of at least one feature")
    k = x.shape[-1]
    if not isinstance(weight, Tensor) or weight.ndim != 2 or weight.shape[0] < 1:
        raise ValueError("weight must be (N,K) with N of at least one")
    n = weight.shape[0]
    _check_like(weight, x, (n, k), "weight")
    _check_like(bias, x, (n,), "bias")
    if output is not None:
        _check_like(output, x, x.shape[:-1] + (n,), name)
    if k > 65535 or n > 65535:
        raise ValueError("at most 65535 input and output features")


def linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, *,
           residual: Tensor | None = None, activation: str = "none") -> Tensor:
    """act(x weight^T + bias) + residual over the last dimension of x.

    x: (...,K), weight: (N,K), bias: (N,), residual and the result: (...,N).
    activation: "none", "relu", "silu", "gelu" (the erf form) or "sigmoid".
    """
    check_linear(x, weight, bias, activation, residual, "residual")
    if forward_ad._current_level >= 0:
        _check_forward_mode(x, weight, bias, residual)
    if _traced():
        return torch.ops.splat200.feature_linear(x, weight, bias, residual, activation)
    if _recorded(x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, residual, activation)
    return stages.feature_linear(x, weight, bias, residual, activation)


def check_group_norm(x: Tensor, groups: int, weight: Tensor | None, bias: Tensor | None,
                     eps: float, activation: str, samples: int, positions: int) -> None:
    """Refuses what `group_norm` does not take, for an x of at least a dimension
    whose leading ones hold so many samples and positions."""
    _check_activation(activation)
    channels = x.shape[-1]
    if isinstance(groups, bool) or not isinstance(groups, Integral) or groups < 1:
        raise ValueError("groups must be a positive integer")
    if channels % groups:
        raise ValueError(f"groups must divide the channels: {channels} channels, {groups} groups")
    _check_like(weight, x, (channels,), "weight")
    _check_like(bias, x, (channels,), "bias")
    if not 2.0 ** -126 <= eps < 2.0 ** 128:  # the kernels take it in fp32
        raise ValueError("eps must be finite and positive in float32's normal range")
    if positions > (1 << 31) - 1 or positions * channels > 1 << 40 or samples * channels > 1 << 30:
        raise ValueError("too many positions or samples")


def group_norm(x: Tensor, groups: int, weight: Tensor | None = None, bias: Tensor | None = None,
               *, eps: float = 1e-5, activation: str = "none", spatial_dims: int = 2) -> Tensor:
    """act((x - mean) / sqrt(var + eps) * weight + bias), channels last.

    The last dimension holds the channels, the `spatial_dims` before it the
    positions of a sample (2: images (...,H,W,C); 1: sets (...,N,C), such as a
    scene's Gaussians).  Mean and biased variance run over a sample's
    positions and the channels of each of `groups` equal groups.  weight and
    bias: (C,).  activation as in `linear`.
    """
    _check_activation(activation)
    _check_input(x)
    if isinstance(spatial_dims, bool) or not isinstance(spatial_dims, Integral) or spatial_dims < 1:
        raise ValueError("spatial_dims must be an integer of at least one")
    if x.ndim < spatial_dims + 1 or x.shape[-1] < 1:
        raise ValueError("x must have spatial_dims dimensions and at least one channel last")
    samples = math.prod(x.shape[:-1 - spatial_dims])
    positions = math.prod(x.shape[-1 - spatial_dims:-1])
    check_group_norm(x, groups, weight, bias, eps, activation, samples, positions)
    if forward_ad._current_level >= 0:
        _check_forward_mode(x, weight, bias)
    groups, eps = int(groups), float(eps)
    if _traced():
        shape = (samples, positions, x.shape[-1])
        return torch.ops.splat200.feature_norm(x.reshape(shape), groups, weight, bias, eps,
                                               activation)[0].reshape(x.shape)
    if _recorded(x, weight, bias):
        return _GroupNorm.apply(x, weight, bias, samples, groups, eps, activation)
    return stages.feature_norm(x, samples, groups, weight, bias, eps, activation, False)[0]


@dataclass(slots=True)
class Linear:
    """One `linear` of a FeatureDecoder; residual=True adds the layer's own input."""

    weight: Tensor
    bias: Tensor | None = None
    activation: str = "none"
    residual: bool = False

    def __call__(self, x: Tensor) -> Tensor:
        return linear(x, self.weight, self.bias, residual=x if self.residual else None,
                      activation=self.activation)


@dataclass(slots=True)
class GroupNorm:
    """One `group_norm` of a FeatureDecoder."""

    groups: int
    weight: Tensor | None = None
    bias: Tensor | None = None
    eps: float = 1e-5
    activation: str = "none"

    def __call__(self, x: Tensor) -> Tensor:
        return group_norm(x, self.groups, self.weight, self.bias, eps=self.eps,
                          activation=self.activation)


class FeatureDecoder:
    """Layers called one after another on a channel-last image (...,H,W,C).

    The layers' dtype is that of the computation: a rendered float32 image is
    converted to it once, at the start.
    """

    def __init__(self, *layers: Linear | GroupNorm):
        if not layers or not all(isinstance(v, (Linear, GroupNorm)) for v in layers):
            raise ValueError("FeatureDecoder takes Linear and GroupNorm layers")
        self.layers = layers

    def parameters(self) -> Iterator[Tensor]:
        for layer in self.layers:
            for t in (layer.weight, layer.bias):
                if t is not None:
                    yield t

    def __call__(self, image: Tensor) -> Tensor:
        first = next(self.parameters(), None)
        if first is not None:
            image = image.to(first.dtype)
        for layer in self.layers:
            image = layer(image)
        return image
