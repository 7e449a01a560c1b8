"""AdamW over many tensors at once, such as a scene's Gaussians and a feature
decoder's layers.

    m' = b1 m + (1 - b1) g,  v' = b2 v + (1 - b2) g^2
    p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v' / (1 - b2^t)) + eps)

* `adamw`: one step in place, one launch for all tensors of a device and dtype;
* `AdamW`: the torch.optim.Optimizer that calls it;
* `Moment8`: a moment held in 8 bits.

Parameters are contiguous CUDA float32, bfloat16 or float16 tensors, their gradients of
the same type.  Both moments are float32, or 8-bit codes with an exponent for each 256
values of the flattened tensor: m as a sign, 4 bits of exponent and 3 of mantissa, v as
its root with 4 and 4, both relative to the run's exponent.  Each step rounds them
down after a dither that is a hash of the value's place and the step: off by less than
a step of the code and right on average, so that averages which move by less than that
are followed; the update itself takes the values before their rounding.  A run that
holds an infinity or a NaN reads as NaN, and makes its parameters NaN in the next step:
gradients that may not be finite are looked at before the step, as torch.amp.GradScaler
does.

The reference has no counterpart; its users bring their own optimizer.
"""

from __future__ import annotations

import struct
from numbers import Integral, Real
from typing import Any, Callable, Iterable, Sequence

import torch
from torch import Tensor

from . import stages

RUN = 256  # values that share an exponent
_RECORD = struct.Struct("=10q5d")  # a SplatAdamwTensor of include/splat200.h


class Moment8:
    """A moment held in 8 bits: codes of the parameter's shape and exponents, one for each
    256 values.  squared: of the second moment, whose root the codes hold."""

    __slots__ = ("codes", "exponents", "squared")

    def __init__(self, codes: Tensor, exponents: Tensor, squared: bool = False):
        if codes.dtype is not torch.uint8 or exponents.dtype is not torch.int8:
            raise ValueError("codes must be uint8 and exponents int8")
        if not codes.is_contiguous() or not exponents.is_contiguous():
            raise ValueError("codes and exponents must be contiguous")
        if exponents.shape != (-(-codes.numel() // RUN),) or exponents.device != codes.device:
            raise ValueError("exponents must have one value for each 256 codes, on their device")
        self.codes, self.exponents, self.squared = codes, exponents, squared

    @classmethod
    def of(cls, values: Tensor, squared: bool = False) -> Moment8:
        """The nearest codes of float32 moments."""
        if not values.is_cuda or values.dtype is not torch.float32:
            raise ValueError("values must be a CUDA float32 tensor")
        return cls(*stages.adamw_encode(values, squared), squared)

    @classmethod
    def zeros_like(cls, parameter: Tensor, squared: bool = False) -> Moment8:
        codes = torch.zeros(parameter.shape, dtype=torch.uint8, device=parameter.device)
        exponents = torch.full((-(-codes.numel() // RUN),), -126, dtype=torch.int8,
                               device=parameter.device)
        return cls(codes, exponents, squared)

    def values(self) -> Tensor:
        """The float32 moments that the codes stand for."""
        if not self.codes.is_cuda:
            raise ValueError("codes must be a CUDA tensor")
        return stages.adamw_decode(self.codes, self.exponents, self.squared)


# The kernel takes these in fp32.
_LARGEST = 2.0 ** 128
_BELOW_ONE = 1.0 - 2.0 ** -24


def _check_settings(betas: tuple[float, float], eps: float, weight_decay: float) -> None:
    if len(betas) != 2 or not all(0.0 <= b <= _BELOW_ONE for b in betas):
        raise ValueError("betas must be two numbers of at least 0 and below 1 in float32")
    if not (eps == 0.0 or 2.0 ** -126 <= eps < _LARGEST):
        raise ValueError("eps must be 0, or finite and positive in float32's normal range")
    if not 0.0 <= weight_decay < _LARGEST:
        raise ValueError("weight_decay must be finite in float32 and not negative")


def _check_lr(lr: Any) -> None:
    if type(lr) is float and 0.0 <= lr < _LARGEST:
        return
    if isinstance(lr, Tensor):
        if lr.numel() != 1 or not lr.is_cuda or lr.dtype is not torch.float32:
            raise ValueError("lr must be a number or a CUDA float32 tensor of one value")
    elif not isinstance(lr, Real) or not 0.0 <= lr < _LARGEST:
        raise ValueError("lr must be finite in float32 and not negative")


def _check_step(step: Any) -> None:
    if type(step) is int and step >= 1:
        return
    if isinstance(step, Tensor):
        if step.numel() != 1 or not step.is_cuda or step.dtype is not torch.int64:
            raise ValueError("step must be an integer or a CUDA int64 tensor of one value")
    elif isinstance(step, bool) or not isinstance(step, Integral) or step < 1:
        raise ValueError("step must be an integer of at least one")


def _check_parameter(p: Tensor) -> None:
    if not isinstance(p, Tensor) or not p.is_cuda or p.dtype not in stages.FEATURE_DTYPES:
        raise ValueError("parameters must be CUDA float32, bfloat16 or float16 tensors")
    if not p.is_contiguous():
        raise ValueError("parameters must be contiguous")


def _check_moment(m: Any, p: Tensor, squared: bool) -> int:
    if isinstance(m, Moment8):
        if (m.codes.shape != p.shape or m.codes.get_device() != p.get_device()
                or m.squared != squared):
            raise ValueError("8-bit moments must have their parameter's shape and device, and "
                             "the second ones be squared")
        return 8
    if (not isinstance(m, Tensor) or m.dtype is not torch.float32 or m.shape != p.shape
            or m.get_device() != p.get_device() or not m.is_contiguous()):
        raise ValueError("moments must be contiguous float32 tensors, or Moment8, of their "
                         "parameter's shape and device")
    return 32


def _each(value: Any, count: int, name: str) -> Sequence:
    if isinstance(value, (list, tuple)):
        if len(value) != count:
            raise ValueError(f"{name} must be one value, or one for each parameter")
        return value
    return (value,) * count


class _Launches:
    """The launches of a step, made after all of its arguments have been checked."""

    def __init__(self) -> None:
        self.records: dict[tuple, list] = {}
        self.written: list[Tensor] = []
        self.held: list[Tensor] = []  # until the launches
        self.places: set[int] = set()
        self.read: set[int] = set()

    def add(self, p: Tensor, g: Tensor, m: Tensor | Moment8, v: Tensor | Moment8,
            step: int | Tensor, lr: float | Tensor, decay: float, betas: tuple[float, float],
            eps: float, maximize: bool) -> None:
        """A parameter, whose numbers have been checked."""
        _check_parameter(p)
        if not isinstance(g, Tensor) or g.layout is not torch.strided:
            raise ValueError("gradients must be dense tensors")
        index = p.get_device()
        if g.dtype is not p.dtype or g.get_device() != index or g.shape != p.shape:
            raise ValueError("gradients must have their parameter's dtype, device and shape")
        bits = _check_moment(m, p, False)
        if _check_moment(v, p, True) != bits:
            raise ValueError("both moments must be held in the same number of bits")
        device_step = device_lr = 0
        if isinstance(step, Tensor):
            if step.get_device() != index:
                raise ValueError("step and lr tensors must be on their parameter's device")
            device_step, step = step.data_ptr(), 0
        if isinstance(lr, Tensor):
            if lr.get_device() != index:
                raise ValueError("step and lr tensors must be on their parameter's device")
            device_lr, lr = lr.data_ptr(), 0.0
        n = p.numel()
        if not n:
            return
        if not g.is_contiguous():
            g = g.contiguous()
            self.held.append(g)
        address, gradient = p.data_ptr(), g.data_ptr()
        if bits == 8:
            record = (address, gradient, m.codes.data_ptr(), v.codes.data_ptr(),
                      m.exponents.data_ptr(), v.exponents.data_ptr())
            self.written += (p, m.codes, v.codes, m.exponents, v.exponents)
        else:
            record = (address, gradient, m.data_ptr(), v.data_ptr())
            self.written += (p, m, v)
        written = {address, *record[2:]}
        if len(written) < len(record) - 1 or not written.isdisjoint(self.places):
            raise ValueError("a parameter or a moment is listed twice")
        self.places |= written
        self.read.add(gradient)
        record = _RECORD.pack(*record, *(0,) * (6 - len(record)), device_step, device_lr, n, step,
                              lr, decay, betas[0], betas[1], eps)
        self.records.setdefault((index, p.dtype, bits, maximize), []).append(record)

    def run(self, counters: Sequence[Tensor] = ()) -> None:
        """counters: device steps, which the launches read one on."""
        if not self.read.isdisjoint(self.places):
            raise ValueError("a gradient is a parameter or a moment of the same step")
        if counters:
            torch._foreach_add_(counters, 1)
        for (index, dtype, bits, maximize), records in self.records.items():
            stages.adamw(index, dtype, bits, records, maximize)
        if self.written:
            torch.autograd.graph.increment_version(self.written)


@torch.no_grad()
def adamw(params: Sequence[Tensor], grads: Sequence[Tensor],
          exp_avgs: Sequence[Tensor | Moment8], exp_avg_sqs: Sequence[Tensor | Moment8], *,
          step: int | Tensor | Sequence, lr: float | Tensor | Sequence,
          betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
          weight_decay: float | Sequence[float] = 1e-2, maximize: bool = False) -> None:
    """One AdamW step of all params in place, their moments with them.

    step counts from 1 and is the number of this step.  step, lr and weight_decay are
    one value or a list with one for each parameter; step may be a CUDA int64 and lr a CUDA
    float32 tensor of one value, which the kernel reads (a captured step then follows
    them).  No parameter or moment may be listed twice or share memory with another or with
    a gradient."""
    count = len(params)
    if not len(grads) == len(exp_avgs) == len(exp_avg_sqs) == count:
        raise ValueError("params, grads, exp_avgs and exp_avg_sqs must have the same length")
    steps, lrs = _each(step, count, "step"), _each(lr, count, "lr")
    decays = _each(weight_decay, count, "weight_decay")
    for s in steps if isinstance(step, (list, tuple)) else (step,):
        _check_step(s)
    for v in lrs if isinstance(lr, (list, tuple)) else (lr,):
        _check_lr(v)
    for w in decays if isinstance(weight_decay, (list, tuple)) else (weight_decay,):
        _check_settings(betas, eps, w)
    launches = _Launches()
    for p, g, m, v, s, r, w in zip(params, grads, exp_avgs, exp_avg_sqs, steps, lrs, decays):
        launches.add(p, g, m, v, s, r, w, betas, eps, maximize)
    launches.run()


def _check_loaded_group(group: dict, own: dict) -> None:
    """Refuses a saved group that this optimizer would not follow; own: the group that
    takes it over."""
    for name in ("amsgrad", "differentiable"):
        if group.get(name):
            raise ValueError(f"a state of {name}=True has no counterpart here")
    # L2 decay, which goes through the moments
    if not group.get("decoupled_weight_decay", True) and group["weight_decay"]:
        raise ValueError("a state whose weight decay is not decoupled has no counterpart here")
    _check_settings(group["betas"], group["eps"], group["weight_decay"])
    if group.get("state_bits", own["state_bits"]) not in (8, 32):
        raise ValueError("state_bits must be 8 or 32")


def _counted(step: Any) -> int:
    """The steps of a state: an integer, or a tensor of one, which torch.optim holds in
    float32."""
    if isinstance(step, Tensor):
        if step.numel() != 1:
            raise ValueError("a state's step must be one number")
        step = step.item()
    if isinstance(step, bool) or not isinstance(step, Real) or not 0 <= step < 1 << 63 \
            or step != int(step):
        raise ValueError("a state's step must be a number of steps")
    return int(step)


def _loaded_state(saved: dict, p: Tensor, bits: int, capturable: bool) -> dict:
    """A parameter's saved state as `AdamW` holds it: of its own or of torch.optim.AdamW."""
    if "max_exp_avg_sq" in saved:
        raise ValueError("a state of amsgrad=True has no counterpart here")
    state = {name: v.to(p.device, copy=True).contiguous() if isinstance(v, Tensor) else v
             for name, v in saved.items() if name != "step"}
    if "step" in saved:
        step = _counted(saved["step"])
        state["step"] = (torch.full((), step, dtype=torch.int64, device=p.device) if capturable
                         else step)
    for name, squared in (("exp_avg", False), ("exp_avg_sq", True)):
        if name not in saved:
            continue
        if not isinstance(state[name], Tensor) or state[name].shape != p.shape:
            raise ValueError(f"a state's {name} must have its parameter's shape")
        if name + "_exponents" in saved:
            moment = Moment8(state[name], state[name + "_exponents"], squared)
            if bits == 32:
                state[name] = moment.values()
                del state[name + "_exponents"]
        elif not state[name].is_floating_point():
            raise ValueError(f"a state's {name} must hold floating-point values")
        else:
            state[name] = state[name].float()
            if bits == 8:
                moment = Moment8.of(state[name], squared)
                state[name], state[name + "_exponents"] = moment.codes, moment.exponents
    return state


class AdamW(torch.optim.Optimizer):
    """AdamW with one launch for all parameters of a device and dtype.

    state_bits: 32 or 8.  The state of a parameter holds "step", "exp_avg" and "exp_avg_sq"
    (with 8 bits the codes, and their "exp_avg_exponents" and "exp_avg_sq_exponents");
    `moments` and `set_moments` take the values they stand for, whatever the bits,
    which is what code that adds or removes Gaussians has to carry over.
    capturable: steps are counted on the device, so that a captured step() can be
    replayed (lr may then be a CUDA float32 tensor).

    load_state_dict takes torch.optim.AdamW's state too, but for amsgrad: its steps are
    converted and its moments held in float32, or in 8 bits where the group has them.  What
    it loads are new tensors, which a step captured before does not follow; moments that
    set_moments takes are written into those that it does."""

    def __init__(self, params: Iterable, lr: float | Tensor = 1e-3,
                 betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, maximize: bool = False,
                 capturable: bool = False):
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      state_bits=state_bits, maximize=maximize,
                                      capturable=capturable))

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            _check_lr(group["lr"])
            _check_settings(group["betas"], group["eps"], group["weight_decay"])
            if group["state_bits"] not in (8, 32):
                raise ValueError("state_bits must be 8 or 32")
            for p in group["params"]:
                _check_parameter(p)
        except ValueError:
            self.param_groups.pop()
            raise

    def _state(self, p: Tensor, group: dict) -> dict:
        state = self.state[p]
        if not state:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW makes a parameter's state in its first step, which "
                                   "must run before a step is captured")
            state["step"] = (torch.zeros((), dtype=torch.int64, device=p.device)
                             if group["capturable"] else 0)
            if group["state_bits"] == 8:
                self._put(state, Moment8.zeros_like(p), Moment8.zeros_like(p, squared=True))
            else:
                self._put(state, torch.zeros_like(p, dtype=torch.float32),
                          torch.zeros_like(p, dtype=torch.float32))
        elif group["capturable"] and not isinstance(state["step"], Tensor):
            # a captured step would hold the number that it has now
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW moves a parameter's step to the device in its first "
                                   "capturable step, which must run before a step is captured")
            state["step"] = torch.full((), _counted(state["step"]), dtype=torch.int64,
                                       device=p.device)
        return state

    @staticmethod
    def _put(state: dict, m: Tensor | Moment8, v: Tensor | Moment8) -> None:
        """Into the state's own tensors where they fit, which a captured step may hold."""
        for name, moment in (("exp_avg", m), ("exp_avg_sq", v)):
            if isinstance(moment, Moment8):
                parts = {name: moment.codes, name + "_exponents": moment.exponents}
            else:
                parts = {name: moment}
                state.pop(name + "_exponents", None)
            for key, value in parts.items():
                held = state.get(key)
                if isinstance(held, Tensor) and held.shape == value.shape \
                        and held.dtype is value.dtype and held.device == value.device:
                    held.copy_(value)
                else:
                    state[key] = value

    @staticmethod
    def _get(state: dict) -> tuple:
        if "exp_avg_exponents" not in state:
            return state["exp_avg"], state["exp_avg_sq"]
        return (Moment8(state["exp_avg"], state["exp_avg_exponents"]),
                Moment8(state["exp_avg_sq"], state["exp_avg_sq_exponents"], True))

    @torch.no_grad()
    def step(self, closure: Callable | None = None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        capturing = torch.cuda.is_current_stream_capturing()
        launches = _Launches()
        counters, counted = [], []
        for group in self.param_groups:
            if capturing and not group["capturable"]:
                raise RuntimeError("a step is captured only of an AdamW with capturable=True")
            _check_lr(group["lr"])
            settings = (group["lr"], group["weight_decay"], group["betas"], group["eps"],
                        group["maximize"])
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self._state(p, group)
                step = state["step"]
                if isinstance(step, Tensor):
                    _check_step(step)  # the kernel reads it as it lies
                    counters.append(step)
                else:
                    counted.append(state)
                    step += 1
                launches.add(p, p.grad, *self._get(state), step, *settings)
        launches.run(counters)
        for state in counted:
            state["step"] += 1
        return loss

    def moments(self, p: Tensor) -> tuple[Tensor, Tensor]:
        """A parameter's moments as float32 (of 32 bits the state's own tensors)."""
        if not self.state.get(p):
            raise KeyError("the parameter has no state yet")
        m, v = self._get(self.state[p])
        return (m.values(), v.values()) if isinstance(m, Moment8) else (m, v)

    @torch.no_grad()
    def set_moments(self, p: Tensor, m: Tensor, v: Tensor) -> None:
        """Replaces the values of a parameter's moments by float32 ones of its shape; its step
        stays."""
        group = next((g for g in self.param_groups if any(q is p for q in g["params"])), None)
        if group is None:
            raise KeyError("not a parameter of this optimizer")
        for t in (m, v):
            if _check_moment(t, p, False) != 32:
                raise ValueError("moments are set from float32 tensors")
        state = self._state(p, group)
        if group["state_bits"] == 8:
            self._put(state, Moment8.of(m), Moment8.of(v, squared=True))
        else:
            self._put(state, m.clone(), v.clone())

    @torch.no_grad()
    def load_state_dict(self, state_dict: dict) -> None:
        states: list[tuple[Tensor, dict]] = []
        # a saved group of torch.optim.AdamW lacks some of the settings
        settings = [{name: group[name] for name in self.defaults} for group in self.param_groups]

        def read(_, saved: dict) -> None:
            """The whole state, before anything of this optimizer changes."""
            for group, own in zip(saved["param_groups"], self.param_groups):
                _check_loaded_group(group, own)
                bits = group.get("state_bits", own["state_bits"])
                capturable = group.get("capturable", own["capturable"])
                for i, p in zip(group["params"], own["params"]):
                    if i in saved["state"]:
                        states.append((p, _loaded_state(saved["state"][i], p, bits, capturable)))

        def take(_) -> None:
            for group, own in zip(self.param_groups, settings):
                for name, value in own.items():
                    group.setdefault(name, value)
                if isinstance(group["lr"], Tensor) and group["params"]:  # read on the host
                    group["lr"] = group["lr"].to(group["params"][0].device, torch.float32)
            # torch casts a state to its parameter's dtype; moments keep theirs
            for p, state in states:
                self.state[p] = state

        # behind the hooks that change what is loaded, before those that look at the result
        hooks = (self.register_load_state_dict_pre_hook(read),
                 self.register_load_state_dict_post_hook(take, prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()
