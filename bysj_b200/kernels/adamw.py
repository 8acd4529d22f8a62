"""AdamW over many tensors in one launch, states in 32 or 8 bits, on B200.

:class:`AdamW` holds the states of all parameters in one buffer each, every
tensor's share padded to a multiple of 256 elements, and steps all of them
with one kernel launch per parameter dtype.  With ``state_bits=8`` an element
keeps one byte for each moment and every 256 elements a float32 scale; with
``master_weights`` bfloat16 parameters are rounded copies of float32 weights.
No reference counterpart (the reference serves inference).
"""
from __future__ import annotations

import math
from typing import Any, Iterable, Sequence

import torch

from .native import _entry, _extension, require_dcu

BLOCK = 256


def _unit_interval(name: str, value: Any) -> float:
    value = float(value)
    if not 0.0 <= value < 1.0:
        raise ValueError(f"AdamW {name} must be in [0, 1)")
    return value


class AdamW:
    """Decoupled-weight-decay Adam over a fixed list of parameters.

    ``params``: contiguous float32 or bfloat16 CUDA tensors on one device
    that share no memory (mixed dtypes are stepped in two launches).  ``lr``,
    ``betas``, ``eps`` and ``weight_decay`` are plain attributes, so a schedule
    may assign them between steps; weights with another decay need an optimizer
    of their own.  ``state_bits``: 32, or 8 for one byte per element and
    moment: the first as sign and 7-bit magnitude, the root of the second in 8
    bits, both relative to the largest of 256 elements.  A step rounds them to
    the nearest code (errors of at most 1/16 and 1/32 of a value).  A moment
    that a step moves by less than half a code (``beta1 > 15/16``, ``beta2 >
    63/64``, as the default) is rounded at random without bias instead, so
    that it keeps following its gradients; the root of the second moment then
    differs from that of 32-bit states by about 11 % root mean square.  The
    random numbers come from the step and the element: equal runs give equal
    bits.  A non-finite gradient leaves no finite moment in its whole block
    there, in its element alone with 32 bits.
    ``master_weights`` keeps float32 weights beside the parameters;
    call :meth:`sync_master` after assigning parameters by hand.

    The states are ``exp_avg`` and ``exp_avg_sq`` (float32 or uint8 codes),
    ``exp_avg_scale`` / ``exp_avg_sq_scale`` and ``master`` (or ``None``): one
    flat buffer each, tensor ``i`` at ``begins[i]``.
    """

    def __init__(self, params: Iterable[torch.Tensor], lr: float = 1.0e-3,
                 betas: Sequence[float] = (0.9, 0.999), eps: float = 1.0e-8,
                 weight_decay: float = 1.0e-2, *, state_bits: int = 32,
                 master_weights: bool = False) -> None:
        self._params = tuple(params)
        if not self.params:
            raise ValueError("AdamW needs at least one parameter")
        for p in self.params:
            if not isinstance(p, torch.Tensor):
                raise TypeError("AdamW parameters must be tensors")
            if p.dtype not in (torch.float32, torch.bfloat16):
                raise TypeError("AdamW parameters must be float32 or bfloat16")
            if not p.is_contiguous():
                raise ValueError("AdamW parameters must be contiguous")
        if len({p.device for p in self.params}) != 1:
            raise ValueError("all AdamW parameters must share a device")
        if len({id(p) for p in self.params}) != len(self.params):
            raise ValueError("AdamW parameters must be different tensors")
        ranges = sorted((p.data_ptr(), p.numel() * p.element_size()) for p in self.params
                        if p.numel())
        if any(at + size > after for (at, size), (after, _) in zip(ranges, ranges[1:])):
            raise ValueError("AdamW parameters must not share memory")
        if state_bits not in (8, 32):
            raise ValueError("AdamW state_bits must be 8 or 32")
        self.lr, self.eps, self.weight_decay = float(lr), float(eps), float(weight_decay)
        if len(betas) != 2:
            raise ValueError("AdamW betas must be two numbers")
        self.betas = (_unit_interval("beta1", betas[0]), _unit_interval("beta2", betas[1]))
        if not (math.isfinite(self.lr) and self.lr >= 0.0):
            raise ValueError("AdamW lr must be finite and non-negative")
        if not (math.isfinite(self.eps) and self.eps > 0.0):
            raise ValueError("AdamW eps must be finite and positive")
        if not (math.isfinite(self.weight_decay) and self.weight_decay >= 0.0):
            raise ValueError("AdamW weight_decay must be finite and non-negative")
        require_dcu(*self.params)
        self.state_bits = state_bits
        self.step_count = 0
        self.begins, length = [], 0
        for p in self.params:
            self.begins.append(length)
            length += -(-p.numel() // BLOCK) * BLOCK
        device = self.params[0].device
        dtype = torch.float32 if state_bits == 32 else torch.uint8
        self.exp_avg = torch.zeros(length, dtype=dtype, device=device)
        self.exp_avg_sq = torch.zeros(length, dtype=dtype, device=device)
        self.exp_avg_scale = self.exp_avg_sq_scale = self.master = None
        self._tensors = _extension("AdamWParams").AdamWParams(self.params, self.begins)
        if state_bits == 8:
            self.exp_avg_scale = torch.zeros(length // BLOCK, device=device)
            self.exp_avg_sq_scale = torch.zeros(length // BLOCK, device=device)
        if master_weights:
            self.master = torch.zeros(length, device=device)
            self.sync_master()

    @property
    def params(self) -> tuple[torch.Tensor, ...]:
        """The parameters, fixed when the optimizer is made."""
        return self._params

    @torch.no_grad()
    def sync_master(self) -> None:
        """Copy the parameters into the float32 master weights."""
        if self.master is not None:
            for p, begin in zip(self.params, self.begins):
                self.master[begin:begin + p.numel()] = p.reshape(-1)

    def step(self, grads: Sequence[torch.Tensor | None] | None = None, *,
             grad_scale: torch.Tensor | None = None) -> None:
        """Step every parameter that has a gradient, in place.

        ``grads``: one tensor (or ``None``: skip) per parameter, of its dtype and shape;
        default the parameters' ``.grad``.  ``grad_scale``: a float32 CUDA
        tensor of one element that multiplies every gradient (a clip factor or
        the inverse of a loss scale), read on the device.  A step is refused while
        the stream is captured: its bias corrections are values of this call.
        """
        if grads is None:
            grads = [p.grad for p in self._params]
        elif not isinstance(grads, list):
            grads = list(grads)
        if len(grads) != len(self._params):
            raise ValueError("AdamW needs one gradient (or None) for each parameter")
        if grad_scale is not None:
            if not isinstance(grad_scale, torch.Tensor) or grad_scale.dtype != torch.float32:
                raise TypeError("AdamW grad_scale must be a float32 tensor")
            if grad_scale.numel() != 1:
                raise ValueError("AdamW grad_scale must have one element")
        step, (beta1, beta2) = self.step_count + 1, self.betas
        _entry("adamw_step")(
            self._tensors, grads, self.exp_avg, self.exp_avg_sq, self.exp_avg_scale,
            self.exp_avg_sq_scale, self.master, grad_scale, beta1, beta2,
            1.0 - self.lr * self.weight_decay, self.lr / (1.0 - beta1 ** step),
            1.0 / math.sqrt(1.0 - beta2 ** step), self.eps, step)
        self.step_count = step

    def zero_grad(self) -> None:
        """Drop the parameters' gradients."""
        for p in self.params:
            p.grad = None

    def state_values(self) -> tuple[torch.Tensor, torch.Tensor]:
        """The moments as float32 buffers: the states themselves with 32 bits."""
        if self.state_bits == 32:
            return self.exp_avg, self.exp_avg_sq
        return _entry("adamw_state_values")(
            self.exp_avg, self.exp_avg_sq, self.exp_avg_scale, self.exp_avg_sq_scale)

    _BUFFERS = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "master")

    def state_dict(self) -> dict[str, Any]:
        """Step count and copies of the state buffers."""
        state: dict[str, Any] = {"step": self.step_count}
        for name in self._BUFFERS:
            value = getattr(self, name)
            state[name] = None if value is None else value.clone()
        return state

    @torch.no_grad()
    def load_state_dict(self, state: dict[str, Any]) -> None:
        """Copy the buffers of a :meth:`state_dict` of the same layout into this one."""
        step = int(state["step"])
        for name in self._BUFFERS:
            own, given = getattr(self, name), state[name]
            if (own is None) != (given is None):
                raise ValueError(f"AdamW state {name} is present on one side only")
            if own is not None and (not isinstance(given, torch.Tensor) or
                                    given.dtype != own.dtype or given.shape != own.shape):
                raise ValueError(f"AdamW state {name} must be {own.dtype} of shape "
                                 f"{tuple(own.shape)}")
        for name in self._BUFFERS:
            if state[name] is not None:
                getattr(self, name).copy_(state[name])
        self.step_count = step


__all__ = ["AdamW", "BLOCK"]
