"""Group norm over frames with an activation, channels last, on B200.

``group_norm(x, groups, ...)`` normalises each frame over its rows and the
channels of a group, and applies an affine map and an activation in the same
pass, forward and backward.  A frame is an entry of the leading dimension,
or, with ``offsets``, a range of it: packed frames of any lengths, as the
segmented operators take them.  No reference counterpart.
"""
from __future__ import annotations

import math

import torch

from . import segment as _segment
from .native import _entry, require_dcu

MAX_CHANNELS = 8192
_ACTIVATIONS = {None: 0, "none": 0, "silu": 1, "sigmoid": 2}


def _validate(x, groups, weight, bias, eps, activation, offsets):
    if not isinstance(x, torch.Tensor):
        raise TypeError("group norm input must be a tensor")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("group norm input must be float32 or bfloat16")
    if x.ndim < 2:
        raise ValueError("group norm input must have at least two dimensions")
    channels = int(x.shape[-1])
    if isinstance(groups, bool) or not isinstance(groups, int):
        raise TypeError("group norm groups must be an int")
    if channels <= 0 or groups <= 0 or channels % groups:
        raise ValueError("group norm groups must divide the (positive) channel count")
    if channels > MAX_CHANNELS:
        raise ValueError(f"group norm takes at most {MAX_CHANNELS} channels")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float32:
            raise TypeError(f"group norm {name} must be a float32 tensor or None")
        if tuple(t.shape) != (channels,):
            raise ValueError(f"group norm {name} must have shape (channels,)")
    if offsets is not None:
        if not isinstance(offsets, torch.Tensor) or offsets.dtype != torch.int64:
            raise TypeError("group norm offsets must be an int64 tensor")
        if offsets.ndim != 1 or offsets.numel() < 2:
            raise ValueError("group norm offsets must be a one-dimensional prefix sum")
    if activation not in _ACTIVATIONS:
        raise ValueError("group norm activation must be None, 'silu' or 'sigmoid'")
    present = [t for t in (x, weight, bias, offsets) if t is not None]
    if not all(t.is_contiguous() for t in present):
        raise ValueError("group norm inputs must be contiguous")
    if len({t.device for t in present}) != 1:
        raise ValueError("all group norm inputs must share a device")
    try:
        eps = float(eps)
    except (TypeError, ValueError) as error:
        raise ValueError("group norm eps must be a finite positive number") from error
    if not math.isfinite(eps) or eps <= 0.0:
        raise ValueError("group norm eps must be a finite positive number")
    return eps


def group_norm(x: torch.Tensor, groups: int, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1.0e-5, *,
               activation: str | None = None, offsets: torch.Tensor | None = None):
    """``act((x - mean) * rstd * weight + bias)``, same shape and dtype as ``x``.

    ``x`` float32 or bfloat16, contiguous, channels last: ``(B, ..., C)``, a
    frame per leading entry, or with ``offsets`` int64 ``(B + 1,)`` packed
    ``(T, ..., C)``, frame ``b`` holding ``x[offsets[b]:offsets[b + 1]]``
    (empty frames allowed).  ``offsets`` cover ``x``: from 0, never falling, to
    ``T``; rows of no frame are left unwritten (checked with
    ``DPA4_CHECK_GROUPING=1``).  ``mean`` and the biased variance run over all of
    a frame's values in each of ``groups`` equal channel groups; an infinity
    or NaN among them makes all of them NaN.  ``weight`` /
    ``bias`` float32 ``(C,)`` or ``None``; ``activation`` ``None``, ``"silu"``
    or ``"sigmoid"``.  Statistics and arithmetic are float32, with one rounding
    to the output.  Gradients for ``x``, ``weight`` and ``bias``, once (second
    and forward-mode derivatives raise); results repeat bit for bit.  Whether a
    CTA takes whole frames goes by their mean size: a long frame among many
    short ones is slow.
    """
    eps = _validate(x, groups, weight, bias, eps, activation, offsets)
    require_dcu(x)  # the others share its device
    if offsets is not None and _segment._should_check(None):
        _segment.check_indices(offsets, x.shape[0], name="group norm")
    return _entry("group_norm")(x, groups, weight, bias, eps, _ACTIVATIONS[activation], offsets)


__all__ = ["MAX_CHANNELS", "group_norm"]
