"""Top-k expert router with counts, balance loss and z loss on B200.

``route_experts(logits, k)`` picks each token's experts and gate weights and
in the same pass gathers what the auxiliary losses need: per-expert counts,
the balance loss (per frame with ``offsets``) and the z loss, all with
gradients for the logits.  ``group_by_source(experts.flatten(), n_experts)``
then groups the tokens of each expert.  No reference counterpart.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import segment as _segment
from .native import _entry, require_dcu

MAX_EXPERTS = 1024
MAX_K = 32


class Routing(NamedTuple):
    """Result of :func:`route_experts`."""

    weights: torch.Tensor  # float32 (tokens, k)
    experts: torch.Tensor  # int64 (tokens, k), -1 in an empty slot
    counts: torch.Tensor   # int64 (experts,), or (frames, experts) with offsets
    balance: torch.Tensor  # float32 scalar
    z: torch.Tensor        # float32 scalar


def _validate(logits, k, mask, offsets):
    if not isinstance(logits, torch.Tensor):
        raise TypeError("router logits must be a tensor")
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("router logits must be float32 or bfloat16")
    if logits.ndim != 2:
        raise ValueError("router logits must have shape (tokens, experts)")
    experts = int(logits.shape[1])
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"router takes 1 to {MAX_EXPERTS} experts")
    if isinstance(k, bool) or not isinstance(k, int):
        raise TypeError("router k must be an int")
    if not 1 <= k <= min(experts, MAX_K):
        raise ValueError(f"router k must be between 1 and min(experts, {MAX_K})")
    if mask is not None:
        if not isinstance(mask, torch.Tensor) or mask.dtype != torch.bool:
            raise TypeError("router mask must be a bool tensor")
        if tuple(mask.shape) != (logits.shape[0],):
            raise ValueError("router mask must have shape (tokens,)")
    if offsets is not None:
        if not isinstance(offsets, torch.Tensor) or offsets.dtype != torch.int64:
            raise TypeError("router offsets must be an int64 tensor")
        if offsets.ndim != 1 or offsets.numel() < 2:
            raise ValueError("router offsets must be a one-dimensional prefix sum")
    present = [t for t in (logits, mask, offsets) if t is not None]
    if not all(t.is_contiguous() for t in present):
        raise ValueError("router inputs must be contiguous")
    if len({t.device for t in present}) != 1:
        raise ValueError("all router inputs must share a device")


def route_experts(logits: torch.Tensor, k: int, *, mask: torch.Tensor | None = None,
                  offsets: torch.Tensor | None = None, renormalize: bool = False) -> Routing:
    """Route each token to its ``k`` largest logits; a :class:`Routing` tuple.

    ``logits`` float32 or bfloat16 ``(T, E)``, ``E <= 1024``, ``k <= 32``;
    ``p = softmax(logits)`` in float32.  Ties go to the lowest index.  An
    expert at ``-inf`` is never chosen; where fewer than ``k`` are left the
    slots are ``-1`` with weight 0.  ``weights`` is ``p`` at the chosen
    experts, divided by its sum with ``renormalize``.  Tokens with a false
    ``mask`` (or without a logit above ``-inf``) are left out of everything,
    whatever their logits and their cotangents hold; so are empty slots.

    ``balance``: the mean over frames (``offsets`` int64 ``(S + 1,)``; without
    it all tokens are one) with ``n > 0`` tokens of
    ``E / (k n^2) sum_e counts_e sum_t p_te``, 1 when the load is even;
    ``counts`` is a constant to it.  ``z``: the mean of ``logsumexp^2``.
    ``weights``, ``balance`` and ``z`` are differentiable, once (second and
    forward-mode derivatives raise).  ``offsets`` cover the tokens, from 0, never
    falling, to ``T`` (checked with ``DPA4_CHECK_GROUPING=1``): tokens before the
    first count with the first frame, tokens after the last with the last.
    """
    _validate(logits, k, mask, offsets)
    require_dcu(logits)  # the others share its device
    if offsets is not None and _segment._should_check(None):
        _segment.check_indices(offsets, logits.shape[0], name="router")
    return Routing(*_entry("route_experts")(logits, k, mask, offsets, bool(renormalize)))


__all__ = ["MAX_EXPERTS", "MAX_K", "Routing", "route_experts"]
