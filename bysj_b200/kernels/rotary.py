"""Rotary positions with several axes on B200, with position gradients.

``rotary_axes(q, k, positions, inv_freq, sections)`` turns the channel pairs
of every head of ``q`` and ``k`` by ``positions[t, axis] * inv_freq[pair]``,
each axis (x, y, z of an atom; time, height, width of a grid) owning a section
of the pairs.  Both tensors go through one launch.  Float positions are
differentiable once, so an energy that depends on coordinates through its
attention scores gives forces (but a loss of those forces no gradient).  No
reference counterpart.
"""
from __future__ import annotations

from typing import Sequence

import torch

from .native import _entry, require_dcu

MAX_AXES = 4


def _validate(q, k, positions, inv_freq, sections) -> list[int]:
    for name, x in (("q", q), ("k", k)):
        if x is None and name == "k":
            continue
        if not isinstance(x, torch.Tensor):
            raise TypeError(f"rotary {name} must be a tensor")
        if x.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"rotary {name} must be float32 or bfloat16")
        if x.ndim != 3:
            raise ValueError(f"rotary {name} must have shape (tokens, heads, dim)")
        if x.shape[2] < 1:
            raise ValueError(f"rotary {name} must have at least one channel")
        if x.shape[2] > 1 and x.stride(2) != 1:
            raise ValueError(f"rotary {name} channels must be contiguous")
    for name, x in (("positions", positions), ("inv_freq", inv_freq)):
        if not isinstance(x, torch.Tensor):
            raise TypeError(f"rotary {name} must be a tensor")
    if k is not None:
        if k.dtype != q.dtype:
            raise TypeError("rotary q and k must have one dtype")
        if k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
            raise ValueError("rotary q and k must have the same tokens and dim")
    if positions.dtype not in (torch.float32, torch.int64):
        raise TypeError("rotary positions must be float32 or int64")
    if inv_freq.dtype != torch.float32:
        raise TypeError("rotary inv_freq must be float32")
    if inv_freq.requires_grad:
        raise RuntimeError("rotary inv_freq has no gradient; detach it")
    try:
        sections = [int(s) for s in sections]
    except (TypeError, ValueError) as error:
        raise ValueError("rotary sections must be a sequence of pair counts") from error
    if not 1 <= len(sections) <= MAX_AXES or min(sections) < 0:
        raise ValueError(f"rotary sections must be 1 to {MAX_AXES} non-negative pair counts")
    if tuple(positions.shape) != (q.shape[0], len(sections)):
        raise ValueError("rotary positions must have shape (tokens, axes)")
    if 2 * sum(sections) > q.shape[2]:
        raise ValueError("rotary sections hold more pairs than half the channels")
    if tuple(inv_freq.shape) != (sum(sections),):
        raise ValueError("rotary inv_freq must have shape (sum(sections),)")
    if not positions.is_contiguous() or not inv_freq.is_contiguous():
        raise ValueError("rotary positions and inv_freq must be contiguous")
    if len({x.device for x in (q, k, positions, inv_freq) if x is not None}) != 1:
        raise ValueError("all rotary inputs must share a device")
    return sections


def rotary_axes(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor,
                inv_freq: torch.Tensor, sections: Sequence[int], *, interleaved: bool = False):
    """Turned ``(q, k)``, new contiguous tensors of the inputs' dtype.

    ``q`` ``(T, Hq, D)`` and ``k`` ``(T, Hk, D)`` (or ``None``) float32 or
    bfloat16, contiguous along the channels (views of a fused projection are
    fine); ``positions`` ``(T, axes)`` float32 or int64; ``inv_freq`` float32,
    one per pair; ``sections`` the number of pairs of each of up to four axes,
    ``P = sum(sections) <= D / 2``.  Pair ``p`` is channels ``(p, p + P)``, or
    ``(2p, 2p + 1)`` when ``interleaved``; channels from ``2P`` on are copied.
    The angle is a float32 product and sine, cosine and rotation are float32,
    with one rounding to the output: at an angle of ``a`` radians the product's
    rounding is ``a 2^-24``, and int64 positions beyond ``2^24`` are rounded to
    float32 first.  Gradients for ``q``, ``k`` and float ``positions`` (not for
    ``inv_freq``), once: a second derivative (a loss of forces that come from
    positions) raises, as a forward-mode derivative does.
    """
    sections = _validate(q, k, positions, inv_freq, sections)
    require_dcu(q)  # the others share its device
    other = q.new_empty((q.shape[0], 0, q.shape[2])) if k is None else k
    yq, yk = _entry("rotary_axes")(q, other, positions, inv_freq, sections, bool(interleaved))
    return yq, (None if k is None else yk)


__all__ = ["MAX_AXES", "rotary_axes"]
