"""float64 NumPy ground truth of the training-step operators (test infrastructure only).

``rotary_axes``, ``group_norm``, ``route_experts`` and ``adamw`` with their
gradients, written from the formulas; the gradients are themselves checked
against differences of the forward functions in the CPU tests.
"""
from __future__ import annotations

import numpy as np

BLOCK = 256


# ---- rotary positions -----------------------------------------------------------

def _angles(positions, inv_freq, sections):
    axis = np.repeat(np.arange(len(sections)), sections)
    return np.asarray(positions, np.float64)[:, axis] * np.asarray(inv_freq, np.float64)


def _pair_index(pairs, interleaved):
    p = np.arange(pairs)
    return (2 * p, 2 * p + 1) if interleaved else (p, p + pairs)


def rotary(x, positions, inv_freq, sections, interleaved=False, inverse=False):
    x = np.asarray(x, np.float64)
    theta = _angles(positions, inv_freq, sections)[:, None]
    cos, sin = np.cos(theta), np.sin(theta) * (-1.0 if inverse else 1.0)
    a, b = _pair_index(sum(sections), interleaved)
    y = x.copy()
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    return y


def rotary_position_grad(xs, grads, positions, inv_freq, sections, interleaved=False):
    a, b = _pair_index(sum(sections), interleaved)
    dtheta = np.zeros((np.shape(positions)[0], sum(sections)))
    for x, g in zip(xs, grads):
        y = rotary(x, positions, inv_freq, sections, interleaved)
        g = np.asarray(g, np.float64)
        dtheta += (g[..., b] * y[..., a] - g[..., a] * y[..., b]).sum(1)
    weighted = dtheta * np.asarray(inv_freq, np.float64)
    edges = np.concatenate([[0], np.cumsum(sections)])
    return np.stack([weighted[:, i:j].sum(1) for i, j in zip(edges[:-1], edges[1:])], 1)


# ---- group norm -------------------------------------------------------------------

def _sigmoid(z):
    return 1.0 / (1.0 + np.exp(-z))


def _activation(z, name):
    if name == "silu":
        s = _sigmoid(z)
        return z * s, s * (1.0 + z * (1.0 - s))
    if name == "sigmoid":
        s = _sigmoid(z)
        return s, s * (1.0 - s)
    return z, np.ones_like(z)


def group_norm(x, offsets, groups, weight, bias, eps, activation, grad=None):
    """x [T, ..., C] with frame offsets [B + 1]; (y, (gx, gw, gb) or None)."""
    x = np.asarray(x, np.float64)
    c = x.shape[-1]
    w = np.ones(c) if weight is None else np.asarray(weight, np.float64)
    b = np.zeros(c) if bias is None else np.asarray(bias, np.float64)
    y, gx = np.zeros_like(x), np.zeros_like(x)
    gw, gb = np.zeros(c), np.zeros(c)
    for lo, hi in zip(offsets[:-1], offsets[1:]):
        if hi <= lo or x[lo:hi].size == 0:
            continue
        v = x[lo:hi].reshape(-1, groups, c // groups)
        mean = v.mean((0, 2), keepdims=True)
        rstd = 1.0 / np.sqrt(((v - mean) ** 2).mean((0, 2), keepdims=True) + eps)
        xhat = ((v - mean) * rstd).reshape(-1, c)
        value, slope = _activation(xhat * w + b, activation)
        y[lo:hi] = value.reshape(x[lo:hi].shape)
        if grad is None:
            continue
        dz = np.asarray(grad, np.float64)[lo:hi].reshape(-1, c) * slope
        gw += (dz * xhat).sum(0)
        gb += dz.sum(0)
        d, h = (dz * w).reshape(v.shape), xhat.reshape(v.shape)
        dx = rstd * (d - d.mean((0, 2), keepdims=True) - h * (d * h).mean((0, 2), keepdims=True))
        gx[lo:hi] = dx.reshape(x[lo:hi].shape)
    return y, (None if grad is None else (gx, gw, gb))


# ---- router -----------------------------------------------------------------------

def route(logits, k, mask=None, offsets=None, renormalize=False, grads=None):
    """(weights, experts, counts, balance, z, grad_logits or None); grads = (gw, g_balance, g_z)."""
    x = np.asarray(logits, np.float64)
    tokens, n_experts = x.shape
    valid = np.ones(tokens, bool) if mask is None else np.asarray(mask, bool).copy()
    valid &= (x != -np.inf).any(1) if n_experts else False
    offsets = [0, tokens] if offsets is None else list(offsets)
    weights, experts = np.zeros((tokens, k)), np.full((tokens, k), -1, np.int64)
    p, lse = np.zeros_like(x), np.zeros(tokens)
    for t in np.flatnonzero(valid):
        top = x[t].max()
        e = np.where(x[t] == -np.inf, 0.0, np.exp(np.where(x[t] == -np.inf, 0.0, x[t] - top)))
        p[t], lse[t] = e / e.sum(), top + np.log(e.sum())
        order = [i for i in np.argsort(-x[t], kind="stable") if x[t, i] != -np.inf][:k]
        experts[t, :len(order)] = order
        weights[t, :len(order)] = p[t, order]
        if renormalize:
            weights[t] /= weights[t].sum()
    frames = len(offsets) - 1
    counts, share, used = np.zeros((frames, n_experts), np.int64), np.zeros((frames, n_experts)), 0
    balance = 0.0
    for s, (lo, hi) in enumerate(zip(offsets[:-1], offsets[1:])):
        n = int(valid[lo:hi].sum())
        if n == 0:
            continue
        used += 1
        chosen = experts[lo:hi][experts[lo:hi] >= 0]
        counts[s] = np.bincount(chosen, minlength=n_experts)
        share[s] = n_experts * counts[s] / (k * n * n)
        balance += (share[s] * p[lo:hi].sum(0)).sum()
    balance, share = balance / max(used, 1), share / max(used, 1)
    n = max(int(valid.sum()), 1)
    z = float((lse ** 2).sum() / n)
    grad = None
    if grads is not None:
        gw, g_balance, g_z = grads
        grad = np.zeros_like(x)
        frame = np.repeat(np.arange(frames), np.diff(offsets))
        for t in np.flatnonzero(valid):
            cot, direct = g_balance * share[frame[t]], np.zeros(n_experts)
            slots = experts[t] >= 0
            index, g = experts[t][slots], np.asarray(gw, np.float64)[t][slots]
            if renormalize:
                w = weights[t][slots]
                direct[index] = w * (g - (w * g).sum())
            else:
                cot = cot.copy()
                cot[index] += g
            grad[t] = p[t] * (cot - (p[t] * cot).sum()) + direct + g_z * 2.0 / n * lse[t] * p[t]
    return weights, experts, counts, balance, z, grad


# ---- AdamW ------------------------------------------------------------------------

def code_values(top, mantissa):
    """Values of the codes 0 .. top: 0, then steps of one mantissa unit up to 1."""
    code = np.arange(1, top + 1)
    octave, part = np.divmod(code - top, 1 << mantissa)
    return np.concatenate([[0.0], 2.0 ** octave * (1.0 + part / (1 << mantissa))])


VALUES_M, VALUES_V = code_values(127, 3), code_values(255, 4)


def adamw(p, g, m, v, step, lr, betas, eps, weight_decay, grad_scale=1.0):
    """One step on float64 arrays: (p, m, v)."""
    g = g * grad_scale
    m = betas[0] * m + (1.0 - betas[0]) * g
    v = betas[1] * v + (1.0 - betas[1]) * g * g
    update = (m / (1.0 - betas[0] ** step)) / (np.sqrt(v / (1.0 - betas[1] ** step)) + eps)
    return p - lr * (update + weight_decay * p), m, v


def adamw_f32(p, g, m, v, step, lr, betas, eps, weight_decay, grad_scale=None):
    """The same step in float32, one rounding an operation: the kernels' arithmetic."""
    f = np.float32
    if grad_scale is not None:
        g = g * f(grad_scale)
    m = m * f(betas[0]) + g * f(1.0 - betas[0])
    v = v * f(betas[1]) + g * f(1.0 - betas[1]) * g
    root = np.sqrt(v)
    correct, size = f(1.0 / np.sqrt(1.0 - betas[1] ** step)), f(lr / (1.0 - betas[0] ** step))
    p = p * f(1.0 - lr * weight_decay) - m / (root * correct + f(eps)) * size
    return p, m, v, root


def philox4x32(counter, key, rounds):
    """Philox 4x32 (Salmon et al., 2011) of counters [n, 4] and one 64-bit key."""
    c = [np.asarray(counter, np.uint64)[:, i] for i in range(4)]
    low = np.uint64(0xFFFFFFFF)
    k = [key & 0xFFFFFFFF, key >> 32]
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low,
             (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1)


def rounding_noise(step, length, betas):
    """Numbers in (0, 1) that round the codes of m and of sqrt(v) at ``step``, [length / BLOCK, BLOCK].

    ``None`` for a moment that a step decays by at least half a code, which
    is rounded to the nearest.
    """
    quads = np.zeros((length // 4, 4), np.uint64)
    quads[:, 0] = np.arange(length // 4)
    words = philox4x32(quads, step, 7).reshape(-1, BLOCK)
    noise = [((words >> np.uint64(16 * i) & np.uint64(0xFFFF)) + 0.5) / 65536.0 for i in range(2)]
    return [n if 1.0 - beta < least else None
            for n, beta, least in zip(noise, betas, (1 / 16, 1 / 64))]


def encode(x, top, values, noise=None):
    """Codes of non-negative float32 blocks [n, BLOCK] by nearest value, and their scales.

    A tie goes to the even mantissa (the odd code: the top code is odd).  The
    ratio is the float32 product with the float32 inverse of the scale.  With
    ``noise`` in (0, 1) a ratio between two values takes the upper one where
    the part of the gap above it does not exceed the noise.
    """
    scale = x.max(1)
    with np.errstate(divide="ignore", over="ignore", invalid="ignore"):
        inverse = np.where(scale > 0, np.float32(1.0) / scale, np.float32(0.0)).astype(np.float32)
        ratio = (x * inverse[:, None]).astype(np.float64)
    ratio[x == 0] = 0.0  # also where the inverse is infinite
    if noise is not None:
        ratio = np.minimum(ratio, 1.0)
        lower = np.searchsorted(values, ratio, side="right") - 1
        upper = np.minimum(lower + 1, top)
        gap = np.where(upper > lower, values[upper] - values[lower], 1.0)
        code = np.where((ratio - values[lower]) / gap + noise >= 1.0, upper, lower)
        if top == 255:
            code = np.where(x > 0, np.maximum(code, 1), 0)
        return code.astype(np.uint8), scale
    middle = (values[1:] + values[:-1]) / 2
    code = np.searchsorted(middle, ratio, side="left")
    tie = (code < top) & (ratio == middle[np.minimum(code, top - 1)]) & (code % 2 == 0)
    code = code + tie
    if top == 255:
        code = np.where(x > 0, np.maximum(code, 1), 0)
    return code.astype(np.uint8), scale


def decode(code, scale, values):
    return (values[code].astype(np.float32) * scale[:, None]).astype(np.float32)


__all__ = ["BLOCK", "VALUES_M", "VALUES_V", "adamw", "adamw_f32", "code_values", "decode",
           "encode", "group_norm", "philox4x32", "rotary", "rotary_position_grad",
           "rounding_noise", "route"]
