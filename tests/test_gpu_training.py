"""Training-step operators on the GPU against their float64 definitions.

Tolerances.  ``U = 2**-24`` and ``B = 2**-8`` are the unit roundoffs of float32
(24 significant bits) and bfloat16 (8), half of ``torch.finfo(dtype).eps``; a
bfloat16 output adds ``B`` times its magnitude to what the float32 arithmetic
leaves.

* rotary: the angle is a float32 product (error ``U |theta|``), sine and
  cosine are within 2 units in the last place, the turn adds two products and
  a sum: ``(U max|theta| + 8 U)`` times the pair's length.  A position
  gradient sums ``heads * pairs`` such terms: that bound times their number
  and largest value.
* group norm: ``x - mean`` carries the rounding of the mean, so values are
  within ``16 U (1 + |mean| rstd)`` of their own scale; the gradients of weight
  and bias sum n terms of that error and either sign (4 sqrt(n)).
* router: a softmax entry is within ``(16 + E / 8) U`` relative (exp, the sum
  of E terms, the division).
* AdamW: the same float32 operations one at a time, bit for bit; the 8-bit
  codes as well.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from bysj_b200 import kernels as K  # noqa: E402
from oracle import training as O  # noqa: E402

U, B = torch.finfo(torch.float32).eps / 2, torch.finfo(torch.bfloat16).eps / 2
F32, BF16 = torch.float32, torch.bfloat16


def half_ulp(dtype):
    return 0.0 if dtype == F32 else B


def f64(t):
    return t.detach().double().cpu().numpy()


def close(got, want, tol):
    got = f64(got) if isinstance(got, torch.Tensor) else got
    assert got.shape == want.shape
    worst = np.max(np.abs(got - want) - tol) if got.size else -1.0
    assert worst <= 0.0, f"off by {worst} beyond the tolerance"


def normal(gen, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- rotary ---------------------------------------------------------------------------

ROTARY = [
    # tokens, q heads, k heads, dim, sections, interleaved, dtype, float positions, packed
    (1, 16, 4, 64, (16, 8, 8), False, BF16, False, True),
    (1, 1, 1, 2, (1,), False, F32, True, False),
    (37, 8, 8, 32, (5, 5, 6), True, F32, True, False),
    (33, 3, 1, 14, (4, 0, 3), False, F32, True, True),
    (129, 5, 2, 7, (1, 2), True, BF16, True, True),
    (5, 2, 2, 66, (33,), False, BF16, False, False),
    (3, 2, 1, 40, (3, 4, 5, 2), False, BF16, True, True),
    (64, 4, 2, 128, (64,), True, F32, False, True),
    (17, 2, 1, 96, (16, 16), False, F32, True, False),
    (9, 7, 3, 48, (8, 8, 8), False, BF16, True, False),
    (4, 1, 0, 8, (2, 2), False, F32, True, False),
    (2, 3, 2, 5, (0, 0), False, F32, True, False),
    (300, 3, 3, 256, (40, 40, 48), False, BF16, True, True),
]


@pytest.mark.parametrize("case", ROTARY, ids=[str(i) for i in range(len(ROTARY))])
def test_rotary_matches_the_definition(cuda, case):
    tokens, hq, hk, dim, sections, inter, dtype, float_pos, packed = case
    gen = generator(tokens + dim)
    if packed:
        qkv = normal(gen, tokens, hq + 2 * hk, dim, dtype=dtype)
        q, k = qkv[:, :hq].detach(), qkv[:, hq:hq + hk].detach()
    else:
        q, k = normal(gen, tokens, hq, dim, dtype=dtype), normal(gen, tokens, hk, dim, dtype=dtype)
    if float_pos:
        pos = torch.rand(tokens, len(sections), generator=gen, device="cuda") * 20.0 - 10.0
    else:
        pos = torch.randint(-50, 50, (tokens, len(sections)), generator=gen, device="cuda")
    freq = torch.rand(sum(sections), generator=gen, device="cuda") + 0.05
    leaves = [q.requires_grad_(), k.requires_grad_()]
    if float_pos:
        leaves.append(pos.requires_grad_())
    out = K.rotary_axes(q, k, pos, freq, sections, interleaved=inter)
    gq, gk = normal(gen, tokens, hq, dim, dtype=dtype), normal(gen, tokens, hk, dim, dtype=dtype)
    grads = torch.autograd.grad(out, leaves, [gq, gk])
    theta = np.abs(f64(pos)).max() * float(freq.max()) if sum(sections) else 0.0
    bound = U * theta + 8 * U
    args = (f64(pos), f64(freq), sections, inter)
    for x, y, g, gx in zip((q, k), out, (gq, gk), grads):
        assert y.is_contiguous() and y.dtype == dtype and gx.dtype == dtype
        for got, given, inverse in ((y, x, False), (gx, g, True)):
            want = O.rotary(f64(given), *args, inverse)
            size = 2.0 * np.abs(f64(given)).max() if want.size else 0.0
            close(got, want, bound * size + half_ulp(dtype) * np.abs(want))
    if float_pos:
        want = O.rotary_position_grad((f64(q), f64(k)), (f64(gq), f64(gk)), *args)
        terms = (hq + hk) * max(max(sections), 1)
        largest = max(np.abs(f64(t)).max() if t.numel() else 0.0 for t in (q, k)) * \
            max(np.abs(f64(t)).max() if t.numel() else 0.0 for t in (gq, gk)) * 4.0
        close(grads[2], want, (bound + terms * U) * terms * largest * 1.05)


def test_rotary_position_gradient_against_differences(cuda):
    gen = generator(3)
    q, k = normal(gen, 11, 3, 12), normal(gen, 11, 2, 12)
    pos = torch.rand(11, 3, generator=gen, device="cuda").requires_grad_()
    freq = torch.tensor([0.3, 1.1, 2.0, 0.7, 0.9], device="cuda")
    gq, gk = normal(gen, 11, 3, 12), normal(gen, 11, 2, 12)
    out = K.rotary_axes(q, k, pos, freq, (2, 2, 1))
    grad, = torch.autograd.grad(out, [pos], [gq, gk])
    way = np.random.default_rng(0).standard_normal((11, 3))

    def value(h):
        at = f64(pos) + h * way
        return sum((O.rotary(f64(x), at, f64(freq), (2, 2, 1)) * f64(g)).sum()
                   for x, g in ((q, gq), (k, gk)))

    h = 1.0e-5
    want = (value(h) - value(-h)) / (2 * h)
    # central differences: h^2 f''' / 6 and rounding 1e-16 |f| / h; float32 sums of 60 terms
    assert abs((f64(grad) * way).sum() - want) <= 1.0e-4 * (np.abs(f64(grad)) * np.abs(way)).sum()


def test_rotary_without_keys_tokens_or_gradients(cuda):
    q = torch.randn(4, 2, 8, device="cuda")
    pos, freq = torch.rand(4, 2, device="cuda"), torch.rand(4, device="cuda")
    y, none = K.rotary_axes(q, None, pos, freq, (2, 2))
    both, _ = K.rotary_axes(q, q, pos, freq, (2, 2))
    assert none is None and torch.equal(y, both)
    y, k = K.rotary_axes(q[:0], q[:0], pos[:0], freq, (2, 2))
    assert y.shape == (0, 2, 8) and k.shape == (0, 2, 8)


# ---- group norm ------------------------------------------------------------------------

NORM = [
    # lengths (or frames x rows), inner, channels, groups, dtype, activation, affine, ragged, shift
    ([192], (), 64, 8, F32, "silu", True, False, 0.0),
    ([5, 0, 1, 700, 33], (), 96, 12, F32, "silu", True, True, 0.5),
    ([5, 0, 1, 70, 33], (3,), 24, 2, BF16, "silu", True, True, 0.5),
    ([40, 40, 40], (4, 2), 16, 16, F32, None, True, False, 0.0),
    ([1, 1], (), 1, 1, F32, "sigmoid", True, False, 0.0),
    ([1], (), 6, 2, F32, None, False, True, 0.0),
    ([300], (), 300, 3, BF16, "silu", True, False, 2.0),
    ([2000, 1], (), 257, 1, F32, "silu", True, True, 0.0),
    ([64, 128], (16,), 64, 32, BF16, None, False, True, 0.0),
    ([513] * 3, (), 128, 32, BF16, "silu", True, False, 1.0),
    ([50, 60], (), 1024, 4, F32, "silu", True, True, 0.0),
    ([500, 300], (), 48, 4, F32, None, True, True, 1000.0),
    ([0, 0, 20000, 0], (), 40, 8, F32, "silu", True, True, 0.0),
    ([3000, 10], (), 8, 1, BF16, "sigmoid", False, True, 0.0),
    # frames cut into slabs, joined across CTAs; vector and single loads
    ([6000, 0, 9000, 1, 4000], (), 64, 8, F32, "silu", True, True, 0.5),
    ([6000, 0, 9000, 1, 4000], (), 65, 5, BF16, "silu", True, True, 0.5),
    ([700] * 9, (16,), 64, 4, F32, "silu", True, False, 0.3),
    ([30000], (), 50, 25, F32, "sigmoid", True, False, 0.0),
    # more slabs than are held at once: the frame is read again
    ([140000], (), 128, 8, F32, "silu", True, False, 0.3),
    ([5, 260000, 0, 9000], (), 72, 3, BF16, "silu", True, True, 0.3),
]


def make_norm(case, seed=0):
    lengths, inner, channels, groups, dtype, act, affine, ragged, shift = case
    gen = generator(seed + channels)
    total = sum(lengths)
    shape = (total, *inner, channels) if ragged else (len(lengths), lengths[0], *inner, channels)
    x = (normal(gen, *shape) + shift).to(dtype)
    grad = normal(gen, *shape, dtype=dtype)
    w = b = None
    if affine:
        w = torch.rand(channels, generator=gen, device="cuda") + 0.5
        b = normal(gen, channels, scale=0.3)
    offsets = np.concatenate([[0], np.cumsum(lengths)])
    return x, grad, w, b, offsets


@pytest.mark.parametrize("case", NORM, ids=[str(i) for i in range(len(NORM))])
def test_group_norm_matches_the_definition(cuda, case):
    lengths, inner, channels, groups, dtype, act, affine, ragged, shift = case
    x, grad, w, b, offsets = make_norm(case)
    leaves = [t.requires_grad_() for t in (x, w, b) if t is not None]
    given = torch.from_numpy(offsets).cuda() if ragged else None
    y = K.group_norm(x, groups, w, b, 1.0e-5, activation=act, offsets=given)
    grads = torch.autograd.grad(y, leaves, grad)
    assert y.shape == x.shape and y.dtype == dtype
    flat = f64(x).reshape(-1, *inner, channels)
    want, (gx, gw, gb) = O.group_norm(flat, offsets, groups, None if w is None else f64(w),
                                      None if b is None else f64(b), 1.0e-5, act,
                                      f64(grad).reshape(flat.shape))
    # a frame of one value has rstd = 1 / sqrt(eps) = 316; otherwise at most about 1 / std = 2
    single = min([n for n in lengths if n > 0]) * int(np.prod(inner)) * (channels // groups)
    rstd = 317.0 if single < 2 else 1.0 / np.sqrt(1.0e-5 + 0.0004) if single < 8 else 2.0
    off = 16 * U * (2.0 + abs(shift) * rstd)
    wmax = 1.5 if affine else 1.0
    xhat = 6.0
    close(y.reshape(flat.shape), want, off * wmax * xhat + half_ulp(dtype) * np.abs(want))
    # dx sums rstd (d - mean d - xhat mean(d xhat)), |act''| <= 1/2: the error of z enters d
    d = np.abs(f64(grad)).max() * 1.1 * wmax
    close(grads[0].reshape(flat.shape), gx,
          rstd * off * d * (2.0 + 2.0 * xhat * xhat) * wmax + half_ulp(dtype) * np.abs(gx))
    if affine:
        n = sum(lengths) * int(np.prod(inner))
        for got, want in ((grads[1], gw), (grads[2], gb)):
            close(got, want, 4 * np.sqrt(n) * off * d * xhat * wmax + 2 * U * np.abs(want))


def test_group_norm_gradient_against_differences(cuda):
    case = ([7, 0, 12], (2,), 6, 2, F32, "silu", True, True, 0.3)
    x, grad, w, b, offsets = make_norm(case)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = K.group_norm(x, 2, w, b, activation="silu", offsets=torch.from_numpy(offsets).cuda())
    grads = torch.autograd.grad(y, leaves, grad)
    rng = np.random.default_rng(1)
    ways = [rng.standard_normal(t.shape) for t in leaves]

    def value(h):
        at = [f64(t) + h * way for t, way in zip(leaves, ways)]
        return (O.group_norm(at[0], offsets, 2, at[1], at[2], 1.0e-5, "silu")[0] * f64(grad)).sum()

    h = 1.0e-5
    want = (value(h) - value(-h)) / (2 * h)
    got = sum((f64(g) * way).sum() for g, way in zip(grads, ways))
    size = sum((np.abs(f64(g)) * np.abs(way)).sum() for g, way in zip(grads, ways))
    assert abs(got - want) <= 1.0e-5 * size


def test_group_norm_repeats_and_keeps_frames_apart(cuda):
    case = ([700, 300, 1], (), 40, 8, F32, "silu", True, True, 0.0)
    x, grad, w, b, offsets = make_norm(case)
    given = torch.from_numpy(offsets).cuda()
    first = K.group_norm(x, 8, w, b, activation="silu", offsets=given)
    assert torch.equal(first, K.group_norm(x, 8, w, b, activation="silu", offsets=given))
    poisoned = x.clone()
    poisoned[700:1000] = float("nan")
    other = K.group_norm(poisoned, 8, w, b, activation="silu", offsets=given)
    assert torch.equal(other[:700], first[:700]) and torch.equal(other[1000:], first[1000:])
    assert torch.isnan(other[700:1000]).all()


def test_group_norm_empty_tensor(cuda):
    w = torch.ones(8, device="cuda", requires_grad=True)
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    y = K.group_norm(x, 2, w, offsets=torch.zeros(3, dtype=torch.int64, device="cuda"))
    gx, gw = torch.autograd.grad(y, [x, w], torch.zeros_like(y))
    assert y.shape == (0, 8) and gx.shape == (0, 8) and torch.equal(gw, torch.zeros_like(w))


# ---- router ---------------------------------------------------------------------------

ROUTE = [
    # tokens, experts, k, lengths or None, masked, renormalize, dtype, barred share, ties
    (1, 64, 4, None, False, True, F32, 0.0, False),
    (1, 1, 1, None, False, False, F32, 0.0, False),
    (50, 8, 8, None, False, True, F32, 0.0, True),
    (300, 16, 2, [100, 0, 1, 199], True, False, F32, 0.0, False),
    (257, 33, 5, [257], True, True, BF16, 0.2, False),
    (100, 128, 8, None, False, True, BF16, 0.0, True),
    (40, 1024, 32, [7, 33], False, False, F32, 0.1, False),
    (64, 5, 3, None, True, True, F32, 0.7, False),
    (512, 256, 6, [64] * 8, False, False, BF16, 0.0, False),
    (1000, 2, 1, None, False, False, F32, 0.0, True),
    (33, 100, 3, [0, 0, 33], True, False, F32, 0.0, False),
]


def make_route(case, seed=0):
    tokens, experts, k, lengths, masked, renorm, dtype, barred, ties = case
    gen = generator(seed + experts)
    logits = normal(gen, tokens, experts, scale=2.0)
    if ties:
        logits = torch.round(logits)
    if barred:
        drop = torch.rand(tokens, experts, generator=gen, device="cuda") < barred
        logits = torch.where(drop, float("-inf"), logits)
    logits = logits.to(dtype)
    mask = None
    if masked:
        mask = torch.rand(tokens, generator=gen, device="cuda") < 0.8
    offsets = None if lengths is None else np.concatenate([[0], np.cumsum(lengths)])
    grads = (normal(gen, tokens, k), torch.tensor(0.7 * tokens, device="cuda"),
             torch.tensor(0.1 * tokens, device="cuda"))
    return logits, mask, offsets, grads


@pytest.mark.parametrize("case", ROUTE, ids=[str(i) for i in range(len(ROUTE))])
def test_router_matches_the_definition(cuda, case):
    tokens, experts, k, lengths, masked, renorm, dtype, barred, ties = case
    logits, mask, offsets, grads = make_route(case)
    x = logits.clone()
    if mask is not None:  # what a masked token holds has no effect
        x[~mask] = float("nan")
    x.requires_grad_()
    given = None if offsets is None else torch.from_numpy(offsets).cuda()
    r = K.route_experts(x, k, mask=mask, offsets=given, renormalize=renorm)
    grad, = torch.autograd.grad([r.weights, r.balance, r.z], [x], list(grads))
    want = O.route(f64(logits), k, None if mask is None else mask.cpu().numpy(), offsets, renorm,
                   (f64(grads[0]), float(grads[1]), float(grads[2])))
    np.testing.assert_array_equal(r.experts.cpu().numpy(), want[1])
    counts = r.counts.cpu().numpy()
    np.testing.assert_array_equal(counts if offsets is not None else counts[None], want[2])
    rel = (16 + experts / 8) * U
    close(r.weights, want[0], 2 * rel * want[0])
    assert r.balance.shape == () and r.z.shape == ()
    close(r.balance.reshape(1), np.array([want[3]]), rel * abs(want[3]) + 1e-9)
    # lse = max + log(sum): |max| <= 10 here
    close(r.z.reshape(1), np.array([want[4]]), rel * 10.0 * 2.0 * np.sqrt(want[4]) + U * want[4])
    # the cotangent of p: the weights', the balance loss's E counts / (k n^2), the z loss's 2 lse / n
    valid = (want[1][:, 0] >= 0).astype(np.int64)
    edges = np.array([0, tokens]) if offsets is None else offsets
    n = np.maximum([valid[a:b].sum() for a, b in zip(edges[:-1], edges[1:])], 1)
    scale = np.abs(f64(grads[0])).max() + \
        float(grads[1]) * (experts / k * want[2].max(1) / n ** 2).max() + \
        float(grads[2]) * 2.0 / max(valid.sum(), 1) * 15.0
    close(grad, want[5], 4 * rel * scale + half_ulp(dtype) * np.abs(want[5]))
    assert torch.equal(r.experts, K.route_experts(x.detach(), k, mask=mask, offsets=given).experts)


def test_router_gradient_against_differences(cuda):
    case = (40, 7, 2, [10, 30], True, True, F32, 0.0, False)
    logits, mask, offsets, grads = make_route(case)
    x = logits.clone().requires_grad_()
    r = K.route_experts(x, 2, mask=mask, offsets=torch.from_numpy(offsets).cuda(),
                        renormalize=True)
    grad, = torch.autograd.grad([r.weights, r.balance, r.z], [x], list(grads))
    way = np.random.default_rng(2).standard_normal(x.shape)

    def value(h):
        w, _, _, balance, z, _ = O.route(f64(x) + h * way, 2, mask.cpu().numpy(), offsets, True)
        return (w * f64(grads[0])).sum() + balance * float(grads[1]) + z * float(grads[2])

    h = 1.0e-5  # small enough that no choice of expert changes
    want = (value(h) - value(-h)) / (2 * h)
    assert abs((f64(grad) * way).sum() - want) <= 1.0e-5 * (np.abs(f64(grad)) * np.abs(way)).sum()


def test_router_empty_rows_nan_and_zero_signs(cuda):
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[-inf, -inf, -inf], [0.0, -0.0, -1.0], [-0.0, 0.0, 0.0], [1.0, -inf, -inf],
                      [-3.4028234663852886e38, -inf, -inf]], device="cuda", requires_grad=True)
    r = K.route_experts(x, 2)
    assert r.experts.tolist() == [[-1, -1], [0, 1], [0, 1], [0, -1], [0, -1]]
    assert r.weights[0].tolist() == [0.0, 0.0] and r.weights[3].tolist() == [1.0, 0.0]
    assert r.counts.tolist() == [4, 2, 0]
    grad, = torch.autograd.grad(r.weights.sum() + r.balance, [x])
    assert torch.equal(grad[0], torch.zeros(3, device="cuda")) and torch.isfinite(grad).all()
    # nothing valid at all: losses are 0
    empty = K.route_experts(torch.full((4, 3), -inf, device="cuda"), 1)
    assert float(empty.balance) == 0.0 and float(empty.z) == 0.0
    empty = K.route_experts(torch.zeros(0, 3, device="cuda"), 2,
                            offsets=torch.zeros(2, dtype=torch.int64, device="cuda"))
    assert float(empty.balance) == 0.0 and empty.weights.shape == (0, 2)
    # a NaN that is not masked shows in the weights and in both losses
    bad = K.route_experts(torch.tensor([[nan, 1.0], [0.0, 1.0]], device="cuda"), 1)
    assert torch.isnan(bad.weights[0]).all() and torch.isnan(bad.balance) and torch.isnan(bad.z)


def test_router_groups_tokens_for_the_experts(cuda):
    x = torch.randn(500, 6, generator=generator(5), device="cuda")
    r = K.route_experts(x, 2)
    order, offsets = K.group_by_source(r.experts.flatten(), 6)
    assert torch.equal(offsets[1:] - offsets[:-1], r.counts)
    assert order.numel() == 1000


# ---- AdamW ------------------------------------------------------------------------------

SIZES = [(1,), (255,), (256,), (257, 1), (3, 1000), (0,), (31, 33), (5120,)]
HYPER = dict(lr=0.01, betas=(0.9, 0.97), eps=1e-8, weight_decay=0.1)


def make_params(gen, sizes, dtypes, flat):
    if flat:  # views at odd offsets of one buffer
        buffer = normal(gen, sum(int(np.prod(s)) for s in sizes) + 1, dtype=dtypes[0])[1:]
        parts = buffer.split([int(np.prod(s)) for s in sizes])
        return [t.view(s) for t, s in zip(parts, sizes)]
    return [normal(gen, *s, dtype=dtypes[i % len(dtypes)]) for i, s in enumerate(sizes)]


def padded(t, length):
    out = np.zeros(length, np.float32)
    out[:t.numel()] = t.detach().float().cpu().numpy().reshape(-1)
    return out


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("dtypes,flat", [((F32,), False), ((BF16,), False), ((F32, BF16), False),
                                         ((F32,), True), ((BF16,), True)])
def test_adamw_steps_match_bit_for_bit(cuda, bits, master, dtypes, flat):
    gen = generator(bits)
    params = make_params(gen, SIZES, dtypes, flat)
    opt = K.AdamW(params, **HYPER, state_bits=bits, master_weights=master)
    lengths = [-(-p.numel() // O.BLOCK) * O.BLOCK for p in params]
    p32 = [padded(p, n) for p, n in zip(params, lengths)]
    m = [np.zeros(n, np.float32) for n in lengths]
    v = [np.zeros(n, np.float32) for n in lengths]
    for step in (1, 2, 3):
        grads = make_params(gen, SIZES, dtypes, flat)
        if step == 2:  # a wide range of magnitudes, zeros among them
            for g in grads:
                g.mul_(torch.exp(normal(gen, *g.shape, scale=6.0)).to(g.dtype))
                g[..., ::3] = 0.0
        grads = [g if i != 4 or step != 3 else None for i, g in enumerate(grads)]
        scale = torch.full((1,), 0.37, device="cuda") if step > 1 else None
        opt.step(grads, grad_scale=scale)
        for i, (p, g) in enumerate(zip(params, grads)):
            if g is None or p.numel() == 0:
                continue
            out = O.adamw_f32(p32[i], padded(g, lengths[i]), m[i], v[i], step, HYPER["lr"],
                              HYPER["betas"], HYPER["eps"], HYPER["weight_decay"],
                              None if scale is None else 0.37)
            p32[i], m[i], v[i], root = out
            begin = opt.begins[i]
            if bits == 8:
                whole = m[i].reshape(-1, O.BLOCK)
                code, size = O.encode(np.abs(whole), 127, O.VALUES_M)
                signed = np.where(whole < 0, code + 128, code).astype(np.uint8)
                at = slice(begin, begin + lengths[i])
                np.testing.assert_array_equal(opt.exp_avg[at].cpu().numpy(), signed.reshape(-1))
                m[i] = (np.where(whole < 0, -1, 1) * O.decode(code, size, O.VALUES_M)).astype(
                    np.float32).reshape(-1)
                code, size = O.encode(root.reshape(-1, O.BLOCK), 255, O.VALUES_V)
                np.testing.assert_array_equal(opt.exp_avg_sq[at].cpu().numpy(), code.reshape(-1))
                v[i] = O.decode(code, size, O.VALUES_V).reshape(-1) ** 2
            n = p.numel()
            rounded = torch.from_numpy(p32[i][:n]).to(p.dtype)
            assert torch.equal(p.detach().cpu().reshape(-1), rounded)
            if not master:
                p32[i][:n] = rounded.float().numpy()
    first, second = (t.cpu().numpy() for t in opt.state_values())
    for i, p in enumerate(params):
        at = slice(opt.begins[i], opt.begins[i] + lengths[i])
        np.testing.assert_array_equal(first[at], m[i])
        np.testing.assert_array_equal(second[at], v[i])
        if master:
            np.testing.assert_array_equal(opt.master[at].cpu().numpy()[:p.numel()],
                                          p32[i][:p.numel()])


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_many_tensors(cuda, bits):
    gen = generator(7)
    params = [normal(gen, 1 + i % 700) for i in range(900)]
    grads = [normal(gen, *p.shape) for p in params]
    before = [p.clone() for p in params]
    opt = K.AdamW(params, **HYPER, state_bits=bits)
    opt.step(grads)
    for p, g, old in zip(params, grads, before):
        want, _, _, _ = O.adamw_f32(old.cpu().numpy(), g.cpu().numpy(), np.float32(0.0),
                                    np.float32(0.0), 1, HYPER["lr"], HYPER["betas"], HYPER["eps"],
                                    HYPER["weight_decay"])
        np.testing.assert_array_equal(p.cpu().numpy(), want)


def test_adamw_float32_step_against_the_definition(cuda):
    gen = generator(9)
    p, g = normal(gen, 5000), normal(gen, 5000)
    old = f64(p)
    opt = K.AdamW([p], **HYPER)
    opt.step([g])
    want, m, v = O.adamw(old, f64(g), 0.0, 0.0, 1, **HYPER)
    # seven roundings of terms no larger than |p| and lr
    close(p, want, 8 * U * (np.abs(old) + HYPER["lr"]))
    close(opt.exp_avg[:5000], m, 4 * U * np.abs(m))
    close(opt.exp_avg_sq[:5000], v, 4 * U * v)


def test_adamw_8bit_states_stay_within_a_rounding(cuda):
    gen = generator(11)
    g = normal(gen, 4096) * torch.exp(normal(gen, 4096))
    opt = K.AdamW([torch.zeros(4096, device="cuda")], **HYPER, state_bits=8)
    opt.step([g])
    first, second = opt.state_values()
    _, m, v = O.adamw(np.zeros(4096), f64(g), 0.0, 0.0, 1, **HYPER)
    floor = np.abs(m).reshape(-1, 256).max(1).repeat(256)
    close(first, m, (1 / 16 + 1e-6) * np.abs(m) + 2.0 ** -16 * floor)
    root = np.sqrt(v)
    floor = root.reshape(-1, 256).max(1).repeat(256)
    close(second.sqrt(), root, (1 / 32 + 1e-6) * root + 1.2 * 2.0 ** -16 * floor)
    assert (f64(second)[v > 0] > 0).all()


def test_adamw_state_dict_continues(cuda):
    gen = generator(13)
    start, grads = normal(gen, 1000, dtype=BF16), [normal(gen, 1000, dtype=BF16) for _ in range(4)]
    one, two = start.clone(), start.clone()
    a = K.AdamW([one], **HYPER, state_bits=8, master_weights=True)
    for g in grads:
        a.step([g])
    b = K.AdamW([two], **HYPER, state_bits=8, master_weights=True)
    for g in grads[:2]:
        b.step([g])
    kept = b.state_dict()
    c = K.AdamW([two], **HYPER, state_bits=8, master_weights=True)
    c.load_state_dict(kept)
    for g in grads[2:]:
        c.step([g])
    assert torch.equal(one, two) and c.step_count == 4
    with pytest.raises(ValueError):
        K.AdamW([two], state_bits=8).load_state_dict(kept)


def test_adamw_uses_parameter_gradients(cuda):
    p = torch.ones(3, device="cuda", requires_grad=True)
    q = torch.ones(3, device="cuda", requires_grad=True)
    opt = K.AdamW([p, q], lr=0.1, weight_decay=0.0)
    (p.sum() * 2.0).backward()
    opt.step()
    assert torch.allclose(p.detach(), torch.full((3,), 0.9, device="cuda"))
    assert torch.equal(q.detach(), torch.ones(3, device="cuda"))
    opt.zero_grad()
    assert p.grad is None


# ---- alignment --------------------------------------------------------------------------

def shifted(t):
    """The same values one element past an aligned address."""
    buffer = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    view = buffer[1:].view(t.shape)
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_unaligned_tensors_give_the_same(cuda, dtype):
    gen = generator(31)
    tol = half_ulp(dtype) * 2 + 64 * U
    for rows in (40, 9000):  # one CTA, and pieces joined
        x, g = normal(gen, rows, 64, dtype=dtype), normal(gen, rows, 64, dtype=dtype)
        outs = []
        for t, grad in ((x, g), (shifted(x), shifted(g))):
            t = t.detach().requires_grad_()
            y = K.group_norm(t[None], 8, activation="silu")
            outs.append((y, *torch.autograd.grad(y, [t], grad[None])))
        for a, b in zip(*outs):
            close(a, f64(b), tol * (1.0 + np.abs(f64(b))))
    x, g = normal(gen, 300, 128, dtype=dtype), normal(gen, 300, 8)
    a, b = (t.detach().requires_grad_() for t in (x, shifted(x)))
    ra, rb = K.route_experts(a, 8, renormalize=True), K.route_experts(b, 8, renormalize=True)
    assert torch.equal(ra.experts, rb.experts) and torch.equal(ra.counts, rb.counts)
    close(ra.weights, f64(rb.weights), 128 * U)
    ga, = torch.autograd.grad(ra.weights, [a], g)
    gb, = torch.autograd.grad(rb.weights, [b], g)
    close(ga, f64(gb), 128 * U * 5 + 2 * half_ulp(dtype) * np.abs(f64(gb)))
    q = normal(gen, 30, 4, 64, dtype=dtype)
    pos, freq = torch.rand(30, 3, device="cuda"), torch.rand(32, device="cuda")
    for inter in (False, True):
        one, _ = K.rotary_axes(q, q, pos, freq, (16, 8, 8), interleaved=inter)
        two, _ = K.rotary_axes(shifted(q), q, pos, freq, (16, 8, 8), interleaved=inter)
        assert torch.equal(one, two)


def test_group_norm_pieces_keep_frames_apart(cuda):
    gen = generator(37)
    x = normal(gen, 20000, 64)
    given = torch.tensor([0, 7000, 7000, 7300, 20000], device="cuda")
    first = K.group_norm(x, 8, activation="silu", offsets=given)
    assert torch.equal(first, K.group_norm(x, 8, activation="silu", offsets=given))
    x[7000:7300] = float("inf")
    other = K.group_norm(x, 8, activation="silu", offsets=given)
    assert torch.equal(other[:7000], first[:7000]) and torch.equal(other[7300:], first[7300:])


def test_adamw_step_is_an_in_place_operation(cuda):
    p = torch.ones(4, device="cuda", requires_grad=True)
    loss = (p * p).sum()
    K.AdamW([p]).step([torch.ones(4, device="cuda")])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


# ---- autograd ---------------------------------------------------------------------------

def test_gradients_are_differentiable_once(cuda):
    gen = generator(23)
    x = normal(gen, 40, 8).requires_grad_()
    q = normal(gen, 5, 2, 8).requires_grad_()
    pos, freq = torch.rand(5, 2, device="cuda"), torch.rand(4, device="cuda")
    for out, leaf in ((K.group_norm(x, 2), x), (K.route_experts(x, 2).weights, x),
                      (K.rotary_axes(q, q, pos, freq, (2, 2))[0], q)):
        grad, = torch.autograd.grad((out * out).sum(), [leaf], create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            grad.sum().backward()


def test_gradients_of_a_part_of_the_outputs(cuda):
    gen = generator(29)
    x = normal(gen, 40, 8).requires_grad_()
    offsets = np.array([0, 40])
    zero = np.zeros((40, 2))
    for pick, grads in ((lambda r: r.balance, (zero, 1.0, 0.0)), (lambda r: r.z, (zero, 0.0, 1.0)),
                        (lambda r: r.weights[:, 0].sum(), (zero + np.array([1.0, 0.0]), 0.0, 0.0))):
        got, = torch.autograd.grad(pick(K.route_experts(x, 2)), [x])
        want = O.route(f64(x), 2, None, offsets, False, grads)[5]
        close(got, want, 4 * 17 * U * 15.0)
    w = torch.ones(8, device="cuda", requires_grad=True)
    y = K.group_norm(x.detach()[None], 2, w)
    got, = torch.autograd.grad(y.sum(), [w])
    want = O.group_norm(f64(x), offsets, 2, f64(w), None, 1e-5, None, np.ones((40, 8)))[1][1]
    close(got, want, 4 * np.sqrt(40) * 16 * U * 2 * 6.0 + 2 * U * np.abs(want))
    q = normal(gen, 5, 2, 8)
    pos = torch.rand(5, 2, device="cuda").requires_grad_()
    freq = torch.rand(4, device="cuda")
    yq, _ = K.rotary_axes(q, None, pos, freq, (2, 2))
    got, = torch.autograd.grad(yq[..., ::2].sum(), [pos])
    g = np.zeros((5, 2, 8))
    g[..., ::2] = 1.0
    want = O.rotary_position_grad([f64(q)], [g], f64(pos), f64(freq), (2, 2))
    close(got, want, 16 * 16 * U * 16.0)


# ---- streams and graphs ------------------------------------------------------------------

def test_operators_run_on_the_current_stream(cuda):
    gen = generator(17)
    x, w = normal(gen, 900, 64), torch.ones(64, device="cuda")
    want = K.group_norm(x, 8, w, activation="silu", offsets=torch.tensor([0, 400, 900]).cuda())
    routed = K.route_experts(x, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    offsets = torch.tensor([0, 400, 900]).cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        y = K.group_norm(x, 8, w, activation="silu", offsets=offsets)
        r = K.route_experts(x, 2)
    side.synchronize()
    assert torch.equal(y, want) and torch.equal(r.weights, routed.weights)
    assert torch.equal(r.balance, routed.balance)


def test_a_step_is_captured_in_a_graph(cuda):
    gen = generator(19)
    x = normal(gen, 1200, 64)
    w = normal(gen, 64, 64, scale=0.1)
    offsets = torch.tensor([0, 500, 1200]).cuda()
    pos, freq = torch.rand(1200, 3, device="cuda"), torch.rand(6, device="cuda")
    opt = K.AdamW([w], lr=0.01)

    def step():
        q, k = K.rotary_axes(x.view(1200, 4, 16), x.view(1200, 4, 16), pos, freq, (2, 2, 2))
        y = K.group_norm(q.reshape(1200, 64), 8, None, None, activation="silu", offsets=offsets)
        r = K.route_experts(y @ w, 2, offsets=offsets)
        return q, k, y, r.weights, r.experts, r.balance, r.z

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        for got, expected in zip(out, want):
            assert torch.equal(got, expected)
    before = w.clone()
    opt.step([torch.ones_like(w)])
    assert not torch.equal(before, w)
