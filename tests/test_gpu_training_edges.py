"""Training-step operators where they can go wrong, on the GPU (B200).

Long runs of the optimizer, outliers and infinities, masked places that hold
anything, and launch shapes that only large or many-framed inputs take.
Tolerances are derived at each test; ``U`` and ``B`` are the unit roundoffs of
float32 and bfloat16.
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


# ---- AdamW: 8-bit states over many steps -------------------------------------------------

@pytest.mark.parametrize("before,after", [(1.0, 0.1), (1.0, 4.0), (0.05, 0.2)])
def test_adamw_8bit_second_moment_follows_at_the_default_betas(cuda, before, after):
    """sqrt(v) of 8-bit states stays near that of 32-bit states while half a block's gradients change.

    A step moves sqrt(v) by (1 - beta2) / 2 = 0.05 % of it at most (downwards), against gaps of 1/31 to
    1/16 between codes.  Rounded at random without bias, a step adds a variance of its move times the
    gap: over s steps at most s * 0.0005 / 16 to log sqrt(v) where nothing renews it (4000 steps here:
    0.35^2), 0.12^2 where gradients do.  Means over 8192 elements stay within the gap's second-order
    effect (1/32) and the skew of the logarithm (0.35^2 / 2).
    """
    gen, n = generator(41), 64 * 256
    size = torch.ones(64, 256, device="cuda")
    params = [torch.zeros(n, device="cuda") for _ in range(2)]
    byte, full = K.AdamW(params[:1], state_bits=8), K.AdamW(params[1:])
    for step in range(6000):
        if step in (0, 2000):
            size[:, 128:] = after if step else before
        g = normal(gen, 64, 256).mul_(size).view(-1)
        byte.step([g])
        full.step([g])
    ratio = (byte.state_values()[1].sqrt() / full.exp_avg_sq.sqrt()).view(64, 256).log()
    for part in (ratio[:, :128], ratio[:, 128:]):
        assert float(part.square().mean().sqrt()) < 0.35 + 0.05
        assert abs(float(part.mean())) < 0.35 ** 2 / 2 + 1 / 32
    # the first moment is exact to its codes: 1/16 a step, renewed by a tenth
    m = byte.state_values()[0] - full.exp_avg
    assert float(m.square().mean().sqrt()) < 0.1 * float(full.exp_avg.square().mean().sqrt())


def test_adamw_8bit_first_moment_decays_when_its_gradients_stop(cuda):
    """At beta1 = 0.95 a step takes 5 % off m, less than half the gap between codes 8 and 9.

    After 400 steps without a gradient m is 0.95^400 = 1.2e-9 of what it was; rounding without bias
    keeps that mean, so of 8192 elements one above 1e-3 has a probability of 1e-2.
    """
    gen, n = generator(43), 64 * 256
    opt = K.AdamW([torch.zeros(n, device="cuda")], betas=(0.95, 0.95), state_bits=8)
    g = normal(gen, 64, 256)
    for step in range(450):
        if step == 50:
            g[:, 128:] = 0.0
        opt.step([g.view(-1)])
    m = opt.state_values()[0].view(64, 256)
    assert float(m[:, 128:].abs().max()) < 1e-3
    # the others keep their constant gradient: within a gap of it
    close(m[:, :128], f64(g[:, :128]), f64(g[:, :128].abs()) / 8 + 2.0 ** -16 * 5)


@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.95, 0.95), (0.97, 0.9999)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_adamw_8bit_random_rounding_bit_for_bit(cuda, betas, dtype):
    gen, sizes = generator(47), [(700,), (1,), (3, 256), (0,), (31, 33)]
    hyper = dict(lr=0.01, betas=betas, eps=1e-8, weight_decay=0.1)
    params = [normal(gen, *s, dtype=dtype) for s in sizes]
    opt = K.AdamW(params, **hyper, state_bits=8, master_weights=dtype == BF16)
    length = opt.exp_avg.numel()

    def packed(tensors):
        out = np.zeros(length, np.float32)
        for t, begin in zip(tensors, opt.begins):
            out[begin:begin + t.numel()] = t.detach().float().cpu().numpy().reshape(-1)
        return out

    p, m, v = packed(params), np.zeros(length, np.float32), np.zeros(length, np.float32)
    for step in range(1, 5):
        grads = [normal(gen, *s, dtype=dtype) for s in sizes]
        if step == 2:
            for g in grads:
                g.mul_(torch.exp(normal(gen, *g.shape, scale=5.0)).to(dtype))
                g[..., ::3] = 0.0
        opt.step(grads)
        p, m, v, root = O.adamw_f32(p, packed(grads), m, v, step, **hyper)
        noise_m, noise_v = O.rounding_noise(step, length, betas)
        whole = m.reshape(-1, O.BLOCK)
        code, scale = O.encode(np.abs(whole), 127, O.VALUES_M, noise_m)
        np.testing.assert_array_equal(
            opt.exp_avg.cpu().numpy(),
            np.where(whole < 0, code + 128, code).astype(np.uint8).reshape(-1))
        m = (np.where(whole < 0, -1, 1) * O.decode(code, scale, O.VALUES_M)).astype(
            np.float32).reshape(-1)
        code, scale = O.encode(root.reshape(-1, O.BLOCK), 255, O.VALUES_V, noise_v)
        np.testing.assert_array_equal(opt.exp_avg_sq.cpu().numpy(), code.reshape(-1))
        v = O.decode(code, scale, O.VALUES_V).reshape(-1) ** 2
        for t, begin in zip(params, opt.begins):
            part = torch.from_numpy(p[begin:begin + t.numel()])
            assert torch.equal(t.cpu().reshape(-1), part.to(dtype))


def test_adamw_8bit_random_rounding_repeats_and_resumes(cuda):
    gen = generator(53)
    start, grads = normal(gen, 1000), [normal(gen, 1000) for _ in range(6)]
    one, two = start.clone(), start.clone()
    a = K.AdamW([one], state_bits=8)
    for g in grads:
        a.step([g])
    b = K.AdamW([two], state_bits=8)
    for g in grads[:3]:
        b.step([g])
    c = K.AdamW([two], state_bits=8)
    c.load_state_dict(b.state_dict())
    for g in grads[3:]:
        c.step([g])
    assert torch.equal(one, two) and torch.equal(a.exp_avg_sq, c.exp_avg_sq)


# ---- AdamW: what a step is given -----------------------------------------------------------

def test_adamw_zero_stays_zero_beside_tiny_values(cuda):
    # the inverse of a scale below 2^-128 is infinite: its product with 0 must not become a code
    p = torch.zeros(300, device="cuda")
    g = torch.zeros(300, device="cuda")
    g[:100], g[100:200] = 1e-39, -1e-39
    opt = K.AdamW([p], state_bits=8, betas=(0.9, 0.95))
    opt.step([g])
    m = opt.state_values()[0]
    assert float(m[:256].abs().max()) > 0.0  # the block holds something
    assert (opt.exp_avg[200:] == 0).all() and (m[200:] == 0.0).all()


def test_adamw_gradient_of_another_shape_is_refused(cuda):
    p = torch.ones(3, 4, device="cuda")
    opt = K.AdamW([p])
    for shape in ((4, 3), (12,), (3, 4, 1)):
        with pytest.raises(RuntimeError, match="shape"):
            opt.step([torch.ones(shape, device="cuda")])
    assert opt.step_count == 0 and torch.equal(p, torch.ones_like(p))


def test_adamw_parameter_that_changed_its_size_is_refused(cuda):
    p, q = torch.ones(4, device="cuda"), torch.ones(300, device="cuda")
    opt = K.AdamW([p, q])
    p.data = torch.ones(400, device="cuda")  # its states would reach into those of q
    with pytest.raises(RuntimeError, match="shape"):
        opt.step([torch.ones(400, device="cuda"), None])


def test_adamw_params_cannot_be_replaced_behind_its_back(cuda):
    p = torch.ones(4, device="cuda")
    opt = K.AdamW([p])
    with pytest.raises(TypeError):
        opt.params[0] = torch.zeros(4, device="cuda")
    with pytest.raises(AttributeError):
        opt.params = [torch.zeros(4, device="cuda")]
    assert opt.params[0] is p


@pytest.mark.parametrize("change,error", [(dict(step=None), TypeError), (dict(exp_avg_sq=[0.0]), ValueError),
                                          (dict(exp_avg_sq=torch.zeros(3)), ValueError),
                                          (dict(master=torch.zeros(256)), ValueError)])
def test_adamw_state_that_does_not_fit_changes_nothing(cuda, change, error):
    p = torch.ones(4, device="cuda")
    opt, other = K.AdamW([p]), K.AdamW([p.clone()])
    other.step([torch.ones(4, device="cuda")])
    with pytest.raises(error):
        opt.load_state_dict({**other.state_dict(), **change})
    assert opt.step_count == 0 and float(opt.exp_avg.abs().max()) == 0.0


def test_adamw_step_is_not_captured(cuda):
    # the bias corrections and the step count are values of the call: a replay would repeat them
    p, g = torch.ones(4, device="cuda"), torch.ones(4, device="cuda")
    opt = K.AdamW([p])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = p + 1.0
        with pytest.raises(RuntimeError, match="captur"):
            opt.step([g])
    graph.replay()
    torch.cuda.synchronize()
    assert opt.step_count == 0 and torch.equal(p, torch.ones_like(p)) and float(y[0]) == 2.0
    opt.step([g])
    assert opt.step_count == 1


def test_adamw_inference_tensor_is_refused_before_the_step(cuda):
    with torch.inference_mode():
        p = torch.ones(4, device="cuda")
    opt = K.AdamW([p])
    with pytest.raises(RuntimeError, match="inference"):
        opt.step([torch.ones(4, device="cuda")])
    assert torch.equal(p.cpu(), torch.ones(4)) and float(opt.exp_avg.abs().max()) == 0.0
    with torch.inference_mode():
        opt.step([torch.ones(4, device="cuda")])
    assert opt.step_count == 1


# ---- derivatives other than backward ---------------------------------------------------------

def operator_calls(gen):
    x = normal(gen, 40, 8)
    q, pos, freq = normal(gen, 5, 2, 8), torch.rand(5, 2, device="cuda"), torch.rand(4, device="cuda")
    w = torch.ones(8, device="cuda")
    return [
        (lambda t: K.group_norm(t, 2, w), x),
        (lambda t: K.group_norm(x, 2, t, t), w),
        (lambda t: K.route_experts(t, 2).weights, x),
        (lambda t: K.rotary_axes(t, q, pos, freq, (2, 2))[0], q),
        (lambda t: K.rotary_axes(q, t, pos, freq, (2, 2))[1], q),
        (lambda t: K.rotary_axes(q, None, t, freq, (2, 2))[0], pos),
        (lambda t: K.rotary_axes(q, None, pos, t, (2, 2))[0], freq),
    ]


@pytest.mark.parametrize("grad_enabled", [True, False])
def test_forward_mode_derivatives_are_refused(cuda, grad_enabled):
    import torch.autograd.forward_ad as fwd

    for call, x in operator_calls(generator(59)):
        with fwd.dual_level(), torch.set_grad_enabled(grad_enabled):
            dual = fwd.make_dual(x, torch.ones_like(x))
            with pytest.raises(RuntimeError, match="jvp|forward-mode"):
                call(dual)


def test_function_transforms_are_refused(cuda):
    for call, x in operator_calls(generator(61)):
        for transform in (lambda f: torch.func.vmap(f)(x[None]),
                          lambda f: torch.func.jvp(f, (x,), (torch.ones_like(x),)),
                          lambda f: torch.func.grad(lambda t: f(t).sum())(x)):
            with pytest.raises(RuntimeError):
                transform(call)


# ---- group norm: outliers, infinities, launch shapes -------------------------------------------

def chunk_rows(rows, row_bytes):
    """Rows of a forward statistics chunk: one for each of four resident CTAs an SM, of 16 KB at least."""
    ctas = torch.cuda.get_device_properties(0).multi_processor_count * 4
    return max(-(-rows // ctas), -(-16384 // row_bytes))
# rows, channels, groups, lengths, where -> value, dtype
OUTLIERS = {
    "first row": (200000, 160, 1, None, [(0, 0, 3000.0)], F32),
    "first row, few channels": (196608, 4, 1, None, [(0, None, 1000.0)], F32),
    "first rows of every frame": (98304, 8, 2, [1000, 40000, 57304], [(0, None, 300.0)], F32),
    "group's first channel": (20000, 1024, 1, None, [(None, 0, 1000.0)], F32),
    "group's last channel": (20000, 64, 4, None, [(None, 63, 1000.0)], F32),
    "small frame": (4000, 4, 1, None, [(0, None, 3000.0)], F32),
    "bfloat16": (100000, 64, 8, None, [(0, None, 1024.0)], BF16),
}


@pytest.mark.parametrize("name", OUTLIERS)
def test_group_norm_variance_beside_outliers(cuda, name):
    rows, channels, groups, lengths, places, dtype = OUTLIERS[name]
    gen = generator(rows)
    x = normal(gen, rows, channels)
    offsets = np.concatenate([[0], np.cumsum([rows] if lengths is None else lengths)])
    for row, channel, value in places:
        at = slice(None) if channel is None else channel
        if row is None:
            x[:, at] += value
        else:
            x[torch.from_numpy(offsets[:-1] + row).cuda(), at] = value
    x = x.to(dtype)
    check_norm(x, groups, offsets, dtype)


@pytest.mark.parametrize("before", [1, 2, 5])
def test_group_norm_variance_of_a_frame_that_begins_at_the_end_of_a_chunk(cuda, before):
    rows, channels = 200000, 8
    edge = 40 * chunk_rows(rows, channels * 4)
    offsets = np.array([0, edge - before, rows])
    x = normal(generator(before), rows, channels)
    x[edge - before] = 1000.0
    check_norm(x, 2, offsets, F32)


def check_norm(x, groups, offsets, dtype):
    """z = (x - mean) rstd beside the float64 definition.

    mean: the weighted mean of partial means, each within a few units of the values' size, rstd: sums of
    squares about means, 64 terms and a few levels of joining: 96 units relative.  z itself is one
    multiply-add, whose constant has the mean's rounding.
    """
    channels = x.shape[-1]
    y = K.group_norm(x, groups, offsets=torch.from_numpy(offsets).cuda())
    flat = x.double()
    for a, b in zip(offsets[:-1], offsets[1:]):
        v = flat[a:b].reshape(b - a, groups, -1)
        mean = v.mean((0, 2), keepdim=True)
        rstd = 1.0 / torch.sqrt((v - mean).square().mean((0, 2), keepdim=True) + 1e-5)
        z = (v - mean) * rstd
        size = 1.0 + v.abs() * rstd + v.abs().mean((0, 2), keepdim=True) * rstd
        tol = 96 * U * (size + z.abs()) + (B if dtype == BF16 else 0.0) * z.abs()
        off = (y[a:b].double().reshape(v.shape) - z).abs() - tol
        assert float(off.max()) <= 0.0, f"off by {float(off.max())} beyond the tolerance"


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("rows", [40, 9000])
@pytest.mark.parametrize("activation", [None, "sigmoid", "silu"])
def test_group_norm_infinities_show(cuda, value, rows, activation):
    # a frame and group that hold one have no mean: all of it is NaN, nothing else is touched
    x = normal(generator(67), 3 * rows, 16)
    offsets = torch.tensor([0, rows, 2 * rows, 3 * rows], device="cuda")
    whole = K.group_norm(x, 4, activation=activation, offsets=offsets)
    for place in (rows, rows + rows // 2, 2 * rows - 1):
        bad = x.clone()
        bad[place, 5] = value
        y = K.group_norm(bad, 4, activation=activation, offsets=offsets)
        assert torch.isnan(y[rows:2 * rows, 4:8]).all()
        y[rows:2 * rows, 4:8] = whole[rows:2 * rows, 4:8]
        assert torch.equal(y, whole)


@pytest.mark.parametrize("frames", [200, 2000])
@pytest.mark.parametrize("dtype,channels", [(F32, 24), (BF16, 64), (F32, 7)])
def test_group_norm_many_small_frames(cuda, frames, dtype, channels):
    """More frames than CTAs are launched: a CTA walks over several and adds up their affine gradients.

    Values as in the one-frame tests (z within 16 units of its size and the mean's); an affine gradient
    sums n terms of either sign with that error, over a few hundred rows a CTA and the CTAs in order.
    """
    gen, rng = generator(frames), np.random.default_rng(frames)
    lengths = rng.integers(0, 12, frames)
    lengths[:3] = 0, 1, 0
    offsets = np.concatenate([[0], np.cumsum(lengths)])
    rows, groups = int(offsets[-1]), 1 if channels == 7 else 4
    x, grad = normal(gen, rows, channels, dtype=dtype), normal(gen, rows, channels, dtype=dtype)
    w, b = torch.rand(channels, generator=gen, device="cuda") + 0.5, normal(gen, channels, scale=0.3)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = K.group_norm(x, groups, w, b, activation="silu", offsets=torch.from_numpy(offsets).cuda())
    grads = torch.autograd.grad(y, leaves, grad)
    want, (gx, gw, gb) = O.group_norm(f64(x), offsets, groups, f64(w), f64(b), 1e-5, "silu", f64(grad))
    half = B if dtype == BF16 else 0.0
    # a frame of six values and more: 1 / std below 20 for these
    v = [f64(x)[i:j].reshape(j - i, groups, -1) for i, j in zip(offsets[:-1], offsets[1:]) if j > i]
    rstd = max(1.0 / np.sqrt(t.var((0, 2)) + 1e-5).min() for t in v)
    off = 16 * U * (2.0 + rstd)
    xhat = max(2.0, np.sqrt(12.0 * channels / groups))
    close(y, want, off * 1.5 * xhat + half * np.abs(want))
    d = np.abs(f64(grad)).max() * 1.1 * 1.5
    close(grads[0], gx, rstd * off * d * (2.0 + 2.0 * xhat * xhat) * 1.5 + half * np.abs(gx))
    for got, ref in ((grads[1], gw), (grads[2], gb)):
        close(got, ref, 4 * np.sqrt(rows) * off * d * xhat * 1.5 + 4 * U * np.sqrt(rows) * np.abs(ref))


def test_group_norm_one_large_frame_among_small_ones(cuda):
    gen = generator(71)
    lengths = np.full(400, 3)
    lengths[200] = 30000
    offsets = np.concatenate([[0], np.cumsum(lengths)])
    check_norm(normal(gen, int(offsets[-1]), 16), 2, offsets, F32)


# ---- router: masked places, launch shapes ---------------------------------------------------------

@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("dtype,experts,k", [(F32, 8, 2), (BF16, 64, 4), (F32, 33, 12)])
def test_router_cotangents_of_masked_tokens_and_empty_slots_have_no_effect(cuda, renormalize, dtype,
                                                                          experts, k):
    gen, nan = generator(73), float("nan")
    x = normal(gen, 50, experts)
    x[10:20, 1:] = float("-inf")   # one expert each, the other slots empty
    x[20:25] = float("-inf")       # none at all
    x = x.to(dtype).requires_grad_()
    mask = torch.ones(50, dtype=torch.bool, device="cuda")
    mask[30:40] = False
    r = K.route_experts(x, k, mask=mask, renormalize=renormalize)
    cotangents = [normal(gen, 50, k), torch.tensor(0.7, device="cuda"), torch.tensor(0.1, device="cuda")]
    want, = torch.autograd.grad([r.weights, r.balance, r.z], [x], cotangents, retain_graph=True)
    empty = r.experts < 0
    for value in (nan, float("inf")):
        spoiled = [cotangents[0].masked_fill(empty, value), *cotangents[1:]]
        got, = torch.autograd.grad([r.weights, r.balance, r.z], [x], spoiled, retain_graph=True)
        assert torch.equal(got, want)
    # a loss that is lost leaves the tokens alone that were left out of it
    spoiled = [cotangents[0], torch.tensor(nan, device="cuda"), torch.tensor(nan, device="cuda")]
    got, = torch.autograd.grad([r.weights, r.balance, r.z], [x], spoiled)
    out = ~mask
    out[20:25] = True
    assert (got[out] == 0.0).all() and torch.isnan(got[~out]).any(1).all()


def check_route(x, k, lengths, mask, renormalize, seed):
    """Against the float64 definition, with the bounds of the other router tests."""
    tokens, experts = x.shape
    gen = generator(seed)
    offsets = None if lengths is None else np.concatenate([[0], np.cumsum(lengths)])
    given = None if offsets is None else torch.from_numpy(offsets).cuda()
    grads = (normal(gen, tokens, k), torch.tensor(0.7 * tokens, device="cuda"),
             torch.tensor(0.1 * tokens, device="cuda"))
    x = x.clone().requires_grad_()
    r = K.route_experts(x, k, mask=mask, offsets=given, renormalize=renormalize)
    grad, = torch.autograd.grad([r.weights, r.balance, r.z], [x], list(grads))
    want = O.route(f64(x), k, None if mask is None else mask.cpu().numpy(), offsets, renormalize,
                   (f64(grads[0]), float(grads[1]), float(grads[2])))
    np.testing.assert_array_equal(r.experts.cpu().numpy(), want[1])
    counts = r.counts.cpu().numpy()
    np.testing.assert_array_equal(counts if offsets is not None else counts[None], want[2])
    rel = (16 + experts / 8) * U
    close(r.weights, want[0], 2 * rel * want[0])
    close(r.balance.reshape(1), np.array([want[3]]), rel * abs(want[3]) + 1e-9)
    top = np.abs(f64(x)[np.isfinite(f64(x))]).max() + np.log(experts)
    close(r.z.reshape(1), np.array([want[4]]), rel * top * 2.0 * np.sqrt(want[4]) + U * want[4])
    valid = (want[1][:, 0] >= 0).astype(np.int64)
    edges = np.array([0, tokens]) if offsets is None else offsets
    n = np.maximum([valid[a:b].sum() for a, b in zip(edges[:-1], edges[1:])], 1)
    scale = np.abs(f64(grads[0])).max() + \
        float(grads[1]) * (experts / k * want[2].max(1) / n ** 2).max() + \
        float(grads[2]) * 2.0 / max(valid.sum(), 1) * (top + 5.0)
    half = B if x.dtype == BF16 else 0.0
    close(grad, want[5], 4 * rel * scale + half * np.abs(want[5]))


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("experts,k", [(512, 8), (1024, 8), (1024, 3), (264, 5), (24, 4), (32, 3),
                                       (20, 7), (28, 1), (8, 8), (256, 2)])
def test_router_launch_shapes(cuda, experts, k, dtype, ties):
    x = normal(generator(experts + k), 90, experts, scale=2.0)
    check_route((torch.round(x) if ties else x).to(dtype), k, None, None, True, 79)


@pytest.mark.parametrize("frames,experts", [(100, 256), (300, 64), (2000, 16)])
def test_router_losses_of_many_frames(cuda, frames, experts):
    # more cells than the forward kernel's last CTA takes: a kernel of several CTAs joins the losses
    rng = np.random.default_rng(frames)
    lengths = rng.integers(0, 7, frames)
    tokens = int(lengths.sum())
    gen = generator(frames)
    x = normal(gen, tokens, experts, scale=1.5)
    mask = torch.rand(tokens, generator=gen, device="cuda") < 0.8
    check_route(x, 2, lengths, mask, False, 83)


# ---- rotary: long positions -----------------------------------------------------------------------

def test_rotary_long_positions(cuda):
    """Angles of thousands of turns: the float32 product is off by a unit roundoff of the angle."""
    gen = generator(89)
    q = normal(gen, 50, 2, 16)
    pos = torch.randint(0, 1 << 17, (50, 2), generator=gen, device="cuda")
    freq = torch.rand(8, generator=gen, device="cuda") + 0.05
    y, _ = K.rotary_axes(q, None, pos, freq, (4, 4))
    want = O.rotary(f64(q), f64(pos), f64(freq), (4, 4))
    theta = float(pos.max()) * float(freq.max())
    close(y, want, (U * theta + 8 * U) * 2.0 * float(q.abs().max()))


# ---- graphs and threads ----------------------------------------------------------------------------

def test_forward_and_backward_are_captured(cuda):
    gen = generator(97)
    x = normal(gen, 1200, 64).requires_grad_()
    pos = torch.rand(1200, 3, device="cuda").requires_grad_()
    offsets, freq = torch.tensor([0, 500, 1200]).cuda(), torch.rand(6, device="cuda")
    g = normal(gen, 1200, 64)

    def step():
        q, k = K.rotary_axes(x.view(1200, 4, 16), x.view(1200, 4, 16), pos, freq, (2, 2, 2))
        y = K.group_norm((q + k).reshape(1200, 64), 8, activation="silu", offsets=offsets)
        r = K.route_experts(y, 4, offsets=offsets, renormalize=True)
        loss = (y * g).sum() + (r.weights * g[:, :4]).sum() + r.balance + r.z
        return (loss.detach(), *torch.autograd.grad(loss, [x, pos]))

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


def test_operators_called_from_two_threads(cuda):
    from concurrent.futures import ThreadPoolExecutor

    gen = generator(101)
    inputs = [normal(gen, 3000, 64) for _ in range(2)]

    def work(x):
        with torch.cuda.stream(torch.cuda.Stream()):
            out = []
            for _ in range(20):
                t = x.clone().requires_grad_()
                y = K.group_norm(t, 8, activation="silu",
                                 offsets=torch.tensor([0, 1000, 3000], device="cuda"))
                r = K.route_experts(y, 4, renormalize=True)
                out.append((y, r.weights, *torch.autograd.grad(r.weights.sum() + r.z + y.sum(), [t])))
            torch.cuda.current_stream().synchronize()
            return out

    torch.cuda.synchronize()
    want = [work(x)[0] for x in inputs]
    with ThreadPoolExecutor(2) as pool:
        results = list(pool.map(work, inputs))
    for outs, first in zip(results, want):
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, first))
