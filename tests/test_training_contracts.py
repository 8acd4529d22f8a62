"""Host-side contracts of the training-step operators, and their oracle (no GPU)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import bysj_b200.kernels as K
from oracle import training as O

NO_GPU = pytest.mark.skipif(torch.cuda.is_available(), reason="guard behaviour on a CPU host")


def rotary_args(**change):
    args = dict(q=torch.zeros(4, 2, 8), k=torch.zeros(4, 1, 8), positions=torch.zeros(4, 2),
                inv_freq=torch.zeros(4), sections=(2, 2))
    args.update(change)
    return args


@pytest.mark.parametrize("change,error", [
    (dict(q=[1.0]), TypeError),
    (dict(q=torch.zeros(4, 2, 8).double()), TypeError),
    (dict(q=torch.zeros(4, 8)), ValueError),
    (dict(k=torch.zeros(4, 1, 8).bfloat16()), TypeError),
    (dict(k=torch.zeros(3, 1, 8)), ValueError),
    (dict(k=torch.zeros(4, 1, 6)), ValueError),
    (dict(q=torch.zeros(4, 8, 2).transpose(1, 2)), ValueError),
    (dict(positions=torch.zeros(4, 2).double()), TypeError),
    (dict(positions=torch.zeros(4, 3)), ValueError),
    (dict(positions=torch.zeros(2, 4).t()), ValueError),
    (dict(inv_freq=torch.zeros(5)), ValueError),
    (dict(inv_freq=torch.zeros(4).double()), TypeError),
    (dict(inv_freq=torch.zeros(4, requires_grad=True)), RuntimeError),
    (dict(sections=(2, 3), inv_freq=torch.zeros(5)), ValueError),
    (dict(sections=(-1, 5)), ValueError),
    (dict(sections=(1,) * 5, positions=torch.zeros(4, 5), inv_freq=torch.zeros(5)), ValueError),
    (dict(sections=()), ValueError),
    (dict(sections="ab"), ValueError),
])
def test_rotary_refuses(change, error):
    with pytest.raises(error):
        K.rotary_axes(**rotary_args(**change))


@pytest.mark.parametrize("args,kwargs,error", [
    (([1.0], 2), {}, TypeError),
    ((torch.zeros(4, 8).half(), 2), {}, TypeError),
    ((torch.zeros(8), 2), {}, ValueError),
    ((torch.zeros(4, 8), 3), {}, ValueError),
    ((torch.zeros(4, 8), 0), {}, ValueError),
    ((torch.zeros(4, 8), 2.0), {}, TypeError),
    ((torch.zeros(4, 8), True), {}, TypeError),
    ((torch.zeros(8, 4).t(), 2), {}, ValueError),
    ((torch.zeros(4, 8), 2, torch.zeros(7)), {}, ValueError),
    ((torch.zeros(4, 8), 2, torch.zeros(8).bfloat16()), {}, TypeError),
    ((torch.zeros(4, 8), 2, None, torch.zeros(8, 1)), {}, ValueError),
    ((torch.zeros(4, 8), 2, None, None, 0.0), {}, ValueError),
    ((torch.zeros(4, 8), 2, None, None, float("nan")), {}, ValueError),
    ((torch.zeros(4, 8), 2, None, None, "x"), {}, ValueError),
    ((torch.zeros(4, 8), 2), dict(activation="relu"), ValueError),
    ((torch.zeros(4, 8), 2), dict(offsets=torch.zeros(3)), TypeError),
    ((torch.zeros(4, 8), 2), dict(offsets=torch.zeros(1, dtype=torch.int64)), ValueError),
    ((torch.zeros(4, 8), 2), dict(offsets=torch.zeros(2, 2, dtype=torch.int64)), ValueError),
])
def test_group_norm_refuses(args, kwargs, error):
    with pytest.raises(error):
        K.group_norm(*args, **kwargs)


@pytest.mark.parametrize("args,kwargs,error", [
    (([1.0], 1), {}, TypeError),
    ((torch.zeros(4, 8).double(), 1), {}, TypeError),
    ((torch.zeros(4, 8, 1), 1), {}, ValueError),
    ((torch.zeros(4, 0), 1), {}, ValueError),
    ((torch.zeros(4, 1025), 1), {}, ValueError),
    ((torch.zeros(4, 8), 0), {}, ValueError),
    ((torch.zeros(4, 8), 9), {}, ValueError),
    ((torch.zeros(4, 64), 33), {}, ValueError),
    ((torch.zeros(4, 8), 1.0), {}, TypeError),
    ((torch.zeros(8, 4).t(), 1), {}, ValueError),
    ((torch.zeros(4, 8), 1), dict(mask=torch.zeros(4)), TypeError),
    ((torch.zeros(4, 8), 1), dict(mask=torch.zeros(5, dtype=torch.bool)), ValueError),
    ((torch.zeros(4, 8), 1), dict(offsets=torch.zeros(2)), TypeError),
    ((torch.zeros(4, 8), 1), dict(offsets=torch.zeros(1, dtype=torch.int64)), ValueError),
])
def test_router_refuses(args, kwargs, error):
    with pytest.raises(error):
        K.route_experts(*args, **kwargs)


@pytest.mark.parametrize("params,kwargs,error", [
    ([], {}, ValueError),
    ([1.0], {}, TypeError),
    ([torch.zeros(3).double()], {}, TypeError),
    ([torch.zeros(3, 4).t()], {}, ValueError),
    ([torch.zeros(3)], dict(state_bits=16), ValueError),
    ([torch.zeros(3)], dict(lr=-1.0), ValueError),
    ([torch.zeros(3)], dict(lr=float("inf")), ValueError),
    ([torch.zeros(3)], dict(eps=0.0), ValueError),
    ([torch.zeros(3)], dict(weight_decay=-0.1), ValueError),
    ([torch.zeros(3)], dict(betas=(0.9,)), ValueError),
    ([torch.zeros(3)], dict(betas=(0.9, 1.0)), ValueError),
])
def test_adamw_refuses(params, kwargs, error):
    with pytest.raises(error):
        K.AdamW(params, **kwargs)


def test_adamw_refuses_the_same_tensor_twice():
    p = torch.zeros(3)
    with pytest.raises(ValueError):
        K.AdamW([p, p])


@NO_GPU
def test_operators_stop_at_the_device_guard():
    calls = [
        lambda: K.rotary_axes(**rotary_args()),
        lambda: K.rotary_axes(**rotary_args(k=None)),
        lambda: K.group_norm(torch.zeros(4, 8), 2),
        lambda: K.route_experts(torch.zeros(4, 8), 2),
        lambda: K.AdamW([torch.zeros(3)]),
    ]
    for call in calls:
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


# ---- the oracle's gradients against differences ----------------------------------------

def difference(value, h=1.0e-6):
    return (value(h) - value(-h)) / (2 * h)


def test_oracle_rotary_gradients():
    rng = np.random.default_rng(0)
    x, g, pos = rng.normal(size=(5, 2, 9)), rng.normal(size=(5, 2, 9)), rng.normal(size=(5, 2))
    freq, sections = rng.random(4), (1, 3)
    dx, dpos = rng.normal(size=x.shape), rng.normal(size=pos.shape)
    for inter in (False, True):
        def value(h):
            return (O.rotary(x + h * dx, pos + h * dpos, freq, sections, inter) * g).sum()

        got = (O.rotary(g, pos, freq, sections, inter, inverse=True) * dx).sum() + \
            (O.rotary_position_grad([x], [g], pos, freq, sections, inter) * dpos).sum()
        assert abs(got - difference(value)) < 1e-7


@pytest.mark.parametrize("act", [None, "silu", "sigmoid"])
def test_oracle_group_norm_gradients(act):
    rng = np.random.default_rng(1)
    x, g, w, b = (rng.normal(size=s) for s in ((9, 6), (9, 6), (6,), (6,)))
    dx, dw, db = (rng.normal(size=t.shape) for t in (x, w, b))
    offsets = [0, 4, 4, 9]

    def value(h):
        return (O.group_norm(x + h * dx, offsets, 3, w + h * dw, b + h * db, 1e-3, act)[0] * g).sum()

    gx, gw, gb = O.group_norm(x, offsets, 3, w, b, 1e-3, act, g)[1]
    assert abs((gx * dx).sum() + (gw * dw).sum() + (gb * db).sum() - difference(value)) < 1e-6


@pytest.mark.parametrize("renormalize", [False, True])
def test_oracle_router_gradient(renormalize):
    rng = np.random.default_rng(2)
    x, gw, dx = rng.normal(size=(8, 5)), rng.normal(size=(8, 2)), rng.normal(size=(8, 5))
    mask, offsets = np.array([1, 1, 0, 1, 1, 1, 1, 0], bool), [0, 3, 3, 8]

    def value(h):
        w, _, _, balance, z, _ = O.route(x + h * dx, 2, mask, offsets, renormalize)
        return (w * gw).sum() + 0.7 * balance + 0.3 * z

    grad = O.route(x, 2, mask, offsets, renormalize, (gw, 0.7, 0.3))[5]
    assert abs((grad * dx).sum() - difference(value)) < 1e-7


def test_oracle_codes():
    for top, values in ((127, O.VALUES_M), (255, O.VALUES_V)):
        assert values[top] == 1.0 and values[0] == 0.0 and (np.diff(values) > 0).all()
        block = np.tile(values.astype(np.float32), 2)[:O.BLOCK][None].copy()
        block[0, -1] = 1.0
        code, scale = O.encode(block, top, values)
        assert scale[0] == 1.0
        np.testing.assert_array_equal(values[code[0]], block[0])
    # ties to the even mantissa, zero only for zero in the root's code
    block = np.zeros((1, O.BLOCK), np.float32)
    block[0, :3] = 1.0, 0.5 * (O.VALUES_V[254] + O.VALUES_V[253]), 1e-12
    code, _ = O.encode(block, 255, O.VALUES_V)
    assert code[0, :4].tolist() == [255, 253, 1, 0]
