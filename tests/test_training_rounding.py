"""Rounding of the optimizer's 8-bit states in the oracle: the generator, the mean and a long run (no GPU)."""
from __future__ import annotations

import ctypes
from pathlib import Path

import numpy as np
import pytest

from oracle import training as O

LIB = Path(__file__).resolve().parents[1] / "bysj_b200" / "libbysj_b200.so"


def test_generator_gives_the_published_words():
    # the known answers of ten rounds
    zero = O.philox4x32(np.zeros((1, 4), np.uint64), 0, 10)[0]
    assert [hex(int(w)) for w in zero] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
    ones = O.philox4x32(np.full((1, 4), 0xFFFFFFFF, np.uint64), (1 << 64) - 1, 10)[0]
    assert [hex(int(w)) for w in ones] == ["0x408f276d", "0x41c83b0e", "0xa20bc7c6", "0x6d5451fd"]


def test_noise_is_uniform_and_differs_from_step_to_step():
    a, b = O.rounding_noise(5, 1 << 18, (0.95, 0.999))
    c, _ = O.rounding_noise(6, 1 << 18, (0.95, 0.999))
    for n in (a, b):
        assert n.shape == (1 << 10, O.BLOCK) and n.min() > 0.0 and n.max() < 1.0
        # mean 1/2 within 5 standard deviations of 1 / sqrt(12 n)
        assert abs(n.mean() - 0.5) < 5.0 / np.sqrt(12.0 * n.size)
    for x, y in ((a, b), (a, c)):
        assert abs(np.corrcoef(x.ravel(), y.ravel())[0, 1]) < 5.0 / np.sqrt(x.size)
    assert O.rounding_noise(5, 256, (0.9, 0.95)) == [None, None]
    assert O.rounding_noise(5, 256, (0.9, 0.999))[0] is None


@pytest.mark.parametrize("top,values", [(127, O.VALUES_M), (255, O.VALUES_V)])
def test_random_rounding_keeps_the_mean(top, values):
    rng = np.random.default_rng(0)
    x = np.exp(rng.uniform(-9.0, 0.0, O.BLOCK)).astype(np.float32)
    x[0] = 1.0
    if top == 127:
        x[1:20] = rng.random(19).astype(np.float32) * 2.0 ** -16  # below the smallest code's value
    rounds = 4000
    code, scale = O.encode(np.tile(x, (rounds, 1)), top, values, rng.random((rounds, O.BLOCK)))
    got = O.decode(code, scale, values)
    assert (got[:, 0] == 1.0).all()
    gap = np.maximum(x / 8.0, values[1])
    # within 5 standard deviations (at most half a gap) of the mean
    assert (np.abs(got.mean(0) - x) <= 5.0 * 0.5 * gap / np.sqrt(rounds)).all()


def test_zero_and_padding_stay_zero():
    x = np.zeros((2, O.BLOCK), np.float32)
    x[0, :3] = 1.0, 1e-12, 0.0
    noise = np.full(x.shape, 1.0 - 2.0 ** -17)
    for top, values in ((127, O.VALUES_M), (255, O.VALUES_V)):
        code, scale = O.encode(x, top, values, noise)
        assert (code[0, 2:] == 0).all() and (code[1] == 0).all() and scale.tolist() == [1.0, 0.0]
        assert code[0, 1] == (1 if top == 255 else 0)


@pytest.mark.parametrize("factor", [0.1, 4.0])
def test_second_moment_follows_over_a_long_run(factor):
    """Two blocks at beta2 = 0.999, half of each with other gradients from step 1500 on.

    Random rounding adds at most 0.0005 / 16 a step to the variance of log sqrt(v): 0.31^2 over the
    3000 steps after the change; means as in the GPU test of the same name.
    """
    rng, betas = np.random.default_rng(1), (0.9, 0.999)
    m = v = np.zeros(2 * O.BLOCK, np.float32)
    exact, zero = np.zeros(2 * O.BLOCK), np.zeros(2 * O.BLOCK, np.float32)
    size = np.ones((2, O.BLOCK))
    for step in range(1, 4501):
        if step == 1500:
            size[:, 128:] = factor
        g = (rng.standard_normal(size.shape) * size).astype(np.float32).ravel()
        exact = betas[1] * exact + (1.0 - betas[1]) * g.astype(np.float64) ** 2
        _, _, v, root = O.adamw_f32(zero, g, m, v, step, 0.0, betas, 1e-8, 0.0)
        noise = O.rounding_noise(step, v.size, betas)[1]
        code, scale = O.encode(root.reshape(-1, O.BLOCK), 255, O.VALUES_V, noise)
        v = O.decode(code, scale, O.VALUES_V).ravel() ** 2
    ratio = 0.5 * np.log(v / exact).reshape(2, O.BLOCK)
    for part in (ratio[:, :128], ratio[:, 128:]):
        assert np.sqrt((part ** 2).mean()) < 0.31 + 0.05
        assert abs(part.mean()) < 0.31 ** 2 / 2 + 1 / 32 + 5 * 0.31 / 16


def test_c_entry_without_a_counter_refuses_slow_moments():
    if not LIB.exists():
        pytest.skip("library not built")
    lib = ctypes.CDLL(str(LIB))
    lib.bysj_last_error.restype = ctypes.c_char_p
    pointer, i64 = ctypes.c_void_p, ctypes.c_int64
    lib.bysj_adamw_step.argtypes = [pointer, i64, ctypes.c_int, ctypes.c_int] + [pointer] * 8
    here = ctypes.create_string_buffer(64)  # stands for the device pointers: a refusal reads none
    at = ctypes.cast(here, ctypes.c_void_p)
    table = (i64 * 4)(at.value, at.value, 16, 0)
    for one_minus_beta1, one_minus_beta2 in ((0.1, 0.001), (0.05, 0.05)):
        hyper = (ctypes.c_float * 8)(1.0 - one_minus_beta1, one_minus_beta1, 1.0 - one_minus_beta2,
                                     one_minus_beta2, 1.0, 0.01, 1.0, 1e-8)
        assert lib.bysj_adamw_step(table, 1, 0, 8, at, at, at, at, None, None, hyper, None) == 1
        assert b"bysj_adamw_step_counted" in lib.bysj_last_error()


@pytest.mark.parametrize("noise", [None, 0.75])
def test_zero_beside_values_whose_scale_has_no_finite_inverse(noise):
    x = np.zeros((1, O.BLOCK), np.float32)
    x[0, :2] = 1e-39, 1e-40
    noise = None if noise is None else np.full(x.shape, noise)
    for top, values in ((127, O.VALUES_M), (255, O.VALUES_V)):
        code, scale = O.encode(x, top, values, noise)
        assert (code[0, :2] == top).all() and (code[0, 2:] == 0).all() and scale[0] == x[0, 0]
