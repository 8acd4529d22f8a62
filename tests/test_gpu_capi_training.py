"""The training-step entries of the C ABI, through ctypes only (B200)."""
from __future__ import annotations

import ctypes
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

from bysj_b200 import kernels as K  # noqa: E402

LIB = Path(__file__).resolve().parents[1] / "bysj_b200" / "libbysj_b200.so"
P, I64, I32, SZ, F = (ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_size_t,
                      ctypes.c_float)


class Side(ctypes.Structure):
    _fields_ = [("x", P), ("y", P), ("saved", P)] + [
        (n, I64) for n in ("heads", "x_token_stride", "x_head_stride", "saved_token_stride",
                           "saved_head_stride")]


class Tensor(ctypes.Structure):
    _fields_ = [("param", P), ("grad", P), ("n", I64), ("first_block", I64)]


class Hyper(ctypes.Structure):
    _fields_ = [(n, F) for n in ("beta1", "one_minus_beta1", "beta2", "one_minus_beta2", "decay",
                                 "size", "correct", "eps")]


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    torch.cuda.init()
    handle = ctypes.CDLL(str(LIB))
    handle.bysj_rotary_axes.argtypes = [P, P, I32, P, I32, P, P, I32, I64, I64, I32, I32, P, P]
    handle.bysj_group_norm_forward_workspace_size.argtypes = [I64] * 4
    handle.bysj_group_norm_forward_workspace_size.restype = SZ
    handle.bysj_group_norm_forward.argtypes = [P, I32, I64, I64, I64, P, I64, I64, P, P, F, I32, P,
                                               P, P, P, SZ, P]
    handle.bysj_route_forward_workspace_size.argtypes = [I64] * 3
    handle.bysj_route_forward_workspace_size.restype = SZ
    handle.bysj_route_forward.argtypes = [P, I32, I64, I64, I64, P, P, I64, I32] + [P] * 9 + [SZ, P]
    handle.bysj_adamw_step.argtypes = [P, I64, I32, I32, P, P, P, P, P, P, P, P]
    handle.bysj_last_error.restype = ctypes.c_char_p
    return handle


def ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def test_rotary(cuda, lib):
    q, k = torch.randn(9, 3, 8, device="cuda"), torch.randn(9, 1, 8, device="cuda")
    pos, freq = torch.rand(9, 2, device="cuda"), torch.rand(4, device="cuda")
    yq, yk = torch.empty_like(q), torch.empty_like(k)
    sections = (I64 * 2)(1, 3)
    sides = [Side(ptr(x), ptr(y), None, x.shape[1], x.stride(0), x.stride(1), 0, 0)
             for x, y in ((q, yq), (k, yk))]

    def call(n_axes=2, inverse=0, grad=None):
        return lib.bysj_rotary_axes(ctypes.byref(sides[0]), ctypes.byref(sides[1]), 0, ptr(pos), 0,
                                    ptr(freq), sections, n_axes, 9, 8, 0, inverse, grad, stream())

    assert call() == 0
    want = K.rotary_axes(q, k, pos, freq, (1, 3))
    assert torch.equal(yq, want[0]) and torch.equal(yk, want[1])
    assert call(n_axes=5) == 1
    assert call(grad=ptr(pos)) == 1 and b"inverse" in lib.bysj_last_error()
    sections[1] = 4
    assert call() == 1


def test_group_norm(cuda, lib):
    x = torch.randn(3000, 48, device="cuda")
    offsets = torch.tensor([0, 1000, 1000, 3000], device="cuda")
    y = torch.empty_like(x)
    mean, rstd = torch.empty(3, 4, device="cuda"), torch.empty(3, 4, device="cuda")
    size = lib.bysj_group_norm_forward_workspace_size(3000, 48, 4, 3)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")

    def call(groups=4, bytes_=size, eps=1e-5, act=1):
        return lib.bysj_group_norm_forward(ptr(x), 0, 3000, 48, groups, ptr(offsets), 3, 1, None,
                                           None, eps, act, ptr(y), ptr(mean), ptr(rstd), ptr(ws),
                                           bytes_, stream())

    assert call() == 0
    assert torch.equal(y, K.group_norm(x, 4, activation="silu", offsets=offsets))
    assert torch.equal(mean[1], torch.zeros(4, device="cuda"))
    assert call(groups=5) == 1 and call(eps=0.0) == 1 and call(act=7) == 1
    assert size > 0 and call(bytes_=0) == 2


def test_route(cuda, lib):
    x = torch.randn(500, 16, device="cuda")
    f32, i64 = dict(device="cuda"), dict(device="cuda", dtype=torch.int64)
    weights, experts = torch.empty(500, 2, **f32), torch.empty(500, 2, **i64)
    counts, share = torch.empty(16, **i64), torch.empty(16, **f32)
    scalars, denom = torch.empty(3, **f32), torch.empty(500, **f32)
    size = lib.bysj_route_forward_workspace_size(500, 16, 1)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")

    def call(k=2, frames=1, n_experts=16, bytes_=size):
        return lib.bysj_route_forward(
            ptr(x), 0, 500, n_experts, k, None, None, frames, 0, ptr(weights), ptr(experts),
            ptr(counts), ptr(scalars), ctypes.c_void_p(scalars.data_ptr() + 4),
            ctypes.c_void_p(scalars.data_ptr() + 8), ptr(denom), ptr(share), ptr(ws), bytes_,
            stream())

    assert call() == 0
    want = K.route_experts(x, 2)
    assert torch.equal(weights, want.weights) and torch.equal(experts, want.experts)
    assert torch.equal(counts, want.counts) and torch.equal(scalars[0], want.balance)
    assert torch.equal(scalars[1], want.z)
    assert call(k=17) == 1 and call(frames=2) == 1 and call(n_experts=2000) == 3
    assert call(bytes_=0) == 2


def test_adamw(cuda, lib):
    p, g = torch.randn(700, device="cuda"), torch.randn(700, device="cuda")
    other = p.clone()
    m, v = torch.zeros(768, device="cuda"), torch.zeros(768, device="cuda")
    table = (Tensor * 1)(Tensor(ptr(p), ptr(g), 700, 0))
    hyper = Hyper(0.9, 1.0 - 0.9, 0.99, 1.0 - 0.99, 1.0 - 0.01 * 0.1, 0.01 / (1.0 - 0.9),
                  1.0 / (1.0 - 0.99) ** 0.5, 1e-8)

    def call(bits=32, dtype=0):
        return lib.bysj_adamw_step(table, 1, dtype, bits, ptr(m), ptr(v), None, None, None, None,
                                   ctypes.byref(hyper), stream())

    assert call() == 0
    K.AdamW([other], lr=0.01, betas=(0.9, 0.99), weight_decay=0.1).step([g])
    assert torch.equal(p, other)
    assert call(bits=16) == 1 and call(dtype=9) == 1 and call(bits=8) == 1
