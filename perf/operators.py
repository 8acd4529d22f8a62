"""Workloads of the training-step operators: rotary_axes, group_norm, route_experts and AdamW.

Each case is one call (forward only, or forward and backward) of one operator
on synthetic inputs.  ``run`` computes it in plain 32-bit torch operations, or,
with ``own = True``, through ``bysj_b200.kernels``.  ``exact`` evaluates the
operator's definition in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 256          # elements that share one scale in an 8-bit optimizer state
ROTARY_BASE = 10000.0


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # One new token of a grid (time, height, width) whose q and k are views of one projection row.
        {"name": "rotary-token", "op": "rotary", "tokens": 1, "q_heads": 16, "k_heads": 4, "dim": 64,
         "sections": "16,8,8", "interleaved": False, "dtype": "bf16", "float_pos": False,
         "packed": True, "train": False},
        # A training step on one 3000-atom frame: positions are coordinates, whose gradient is a force.
        {"name": "rotary-atoms-train", "op": "rotary", "tokens": 3000, "q_heads": 8, "k_heads": 8,
         "dim": 32, "sections": "5,5,6", "interleaved": True, "dtype": "f32", "float_pos": True,
         "packed": False, "train": True},
        # A training step on four boxes of 24576 tokens, fused projection, grid positions.
        {"name": "rotary-boxes-train", "op": "rotary", "tokens": 98304, "q_heads": 16, "k_heads": 4,
         "dim": 64, "sections": "16,8,8", "interleaved": False, "dtype": "bf16", "float_pos": False,
         "packed": True, "train": True},
        # Inference on one 192-atom frame: a latency case.
        {"name": "norm-frame", "op": "norm", "rows": 192, "frames": 1, "ragged": False, "inner": 1,
         "channels": 64, "groups": 8, "dtype": "f32", "act": "silu", "affine": True, "train": False},
        # A training batch of packed frames of different sizes, an empty one among them.
        {"name": "norm-ragged-train", "op": "norm", "rows": 180001, "frames": 61, "ragged": True,
         "inner": 1, "channels": 96, "groups": 12, "dtype": "f32", "act": "silu", "affine": True,
         "train": True},
        # A training batch of sixteen 24576-atom frames of 128 channels.
        {"name": "norm-batch-train", "op": "norm", "rows": 393216, "frames": 16, "ragged": False,
         "inner": 1, "channels": 128, "groups": 32, "dtype": "bf16", "act": "silu", "affine": True,
         "train": True},
        # Routing one token when serving.
        {"name": "route-token", "op": "route", "tokens": 1, "experts": 64, "k": 4, "frames": 0,
         "masked": False, "renormalize": True, "dtype": "f32", "train": False},
        # A training step on packed frames of 24576 atoms in all, padding masked, one loss per frame.
        {"name": "route-frames-train", "op": "route", "tokens": 24576, "experts": 16, "k": 2,
         "frames": 9, "masked": True, "renormalize": False, "dtype": "f32", "train": True},
        # A training step on one 500k-token batch.
        {"name": "route-batch-train", "op": "route", "tokens": 500000, "experts": 128, "k": 8,
         "frames": 0, "masked": False, "renormalize": True, "dtype": "bf16", "train": True},
        # One step of a small model of 46 tensors, most of them tiny: a latency case.
        {"name": "adamw-small", "op": "adamw", "width": 64, "layers": 4, "extra": 89, "dtype": "f32",
         "bits": 32, "master": False, "flat": False, "clip": True, "step": 7},
        # bf16 weights with 32-bit masters and 8-bit states, odd widths.
        {"name": "adamw-8bit", "op": "adamw", "width": 803, "layers": 5, "extra": 1001,
         "dtype": "bf16", "bits": 8, "master": True, "flat": False, "clip": True, "step": 100},
        # 32-bit weights and states of a model of about 100 M parameters.
        {"name": "adamw-large", "op": "adamw", "width": 1312, "layers": 5, "extra": 1000,
         "dtype": "f32", "bits": 32, "master": False, "flat": False, "clip": False, "step": 1000},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "norm", "route", "adamw"])
    if op == "rotary":
        q_heads = rng.randint(1, 16)
        k_heads = rng.randint(1, min(q_heads, 8))
        dim = 2 * _log_uniform(rng, 4, 64)
        axes = rng.randint(1, 4)
        pairs = dim // 2 if rng.random() < 0.7 else rng.randint(1, dim // 2)
        cuts = sorted(rng.randint(0, pairs) for _ in range(axes - 1))
        sections = [b - a for a, b in zip([0] + cuts, cuts + [pairs])]
        top = max(1, (98304 * 20 * 64) // ((q_heads + k_heads) * dim))
        dtype = rng.choice(["f32", "bf16"])
        if dtype == "f32":
            top = max(1, top // 4)
        return {"op": op, "tokens": _log_uniform(rng, 1, min(top, 98304)), "q_heads": q_heads,
                "k_heads": k_heads, "dim": dim, "sections": ",".join(map(str, sections)),
                "interleaved": rng.random() < 0.5, "dtype": dtype,
                "float_pos": rng.random() < 0.5, "packed": rng.random() < 0.5,
                "train": rng.random() < 0.6}
    if op == "norm":
        groups = _log_uniform(rng, 1, 32)
        channels = groups * rng.randint(1, max(1, 160 // groups))
        inner = rng.choice([1, 1, 1, 4, 16])
        dtype = rng.choice(["f32", "bf16"])
        top = (393216 * 128 // (2 if dtype == "f32" else 1)) // (channels * inner)
        rows = _log_uniform(rng, 1, min(top, 400000))
        ragged = rng.random() < 0.5
        frames = _log_uniform(rng, 1, 64)
        if not ragged:
            frames = min(frames, rows)
            rows = rows // frames * frames
        return {"op": op, "rows": rows, "frames": frames, "ragged": ragged, "inner": inner,
                "channels": channels, "groups": groups, "dtype": dtype,
                "act": rng.choice(["silu", "silu", "none"]), "affine": rng.random() < 0.8,
                "train": rng.random() < 0.6}
    if op == "route":
        experts = _log_uniform(rng, 2, 256)
        dtype = rng.choice(["f32", "bf16"])
        top = min(500000, 500000 * 128 // experts // (2 if dtype == "f32" else 1))
        return {"op": op, "tokens": _log_uniform(rng, 1, top), "experts": experts,
                "k": rng.randint(1, min(8, experts)), "frames": rng.choice([0, 0, 1, 5, 40]),
                "masked": rng.random() < 0.5, "renormalize": rng.random() < 0.5, "dtype": dtype,
                "train": rng.random() < 0.6}
    width = _log_uniform(rng, 9, 800)
    layers = rng.randint(1, 5)
    dtype = rng.choice(["f32", "bf16"])
    return {"op": op, "width": width, "layers": layers, "extra": rng.randint(1, 999),
            "dtype": dtype, "bits": rng.choice([8, 32]),
            "master": dtype == "bf16" and rng.random() < 0.6, "flat": rng.random() < 0.3,
            "clip": rng.random() < 0.5, "step": rng.choice([1, 10, 1000])}


def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _generator(seed, device):
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    return gen


def _cut(total, parts, seed):
    """`parts` segment lengths of different sizes that sum to `total`; from three parts on one is empty."""
    gen = torch.Generator().manual_seed(seed)
    weight = torch.rand(parts, generator=gen, dtype=torch.float64) + 0.25
    if parts > 2:
        weight[parts // 2] = 0.0
    ends = torch.round(torch.cumsum(weight, 0) / weight.sum() * total).to(torch.int64)
    ends[-1] = total
    return torch.cat([torch.zeros(1, dtype=torch.int64), ends])


# ---------------------------------------------------------------------------
# rotary positions with several axes
# ---------------------------------------------------------------------------

def _sections(case):
    return [int(s) for s in case["sections"].split(",")]


def _rotary_inputs(case, seed):
    gen = _generator(seed, "cuda")
    tokens, hq, hk, dim = case["tokens"], case["q_heads"], case["k_heads"], case["dim"]
    dtype, sections = _dtype(case), _sections(case)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    if case["packed"]:
        # q | k | v of one projection: q and k are views of its rows
        qkv = normal(tokens, hq + 2 * hk, dim)
        q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    else:
        q, k = normal(tokens, hq, dim), normal(tokens, hk, dim)
    if case["float_pos"]:
        # coordinates in a 62.65 A box with the wave numbers that are periodic in it
        pos = torch.rand(tokens, len(sections), generator=gen, device="cuda") * 62.65
        freq = [2.0 * math.pi * (i + 1) / 62.65 / (1 + i // 8) for s in sections for i in range(s)]
    else:
        pos = torch.randint(0, 100, (tokens, len(sections)), generator=gen, device="cuda")
        freq = [ROTARY_BASE ** (-i / s) for s in sections for i in range(s)]
    state = {"q": q, "k": k, "positions": pos,
             "inv_freq": torch.tensor(freq, dtype=torch.float32, device="cuda")}
    if case["train"]:
        state["grad_q"], state["grad_k"] = normal(tokens, hq, dim), normal(tokens, hk, dim)
    return state


def _rotary_prepare(case, seed):
    state = _rotary_inputs(case, seed)
    if own and case["train"]:
        for name in ("q", "k"):
            state[name] = state[name].detach().requires_grad_()
        if case["float_pos"]:
            state["positions"].requires_grad_()
    return state


def _pair_views(x, pairs, interleaved):
    if interleaved:
        return x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
    return x[..., :pairs], x[..., pairs:2 * pairs]


def _rotary_plain(state, case):
    sections, inter = _sections(case), case["interleaved"]
    pairs = sum(sections)
    axis = torch.tensor([a for a, s in enumerate(sections) for _ in range(s)], device="cuda")
    theta = state["positions"].to(torch.float32)[:, axis] * state["inv_freq"]
    cos, sin = torch.cos(theta)[:, None], torch.sin(theta)[:, None]

    def rotate(x, s):
        x = x.to(torch.float32)
        out = x.clone()
        x1, x2 = _pair_views(x, pairs, inter)
        y1, y2 = _pair_views(out, pairs, inter)
        y1.copy_(x1 * cos - x2 * s)
        y2.copy_(x2 * cos + x1 * s)
        return out

    dtype = state["q"].dtype
    out = {"q": rotate(state["q"], sin).to(dtype), "k": rotate(state["k"], sin).to(dtype)}
    if case["train"]:
        dtheta = 0.0
        for name in ("q", "k"):
            grad = rotate(state["grad_" + name], -sin)
            out["grad_" + name] = grad.to(dtype)
            if case["float_pos"]:
                x1, x2 = _pair_views(state[name].to(torch.float32), pairs, inter)
                g1, g2 = _pair_views(grad, pairs, inter)
                dtheta = dtheta + (g2 * x1 - g1 * x2).sum(1)
        if case["float_pos"]:
            weighted = dtheta * state["inv_freq"]
            out["grad_positions"] = torch.stack(
                [p.sum(1) for p in torch.split(weighted, sections, dim=1)], dim=1)
    return out


def _rotary_own(state, case):
    from bysj_b200 import kernels as K

    q, k = K.rotary_axes(state["q"], state["k"], state["positions"], state["inv_freq"],
                         _sections(case), interleaved=case["interleaved"])
    out = {"q": q, "k": k}
    if case["train"]:
        wanted = [state["q"], state["k"]] + ([state["positions"]] if case["float_pos"] else [])
        grads = torch.autograd.grad([q, k], wanted, [state["grad_q"], state["grad_k"]])
        out["grad_q"], out["grad_k"] = grads[0], grads[1]
        if case["float_pos"]:
            out["grad_positions"] = grads[2]
    return out


def _rotary_exact(case, seed):
    state = _rotary_inputs(case, seed)
    sections, inter = _sections(case), case["interleaved"]
    pairs = sum(sections)
    pos = state["positions"].double().requires_grad_()
    spread = torch.repeat_interleave(pos, torch.tensor(sections, device="cuda"), dim=1)
    phase = spread * state["inv_freq"].double()
    turn = torch.polar(torch.ones_like(phase), phase)[:, None]
    out, grads = {}, 0.0
    for name in ("q", "k"):
        x = state[name].detach().double().contiguous().requires_grad_()
        head, tail = x[..., :2 * pairs], x[..., 2 * pairs:]
        z = (torch.view_as_complex(head.unflatten(-1, (pairs, 2)).contiguous()) if inter
             else torch.complex(head[..., :pairs], head[..., pairs:]))
        z = z * turn
        y = (torch.view_as_real(z).flatten(-2) if inter else torch.cat([z.real, z.imag], -1))
        y = torch.cat([y, tail], -1)
        out[name] = y.detach()
        if case["train"]:
            g = torch.autograd.grad(y, [x, pos], state["grad_" + name].double(), retain_graph=True)
            out["grad_" + name] = g[0]
            grads = grads + g[1]
    if case["train"] and case["float_pos"]:
        out["grad_positions"] = grads
    order = ["q", "k"] + (["grad_q", "grad_k"] if case["train"] else [])
    order += ["grad_positions"] if case["train"] and case["float_pos"] else []
    return {name: out[name] for name in order}


def _rotary_work(case):
    t, dim = case["tokens"], case["dim"]
    item = 4 if case["dtype"] == "f32" else 2
    values = t * (case["q_heads"] + case["k_heads"]) * dim
    axes = len(_sections(case))
    pos = t * axes * (4 if case["float_pos"] else 8)
    rotated = t * (case["q_heads"] + case["k_heads"]) * sum(_sections(case))
    moved, flops = 2 * values * item + pos, 6 * rotated
    if case["train"]:
        moved += 2 * values * item
        flops += 6 * rotated
        if case["float_pos"]:
            moved += t * axes * 4
            flops += 4 * rotated
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------------------
# group norm with an activation, channels last
# ---------------------------------------------------------------------------

def _norm_shape(case):
    inner = (case["inner"],) if case["inner"] > 1 else ()
    if case["ragged"]:
        return (case["rows"], *inner, case["channels"])
    return (case["frames"], case["rows"] // case["frames"], *inner, case["channels"])


def _norm_inputs(case, seed):
    gen = _generator(seed, "cuda")
    dtype, channels = _dtype(case), case["channels"]
    shape = _norm_shape(case)
    shift = torch.randn(channels, generator=gen, device="cuda") * 0.5
    x = torch.randn(shape, generator=gen, device="cuda")
    state = {"x": (x * 1.5 + shift).to(dtype), "weight": None, "bias": None, "offsets": None}
    if case["affine"]:
        state["weight"] = torch.rand(channels, generator=gen, device="cuda") + 0.5
        state["bias"] = torch.randn(channels, generator=gen, device="cuda") * 0.1
    if case["ragged"]:
        state["offsets"] = _cut(case["rows"], case["frames"], seed).cuda()
    if case["train"]:
        state["grad"] = torch.randn(shape, generator=gen, device="cuda").to(dtype)
    return state


def _norm_prepare(case, seed):
    state = _norm_inputs(case, seed)
    if own and case["train"]:
        for name in ("x", "weight", "bias"):
            if state[name] is not None:
                state[name].requires_grad_()
    return state


def _norm_plain(state, case):
    x = state["x"]
    groups, channels = case["groups"], case["channels"]
    rows = x.numel() // channels
    v = x.to(torch.float32).reshape(rows, groups, channels // groups)
    frames = case["frames"]
    if case["ragged"]:
        lengths = (state["offsets"][1:] - state["offsets"][:-1]) * case["inner"]
        frame = torch.repeat_interleave(torch.arange(frames, device="cuda"), lengths,
                                        output_size=rows)
        count = (lengths.to(torch.float32) * (channels // groups)).clamp(min=1.0)[:, None]

        def total(rows_groups):      # [rows, groups] -> [frames, groups]
            zero = torch.zeros(frames, groups, device="cuda")
            return zero.index_add_(0, frame, rows_groups)

        def spread(values):          # [frames, groups] -> [rows, groups, 1]
            return values[frame][:, :, None]
    else:
        count = float(rows // frames * (channels // groups))

        def total(rows_groups):
            return rows_groups.reshape(frames, rows // frames, groups).sum(1)

        def spread(values):
            return values.repeat_interleave(rows // frames, dim=0)[:, :, None]

    mean = total(v.sum(2)) / count
    centred = v - spread(mean)
    var = total((centred * centred).sum(2)) / count
    rstd = 1.0 / torch.sqrt(var + 1.0e-5)
    xhat = centred * spread(rstd)
    weight = None if state["weight"] is None else state["weight"].reshape(groups, -1)
    z = xhat if weight is None else xhat * weight + state["bias"].reshape(groups, -1)
    sigma = 1.0 / (1.0 + torch.exp(-z)) if case["act"] == "silu" else None
    y = z if sigma is None else z * sigma
    out = {"y": y.reshape(x.shape).to(x.dtype)}
    if case["train"]:
        dz = state["grad"].to(torch.float32).reshape(v.shape)
        if sigma is not None:
            dz = dz * (sigma * (1.0 + z * (1.0 - sigma)))
        dxhat = dz if weight is None else dz * weight
        c1 = total(dxhat.sum(2)) / count
        c2 = total((dxhat * xhat).sum(2)) / count
        dx = spread(rstd) * (dxhat - spread(c1) - xhat * spread(c2))
        out["grad_x"] = dx.reshape(x.shape).to(x.dtype)
        if weight is not None:
            out["grad_weight"] = (dz * xhat).sum(0).reshape(-1)
            out["grad_bias"] = dz.sum(0).reshape(-1)
    return out


def _norm_own(state, case):
    from bysj_b200 import kernels as K

    act = None if case["act"] == "none" else case["act"]
    y = K.group_norm(state["x"], case["groups"], state["weight"], state["bias"], 1.0e-5,
                     activation=act, offsets=state["offsets"])
    out = {"y": y}
    if case["train"]:
        names = [n for n in ("x", "weight", "bias") if state[n] is not None]
        grads = torch.autograd.grad(y, [state[n] for n in names], state["grad"])
        out.update({"grad_" + n: g for n, g in zip(names, grads)})
    return out


def _norm_exact(case, seed):
    state = _norm_inputs(case, seed)
    groups, channels = case["groups"], case["channels"]
    if case["ragged"]:
        ends = state["offsets"].tolist()
        parts = [(state["x"][a:b], (a, b)) for a, b in zip(ends[:-1], ends[1:])]
    else:
        parts = [(state["x"][i], i) for i in range(case["frames"])]
    out = {"y": torch.empty(state["x"].shape, dtype=torch.float64, device="cuda")}
    leaves = []
    if case["affine"]:
        leaves = [state["weight"].double().requires_grad_(), state["bias"].double().requires_grad_()]
    if case["train"]:
        out["grad_x"] = torch.empty_like(out["y"])
        if case["affine"]:
            out["grad_weight"] = torch.zeros(channels, dtype=torch.float64, device="cuda")
            out["grad_bias"] = torch.zeros_like(out["grad_weight"])
    for part, where in parts:
        if part.numel() == 0:
            continue
        place = slice(*where) if case["ragged"] else where
        x = part.double().requires_grad_()
        columns = x.reshape(-1, groups, channels // groups)
        var, mean = torch.var_mean(columns, dim=(0, 2), unbiased=False, keepdim=True)
        z = ((columns - mean) / torch.sqrt(var + 1.0e-5)).reshape(-1, channels)
        if leaves:
            z = z * leaves[0] + leaves[1]
        y = (z * torch.sigmoid(z) if case["act"] == "silu" else z).reshape(x.shape)
        out["y"][place] = y.detach()
        if case["train"]:
            g = torch.autograd.grad(y, [x, *leaves], state["grad"][place].double())
            out["grad_x"][place] = g[0]
            if leaves:
                out["grad_weight"] += g[1]
                out["grad_bias"] += g[2]
    return out


def _norm_work(case):
    item = 4 if case["dtype"] == "f32" else 2
    values = case["rows"] * case["inner"] * case["channels"]
    channel_bytes = 8 * case["channels"] if case["affine"] else 0
    moved = 2 * values * item + channel_bytes
    flops = values * (12 if case["act"] == "silu" else 7)
    if case["train"]:
        moved += 2 * values * item + 2 * channel_bytes
        flops += values * (24 if case["act"] == "silu" else 14)
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------------------
# top-k router with per-expert counts, a balance loss and a z loss
# ---------------------------------------------------------------------------

def _route_inputs(case, seed):
    gen = _generator(seed, "cuda")
    tokens, experts, k = case["tokens"], case["experts"], case["k"]
    # a router in training: some experts are preferred
    preference = torch.randn(experts, generator=gen, device="cuda") * 0.5
    logits = torch.randn(tokens, experts, generator=gen, device="cuda") * 1.5 + preference
    state = {"logits": logits.to(_dtype(case)), "mask": None, "offsets": None}
    if case["masked"]:
        state["mask"] = torch.rand(tokens, generator=gen, device="cuda") < 0.9
    if case["frames"]:
        state["offsets"] = _cut(tokens, case["frames"], seed).cuda()
    if case["train"]:
        state["grad_weights"] = torch.randn(tokens, k, generator=gen, device="cuda")
        state["grad_balance"] = torch.tensor(0.01 * tokens, device="cuda")
        state["grad_z"] = torch.tensor(0.001 * tokens, device="cuda")
    return state


def _route_prepare(case, seed):
    state = _route_inputs(case, seed)
    if own and case["train"]:
        state["logits"].requires_grad_()
    return state


def _route_plain(state, case):
    tokens, experts, k = case["tokens"], case["experts"], case["k"]
    logits = state["logits"].to(torch.float32)
    valid = torch.ones(tokens, dtype=torch.bool, device="cuda")
    if state["mask"] is not None:
        valid = state["mask"]
    live = valid.to(torch.float32)[:, None]
    frames = max(1, case["frames"])
    if state["offsets"] is not None:
        frame = torch.repeat_interleave(torch.arange(frames, device="cuda"),
                                        state["offsets"][1:] - state["offsets"][:-1],
                                        output_size=tokens)
    else:
        frame = torch.zeros(tokens, dtype=torch.int64, device="cuda")
    top = logits.max(1, keepdim=True).values
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    p = e / total
    lse = top + torch.log(total)
    column = torch.arange(experts, device="cuda")
    left, chosen = logits.clone(), []
    for _ in range(k):
        best = left.max(1, keepdim=True).values
        index = torch.where(left == best, column, experts).min(1, keepdim=True).values
        left.scatter_(1, index, -math.inf)
        chosen.append(index)
    index = torch.cat(chosen, 1)
    picked = p.gather(1, index)
    norm = picked.sum(1, keepdim=True)
    weights = (picked / norm if case["renormalize"] else picked) * live

    def per_frame(values):          # [tokens, n] -> [frames, n]
        if frames == 1:
            return values.sum(0, keepdim=True)
        zero = torch.zeros(frames, values.shape[1], dtype=values.dtype, device="cuda")
        return zero.index_add_(0, frame, values)

    slots = torch.zeros(tokens, experts, dtype=torch.int32, device="cuda")
    slots.scatter_(1, index, 1)
    slots = slots * valid[:, None]
    counts = per_frame(slots).to(torch.int64)
    number = per_frame(live)
    used = (number > 0).to(torch.float32)
    share = counts.to(torch.float32) * (experts / k) / (number * number).clamp(min=1.0)
    share = share / used.sum().clamp(min=1.0)
    balance = (share * per_frame(p * live)).sum()
    everyone = number.sum().clamp(min=1.0)
    z = (lse * lse * live).sum() / everyone
    out = {"weights": weights, "experts": torch.where(valid[:, None], index, -1),
           "counts": counts if state["offsets"] is not None else counts[0],
           "balance": balance, "z": z}
    if case["train"]:
        gw = state["grad_weights"]
        gp = state["grad_balance"] * share[frame]
        direct = torch.zeros_like(p)
        if case["renormalize"]:
            w = picked / norm
            direct.scatter_(1, index, w * (gw - (w * gw).sum(1, keepdim=True)))
        else:
            gp = gp.scatter_add(1, index, gw)
        grad = p * (gp - (p * gp).sum(1, keepdim=True)) + direct
        grad = grad + state["grad_z"] * 2.0 * lse / everyone * p
        out["grad_logits"] = torch.where(valid[:, None], grad, 0.0).to(state["logits"].dtype)
    return out


def _route_own(state, case):
    from bysj_b200 import kernels as K

    r = K.route_experts(state["logits"], case["k"], mask=state["mask"], offsets=state["offsets"],
                        renormalize=case["renormalize"])
    out = {"weights": r.weights, "experts": r.experts, "counts": r.counts, "balance": r.balance,
           "z": r.z}
    if case["train"]:
        out["grad_logits"], = torch.autograd.grad(
            [r.weights, r.balance, r.z], [state["logits"]],
            [state["grad_weights"], state["grad_balance"], state["grad_z"]])
    return out


def _route_exact(case, seed):
    state = _route_inputs(case, seed)
    tokens, experts, k = case["tokens"], case["experts"], case["k"]
    x = state["logits"].double().requires_grad_()
    keep = torch.arange(tokens, device="cuda")
    if state["mask"] is not None:
        keep = keep[state["mask"]]
    logp = torch.log_softmax(x[keep], dim=1)
    lse = torch.logsumexp(x[keep], dim=1)
    index = torch.sort(x.detach()[keep], dim=1, descending=True, stable=True).indices[:, :k]
    gate = logp.gather(1, index)
    gate = torch.softmax(gate, dim=1) if case["renormalize"] else torch.exp(gate)
    ends = [0, tokens] if state["offsets"] is None else state["offsets"].tolist()
    place = torch.searchsorted(keep, torch.tensor(ends, device="cuda")).tolist()
    counts, losses = [], []
    for a, b in zip(place[:-1], place[1:]):
        counts.append(torch.bincount(index[a:b].reshape(-1), minlength=experts))
        if b > a:
            fraction = counts[-1].double() / (k * (b - a))
            losses.append(experts * (fraction * torch.exp(logp[a:b]).mean(0)).sum())
    balance = torch.stack(losses).mean() if losses else x.sum() * 0.0
    z = (lse * lse).mean() if keep.numel() else x.sum() * 0.0
    weights = torch.zeros(tokens, k, dtype=torch.float64, device="cuda").index_copy(0, keep, gate)
    chosen = torch.full((tokens, k), -1, dtype=torch.int64, device="cuda").index_copy(0, keep, index)
    counts = torch.stack(counts)
    out = {"weights": weights.detach(), "experts": chosen,
           "counts": counts if state["offsets"] is not None else counts[0],
           "balance": balance.detach(), "z": z.detach()}
    if case["train"]:
        out["grad_logits"], = torch.autograd.grad(
            [weights, balance, z], [x],
            [state[n].double() for n in ("grad_weights", "grad_balance", "grad_z")])
    return out


def _route_work(case):
    t, e, k = case["tokens"], case["experts"], case["k"]
    item = 4 if case["dtype"] == "f32" else 2
    moved = t * e * item + t * k * 12 + max(1, case["frames"]) * e * 8 + 8
    moved += t if case["masked"] else 0
    flops = t * e * 6
    if case["train"]:
        moved += t * e * item + t * k * 4
        flops += t * e * 6
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------------------
# AdamW over many tensors, states in 32 or 8 bits
#
# The states of all tensors lie in one buffer each: a tensor's share begins at
# a multiple of BLOCK elements, and what pads it to the next is zero.
# ---------------------------------------------------------------------------

HYPER = {"lr": 1.0e-3, "betas": (0.9, 0.95), "eps": 1.0e-8, "weight_decay": 0.1}


def _adamw_shapes(case):
    w, extra = case["width"], case["extra"]
    shapes = [(extra, w)]
    for _ in range(case["layers"]):
        shapes += [(w,), (3 * w, w), (3 * w,), (w, w), (w,), (w,), (4 * w, w), (4 * w,), (w, 4 * w),
                   (w,), (1,)]
    return shapes + [(extra,)]


def _places(shapes):
    """(begin, elements) of each tensor in the state buffers, and their length."""
    places, begin = [], 0
    for shape in shapes:
        n = math.prod(shape)
        places.append((begin, n))
        begin += -(-n // BLOCK) * BLOCK
    return places, begin


def _tensors(shapes, flat, values):
    """Tensors of `shapes`, each on its own or, where `flat`, as views that follow one another in one buffer."""
    parts = values.split([math.prod(s) for s in shapes])
    return [(t if flat else t.clone()).view(s) for t, s in zip(parts, shapes)]


def _adamw_inputs(case, seed):
    gen = _generator(seed, "cuda")
    shapes, dtype, flat = _adamw_shapes(case), _dtype(case), case["flat"]
    places, length = _places(shapes)
    total = sum(n for _, n in places)
    weights = torch.randn(total, generator=gen, device="cuda") * 0.05
    grads = torch.randn(total, generator=gen, device="cuda") * 0.01
    state = {"params": _tensors(shapes, flat, weights.to(dtype)),
             "grads": _tensors(shapes, flat, grads.to(dtype)), "master": None, "step": case["step"],
             "scale": torch.rand(1, generator=gen, device="cuda") + 0.5 if case["clip"] else None,
             "exp_avg_scale": None, "exp_avg_sq_scale": None}
    inside = torch.zeros(length, dtype=torch.bool, device="cuda")
    for begin, n in places:
        inside[begin:begin + n] = True
    if case["master"]:
        state["master"] = torch.zeros(length, device="cuda")
        for (begin, n), part in zip(places, weights.split([n for _, n in places])):
            state["master"][begin:begin + n] = part
    if case["bits"] == 32:
        first = torch.randn(length, generator=gen, device="cuda") * 0.003
        second = torch.randn(length, generator=gen, device="cuda").square() * 1.0e-4
        state["exp_avg"], state["exp_avg_sq"] = first * inside, second * inside
        return state
    # codes whose largest in each block is the top one, as a step leaves them
    code = torch.randint(40, 128, (length,), generator=gen, device="cuda")
    code[::BLOCK] = 127
    sign = torch.randint(0, 2, (length,), generator=gen, device="cuda")
    state["exp_avg"] = ((code + 128 * sign) * inside).to(torch.uint8)
    code = torch.randint(150, 256, (length,), generator=gen, device="cuda")
    code[::BLOCK] = 255
    state["exp_avg_sq"] = (code * inside).to(torch.uint8)
    blocks = length // BLOCK
    state["exp_avg_scale"] = torch.rand(blocks, generator=gen, device="cuda") * 0.01 + 0.001
    state["exp_avg_sq_scale"] = torch.rand(blocks, generator=gen, device="cuda") * 0.01 + 0.005
    return state


def _adamw_prepare(case, seed):
    state = _adamw_inputs(case, seed)
    if own:
        from bysj_b200 import kernels as K

        opt = K.AdamW(state["params"], **HYPER, state_bits=case["bits"], master_weights=case["master"])
        opt.load_state_dict({key: state[key] for key in
                             ("step", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale",
                              "master")})
        state = {"opt": opt, "params": state["params"], "grads": state["grads"],
                 "scale": state["scale"]}
    return state


def _decode(code, top, mantissa):
    code = code.to(torch.int32)
    bits = (code - top + (127 << mantissa)) << (23 - mantissa)
    return torch.where(code > 0, bits.view(torch.float32), 0.0)


def _spread_blocks(scale):
    return scale.repeat_interleave(BLOCK)


def _encode(x, scale, top, mantissa):
    """Nearest code of x / scale for x >= 0, not yet cut at the bottom end, and the ratio."""
    inverse = torch.where(scale > 0, 1.0 / scale, 0.0)
    ratio = x * _spread_blocks(inverse)
    shift = 23 - mantissa
    bits = ratio.view(torch.int32)
    code = (bits + ((1 << (shift - 1)) - 1) + ((bits >> shift) & 1)) >> shift
    return (code - (127 << mantissa) + top).clamp(max=top), ratio


def _adamw_constants(step):
    beta1, beta2 = HYPER["betas"]
    return {"b1": beta1, "c1": 1.0 - beta1, "b2": beta2, "c2": 1.0 - beta2,
            "decay": 1.0 - HYPER["lr"] * HYPER["weight_decay"],
            "size": HYPER["lr"] / (1.0 - beta1 ** step),
            "correct": 1.0 / math.sqrt(1.0 - beta2 ** step)}


def _adamw_plain(state, case):
    state["step"] += 1
    c = _adamw_constants(state["step"])
    places, length = _places(_adamw_shapes(case))
    g = torch.zeros(length, device="cuda")
    for (begin, n), grad in zip(places, state["grads"]):
        g[begin:begin + n] = grad.reshape(-1)
    if state["scale"] is not None:
        g = g * state["scale"]
    m, v = state["exp_avg"], state["exp_avg_sq"]
    if case["bits"] == 8:
        magnitude = _decode(m & 127, 127, 3) * _spread_blocks(state["exp_avg_scale"])
        u = _decode(v, 255, 4) * _spread_blocks(state["exp_avg_sq_scale"])
        m, v = torch.where(m >= 128, -magnitude, magnitude), u * u
    m = m * c["b1"] + g * c["c1"]
    v = v * c["b2"] + g * c["c2"] * g
    root = torch.sqrt(v)
    update = m / (root * c["correct"] + HYPER["eps"]) * c["size"]
    for (begin, n), param in zip(places, state["params"]):
        p = param.reshape(-1) if state["master"] is None else state["master"][begin:begin + n]
        p = p.to(torch.float32) * c["decay"] - update[begin:begin + n]
        if state["master"] is not None:
            state["master"][begin:begin + n] = p
        param.copy_(p.to(param.dtype).view(param.shape))
    out = {"params": state["params"]}
    if state["master"] is not None:
        out["master"] = state["master"]
    if case["bits"] == 32:
        state["exp_avg"].copy_(m)
        state["exp_avg_sq"].copy_(v)
        out["exp_avg"], out["exp_avg_sq"] = state["exp_avg"], state["exp_avg_sq"]
        return out
    scale = m.abs().view(-1, BLOCK).amax(1)
    code, ratio = _encode(m.abs(), scale, 127, 3)
    low = torch.where(ratio >= 0.5 * 1.25 * 2.0 ** -16, 1, 0)
    code = torch.where(code >= 1, code, low)
    state["exp_avg"].copy_(torch.where(m < 0, code + 128, code))
    state["exp_avg_scale"].copy_(scale)
    value = _decode(code, 127, 3) * _spread_blocks(scale)
    out["exp_avg"] = torch.where(m < 0, -value, value)
    scale = root.view(-1, BLOCK).amax(1)
    code, _ = _encode(root, scale, 255, 4)
    code = torch.where(root > 0, code.clamp(min=1), 0)
    state["exp_avg_sq"].copy_(code)
    state["exp_avg_sq_scale"].copy_(scale)
    value = _decode(code, 255, 4) * _spread_blocks(scale)
    out["exp_avg_sq"] = value * value
    return out


def _adamw_own(state, case):
    opt = state["opt"]
    opt.step(state["grads"], grad_scale=state["scale"])
    first, second = opt.state_values()
    out = {"params": state["params"]}
    if case["master"]:
        out["master"] = opt.master
    out["exp_avg"], out["exp_avg_sq"] = first, second
    return out


def _adamw_exact(case, seed):
    state = _adamw_inputs(case, seed)
    beta1, beta2 = HYPER["betas"]
    step = state["step"] + 1
    places, length = _places(_adamw_shapes(case))
    # the values of the codes, ascending: octaves of 8 and of 16 steps below 1
    grid = {}
    for top, mantissa in ((127, 3), (255, 4)):
        values = [0.0]
        for code in range(1, top + 1):
            octave, part = divmod(code - top, 1 << mantissa)
            values.append(2.0 ** octave * (1.0 + part / (1 << mantissa)))
        grid[top] = torch.tensor(values, dtype=torch.float64, device="cuda")

    def loaded(code, scale, top):
        return (grid[top][code.long()].view(-1, BLOCK) * scale.double()[:, None]).view(-1)

    def stored(x, top):
        """The value that x >= 0 has after its block went through the codes."""
        whole = x.view(-1, BLOCK)
        scale = whole.max(1, keepdim=True).values
        ratio = whole / torch.where(scale > 0, scale, 1.0)
        values = grid[top]
        middle = (values[1:] + values[:-1]) / 2
        code = torch.bucketize(ratio, middle)
        # a tie goes to the even mantissa, whose code is odd as the top code (1.0) is
        tie = (ratio == middle[code.clamp(max=top - 1)]) & (code < top) & (code % 2 == 0)
        code = code + tie.to(code.dtype)
        if top == 255:
            code = torch.where(whole > 0, code.clamp(min=1), 0)
        return (values[code] * scale).view(-1)

    index = torch.cat([torch.arange(begin, begin + n, device="cuda") for begin, n in places])
    g = torch.zeros(length, dtype=torch.float64, device="cuda")
    g[index] = torch.cat([t.reshape(-1) for t in state["grads"]]).double()
    p = torch.zeros_like(g)
    p[index] = torch.cat([t.reshape(-1) for t in state["params"]]).double()
    if state["master"] is not None:
        p = state["master"].double()
    if state["scale"] is not None:
        g = g * state["scale"].double()
    m, v = state["exp_avg"], state["exp_avg_sq"]
    if case["bits"] == 8:
        sign = 1.0 - 2.0 * (m // 128).double()
        m = sign * loaded(m % 128, state["exp_avg_scale"], 127)
        v = loaded(v, state["exp_avg_sq_scale"], 255) ** 2
    m = beta1 * m.double() + (1.0 - beta1) * g
    v = beta2 * v.double() + (1.0 - beta2) * g ** 2
    update = (m / (1.0 - beta1 ** step)) / (torch.sqrt(v / (1.0 - beta2 ** step)) + HYPER["eps"])
    p = p - HYPER["lr"] * (update + HYPER["weight_decay"] * p)
    out = {"params": [p[begin:begin + n].view(t.shape) for (begin, n), t in
                      zip(places, state["params"])]}
    if state["master"] is not None:
        out["master"] = p
    if case["bits"] == 8:
        m = torch.sign(m) * stored(m.abs(), 127)
        v = stored(torch.sqrt(v), 255) ** 2
    out["exp_avg"], out["exp_avg_sq"] = m, v
    return out


def _adamw_work(case):
    n = sum(math.prod(s) for s in _adamw_shapes(case))
    item = 4 if case["dtype"] == "f32" else 2
    moved = n * (item + 8 if case["master"] else 2 * item) + n * item
    if case["bits"] == 32:
        moved += 16 * n
    else:
        # codes and block scales in and out, and the values that they stand for
        moved += 4 * n + 16 * (n // BLOCK) + 8 * n
    return {"bytes": moved, "flops": 15 * n}


# ---------------------------------------------------------------------------
# the four operators behind one interface
# ---------------------------------------------------------------------------

_PREPARE = {"rotary": _rotary_prepare, "norm": _norm_prepare, "route": _route_prepare,
            "adamw": _adamw_prepare}
_PLAIN = {"rotary": _rotary_plain, "norm": _norm_plain, "route": _route_plain, "adamw": _adamw_plain}
_OWN = {"rotary": _rotary_own, "norm": _norm_own, "route": _route_own, "adamw": _adamw_own}
_EXACT = {"rotary": _rotary_exact, "norm": _norm_exact, "route": _route_exact, "adamw": _adamw_exact}
_WORK = {"rotary": _rotary_work, "norm": _norm_work, "route": _route_work, "adamw": _adamw_work}


def prepare(case, seed):
    state = _PREPARE[case["op"]](case, seed)
    state["case"] = case
    return state


def run(state):
    case = state["case"]
    return (_OWN if own else _PLAIN)[case["op"]](state, case)


def work(case):
    return _WORK[case["op"]](case)


def exact(case, seed):
    return _EXACT[case["op"]](case, seed)
