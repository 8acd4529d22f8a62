"""Train a small routed attention block on frames of atoms.

One step runs the training-step operators together with the segmented ones:

    type embedding -> group_norm (+ SiLU, per frame) -> q, k, v
    -> rotary_axes (coordinates turn q and k) -> edge scores
    -> segment_softmax / segment_sum over each atom's neighbours
    -> group_norm -> route_experts -> group_by_source -> the experts' products
    -> segment_sum of the atoms' energies per frame
    -> energy error + balance loss + z loss -> backward -> AdamW (8-bit states)

The target is a pair energy of the same synthetic periodic boxes.  Needs a B200:

    python examples/train_atom_block.py --steps 200
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from bysj_b200 import kernels as K  # noqa: E402
from bysj_b200 import workloads as W  # noqa: E402

RCUT = 6.0


def make_frames(count: int, atoms: int, seed: int, device: str):
    """Packed frames: atoms and edges of `count` boxes one after another, and their pair energies."""
    box = 12.4
    graphs = [W.water_box(atoms, box=box, rcut=RCUT, seed=seed + i, device=device)
              for i in range(count)]
    r2 = [(g.edge_vec ** 2).sum(-1) for g in graphs]
    energy = torch.stack([(0.5 * torch.exp(-d / 4.0) * (1.0 + g.types[g.src] + g.types[g.dst])).sum()
                          for g, d in zip(graphs, r2)]).float()
    frame = {
        "types": torch.cat([g.types for g in graphs]),
        "pos": torch.cat([g.pos for g in graphs]).float(),
        "src": torch.cat([g.src + i * atoms for i, g in enumerate(graphs)]),
        "dst": torch.cat([g.dst + i * atoms for i, g in enumerate(graphs)]),
        "env": (1.0 - torch.cat(r2) / RCUT ** 2).clamp(min=0.0).contiguous(),
        "frames": torch.arange(count + 1, device=device) * atoms,
        "frame_of": torch.arange(count, device=device).repeat_interleave(atoms),
        "energy": (energy - energy.mean()) / energy.std(),
        "box": box,
    }
    frame["offsets"] = K.segment_offsets(frame["dst"], count * atoms)
    return frame


class AtomBlock(torch.nn.Module):
    """Attention over neighbours and a routed feed-forward, C channels, H heads, E experts."""

    def __init__(self, channels=64, heads=4, experts=8, top_k=2, waves=2):
        super().__init__()
        c, self.heads, self.experts, self.top_k = channels, heads, experts, top_k
        self.sections = (waves, waves, waves)

        def matrix(*shape):
            return torch.nn.Parameter(torch.randn(*shape) / math.sqrt(shape[-2]))

        self.embed = torch.nn.Parameter(torch.randn(2, c))
        self.norm1_w, self.norm2_w = (torch.nn.Parameter(torch.ones(c)) for _ in range(2))
        self.norm1_b, self.norm2_b = (torch.nn.Parameter(torch.zeros(c)) for _ in range(2))
        self.qkv, self.out = matrix(c, 3 * c), matrix(c, c)
        self.router = matrix(c, experts)
        self.up, self.down = matrix(experts, c, 2 * c), matrix(experts, 2 * c, c)
        self.head = matrix(c, 1)

    def forward(self, f):
        c, h = self.embed.shape[1], self.heads
        x = self.embed[f["types"]]
        y = K.group_norm(x, h, self.norm1_w, self.norm1_b, activation="silu", offsets=f["frames"])
        q, k, v = (y @ self.qkv).view(-1, 3 * h, c // h).split(h, 1)
        # waves that are periodic in the box: a score depends on minimum-image differences
        wave = torch.arange(1, self.sections[0] + 1, device=x.device, dtype=torch.float32)
        inv_freq = (2.0 * math.pi / f["box"] * wave).repeat(3)
        q, k = K.rotary_axes(q, k, f["pos"], inv_freq, self.sections)
        score = (q[f["dst"]] * k[f["src"]]).sum(-1) / math.sqrt(c // h)
        alpha = K.segment_softmax(score.contiguous(), f["env"], f["offsets"])
        message = (alpha[:, :, None] * v[f["src"]]).reshape(-1, c)
        x = x + K.segment_sum(message, f["dst"], f["offsets"]) @ self.out

        y = K.group_norm(x, h, self.norm2_w, self.norm2_b, offsets=f["frames"])
        routing = K.route_experts(y @ self.router, self.top_k, offsets=f["frames"],
                                  renormalize=True)
        order, begin = K.group_by_source(routing.experts.flatten(), self.experts)
        ends = begin.tolist()
        rows = y[order // self.top_k]  # grouped by expert
        parts = [torch.nn.functional.silu(rows[a:b] @ self.up[e]) @ self.down[e]
                 for e, (a, b) in enumerate(zip(ends[:-1], ends[1:]))]
        slots = torch.empty_like(rows).index_copy(0, order, torch.cat(parts))
        x = x + (slots.view(-1, self.top_k, c) * routing.weights[..., None]).sum(1)

        energy = K.segment_sum((x @ self.head).contiguous(), f["frame_of"], f["frames"])
        return energy.squeeze(-1) / math.sqrt(x.shape[0]), routing


def train(steps=100, frames=8, atoms=192, seed=0, device="cuda", log=None):
    """Loss of every step."""
    torch.manual_seed(seed)
    data = make_frames(frames, atoms, seed, device)
    model = AtomBlock().to(device)
    params = list(model.parameters())
    opt = K.AdamW(params, lr=3.0e-3, betas=(0.9, 0.95), weight_decay=0.01, state_bits=8)
    losses = []
    for step in range(steps):
        energy, routing = model(data)
        error = ((energy - data["energy"]) ** 2).mean()
        loss = error + 0.01 * routing.balance + 0.001 * routing.z
        opt.zero_grad()
        loss.backward()
        norm = torch.stack([p.grad.norm() for p in params]).norm()
        opt.step(grad_scale=(1.0 / norm.clamp(min=1.0)).float().reshape(1))
        losses.append(error.detach())
        if log and step % 20 == 0:
            log(f"step {step}: energy error {float(error.detach()):.4f}, "
                f"balance {float(routing.balance.detach()):.3f}, "
                f"tokens of an expert {routing.counts.sum(0).tolist()}")
    return torch.stack(losses).tolist()


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--frames", type=int, default=8)
    parser.add_argument("--atoms", type=int, default=192)
    args = parser.parse_args()
    history = train(args.steps, args.frames, args.atoms, log=print)
    print(f"energy error {history[0]:.4f} -> {history[-1]:.4f}")
