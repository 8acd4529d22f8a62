"""The training example runs all operators together and learns (B200)."""
from __future__ import annotations

import importlib.util
import math
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "train_atom_block.py"


def test_example_learns(cuda):
    spec = importlib.util.spec_from_file_location("train_atom_block", EXAMPLE)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses = example.train(steps=60, frames=4)
    assert all(math.isfinite(v) for v in losses)
    # the targets have unit variance: better than half of what the first step left
    assert min(losses[-10:]) < 0.5 * losses[0]
