"""More refusals of the training-step operators (no GPU)."""
from __future__ import annotations

import pytest
import torch

import bysj_b200.kernels as K


@pytest.mark.parametrize("make", [
    lambda t: [t, t.view(-1)],                  # the same elements
    lambda t: [t[:3], t[2:]],                   # one row in common
    lambda t: [t[1], t],                        # a part
    lambda t: [torch.zeros(2), t, t[5, 3:]],    # the last element
])
def test_adamw_refuses_parameters_that_share_memory(make):
    # two blocks of one launch would read and write the shared elements in any order
    with pytest.raises(ValueError, match="share memory"):
        K.AdamW(make(torch.zeros(6, 4)))


@pytest.mark.skipif(torch.cuda.is_available(), reason="guard behaviour on a CPU host")
def test_adamw_takes_neighbours_and_empty_tensors():
    t = torch.zeros(6, 4)
    with pytest.raises(RuntimeError, match="CUDA"):  # the device guard comes next
        K.AdamW([t[3:], t[:3], t[3:3], torch.zeros(0)])
