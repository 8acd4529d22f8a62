"""Refusals of the torch shim are exceptions, numbers in their messages included (no GPU)."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

from bysj_b200 import _build

ROOT = Path(__file__).resolve().parents[1]


def test_a_message_with_numbers_does_not_end_the_process():
    if not _build.extension_path().exists():
        pytest.skip("extension not built (python -m bysj_b200._build)")
    code = ("import torch\n"
            "from bysj_b200 import _C\n"
            "try:\n"
            "    _C.AdamWParams([torch.zeros(3)], [0, 256])\n"
            "except RuntimeError as error:\n"
            "    print(str(error).splitlines()[0])\n")
    # in a process of its own: the fault that it looks for is a crash
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    assert "1 parameters, 2 begins" in done.stdout
