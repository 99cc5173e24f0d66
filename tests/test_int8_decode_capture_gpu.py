"""The decode workload over 8-bit block caches captured before any step has run."""

from __future__ import annotations

import os
import subprocess
import sys

import pytest
import torch

from .gpu_util import need_gpu

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# In a process of its own: what a first call sets up is set up once a process.
SCRIPT = """
import torch
from unicache_b200 import kernels
from unicache_b200.workloads import Int8BlockDecode

shape = dict(prompts=[700, 1, 63, 64, 1290], new_tokens=20, layers=2, hidden=512, q_heads=14, kv_heads=2, seed=3)
captured = Int8BlockDecode("cuda", **shape)
captured.capture()
eager = Int8BlockDecode("cuda", **shape)
for _ in range(10):
    assert torch.equal(captured.replay(), eager.step())
for a, b in zip(captured.caches, eager.caches):
    assert torch.equal(a.lengths, b.lengths)
    for name in ("key_code", "key_scale", "value_code", "value_scale", "key_low", "key_high"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name
assert kernels.device_status() == 0
print("equal")
"""


def test_a_step_may_be_captured_first():
    need_gpu()
    torch.cuda.synchronize()
    done = subprocess.run([sys.executable, "-c", SCRIPT], capture_output=True, text=True, timeout=300,
                          cwd=ROOT)
    assert done.returncode == 0 and done.stdout.strip() == "equal", done.stderr[-2000:]
