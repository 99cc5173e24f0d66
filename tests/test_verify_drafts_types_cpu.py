"""What verify_drafts allocates has the types that its kernels write, whatever type torch takes by default."""

from __future__ import annotations

import pytest
import torch

from unicache_b200 import kernels


@pytest.mark.parametrize("default", [torch.float32, torch.float64, torch.bfloat16, torch.float16])
def test_output_patterns_name_their_types(default, monkeypatch):
    device = torch.device
    monkeypatch.setattr(torch, "device", lambda *_: device("meta"))
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:  # no sequences: the library is not asked for the workspace
        patterns = kernels._verify_patterns.__wrapped__(0, 0, 4, 100, kernels.dtype_code(torch.bfloat16))
    finally:
        torch.set_default_dtype(before)
    assert [p.dtype for p in patterns] == [torch.int32, torch.float32, torch.int32, torch.uint8]
