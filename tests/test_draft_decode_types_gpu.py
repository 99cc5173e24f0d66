"""The drafted decode, built and run under another default type of torch."""

from __future__ import annotations

import pytest
import torch

from unicache_b200 import kernels
from unicache_b200.workloads import DraftDecode

from .gpu_util import need_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("default", [torch.float64, torch.bfloat16, torch.float16])
def test_a_step_under_another_default_type(default):
    need_gpu()
    kernels.device_status()
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        model = DraftDecode("cuda", prompts=[70, 33], samples=2, new_tokens=16, vocab=500)
        tokens, accepted, logprobs = model.step()
    finally:
        torch.set_default_dtype(before)
    assert logprobs.dtype is torch.float32 and tokens.dtype is torch.int32
    same = DraftDecode("cuda", prompts=[70, 33], samples=2, new_tokens=16, vocab=500)
    for got, want in zip((tokens, accepted, logprobs), same.step()):
        assert torch.equal(got, want)
    assert model.pool.lengths.tolist() == [n + 1 + int(a) for n, a in zip([70, 33, 70, 33], accepted)]
    assert kernels.device_status() == 0
