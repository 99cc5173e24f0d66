"""verify_drafts under another default type of torch: the same results in the same types."""

from __future__ import annotations

import pytest
import torch

from unicache_b200 import verify_drafts

from .gpu_util import need_gpu
from .test_verify_drafts_gpu import inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("i,default", list(enumerate([torch.float64, torch.bfloat16, torch.float16, torch.float32])))
def test_another_default_type_changes_nothing(i, default):
    need_gpu()
    logits, drafts, uniforms, probs = inputs(37, 4, 2311 + i, seed=i)  # shapes that no other test has called before
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        got = verify_drafts(logits, drafts, uniforms, draft_probs=probs)
    finally:
        torch.set_default_dtype(before)
    want = verify_drafts(logits, drafts, uniforms, draft_probs=probs)
    again = verify_drafts(logits[:, :, :2300], drafts % 2300, uniforms, draft_probs=probs[:, :, :2300])
    assert [x.dtype for x in got] == [torch.int32, torch.int32, torch.float32] == [x.dtype for x in again]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
