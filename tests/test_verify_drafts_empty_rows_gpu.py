"""Rows whose mask leaves no token: no draft stays on one, greedy or drawn, whichever token it is and however the row lies in memory."""

from __future__ import annotations

import math

import pytest
import torch

from unicache_b200 import kernels, verify_drafts

from .gpu_util import need_gpu
from .test_verify_drafts_gpu import check, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 3, 64, 1003, 5001])
@pytest.mark.parametrize("shift", [0, 1, 3, 8])
def test_a_draft_on_a_row_without_a_token_falls(dtype, vocab, shift):
    need_gpu()
    seqs, n = 8, 3
    inside, _, uniforms, _ = inputs(seqs, n, vocab, dtype=dtype, probs=None, seed=vocab)
    wide = torch.zeros(seqs, n + 1, vocab + 16, device="cuda", dtype=dtype)
    logits = wide[:, :, shift:shift + vocab]  # row starts at every alignment of 16 bytes
    logits.copy_(inside)
    drafts = logits[:, :n].float().argmax(-1)
    for s in range(seqs):
        logits[s, s % (n + 1)] = -math.inf
        if s % (n + 1) < n:
            drafts[s, s % (n + 1)] = [0, vocab - 1][s // 4]
    heat = torch.tensor([0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 1.0], device="cuda")
    tokens, accepted, logprobs = check(logits, drafts, uniforms * 0.0, None, heat)
    assert accepted.tolist() == [0, 1, 2, 3] * 2
    for s in range(seqs):
        assert tokens[s].tolist() == drafts[s, :s % 4].tolist() + [-1] * (4 - s % 4)
    # a row that has no token is nobody's best, all rows' lowest numbers are ordinary ones
    logits.fill_(torch.finfo(dtype).min)
    drafts.zero_()
    tokens, accepted, logprobs = verify_drafts(logits, drafts, uniforms, temperature=0.0)
    assert accepted.tolist() == [n] * seqs and not tokens.any() and kernels.device_status() == 0
    # below 16: the logarithm is off by a unit of 2^-20 at most, its rounding and that of the expectation by half of one each
    assert torch.allclose(logprobs, torch.full_like(logprobs, -math.log(vocab)), rtol=0, atol=2.0 ** -19)
