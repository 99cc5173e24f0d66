"""The drafted decode over a block pool: the operators together, as a serving step runs them."""

from __future__ import annotations

import pytest
import torch

from oracle.verify import verify
from unicache_b200 import kernels
from unicache_b200.workloads import DraftDecode

from .gpu_util import host, need_gpu
from .test_block8_gpu import check_attention

pytestmark = pytest.mark.gpu

SHAPE = dict(prompts=[100, 61, 129], new_tokens=90, samples=3, drafts=3, vocab=1500, seed=5)


def renew(*models, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    fresh = torch.rand(models[0].uniforms.shape, generator=gen, device="cuda")
    for m in models:
        m.uniforms.copy_(fresh)


@pytest.mark.parametrize("temperature", [1.0, 0.0])
def test_captured_steps_equal_eager_ones_and_the_oracle(temperature):
    need_gpu()
    kernels.device_status()
    eager, captured = (DraftDecode("cuda", **SHAPE, temperature=temperature) for _ in range(2))
    stayed, lengths = 0, eager.pool.lengths.tolist()
    assert lengths == SHAPE["prompts"] * 3
    for step in range(20):  # across block ends of every sequence
        renew(eager, captured, seed=step)
        tokens, accepted, logprobs = eager.step()
        got = captured.step() if step == 0 else captured.replay()
        assert torch.equal(got[0], tokens) and torch.equal(got[1], accepted) and torch.equal(got[2], logprobs)
        if step == 0:
            captured.capture()
        # what stays of the drafts is what the logits say
        r = eager.result
        for s in range(tokens.shape[0]):
            count = int(r["counts"][s])
            assert count == min(3, 63 - lengths[s] % 64)
            want = verify(host(r["logits"][s]), r["drafts"][s].tolist(), eager.uniforms[s, 3:].tolist(), host(r["probs"][s]),
                          temperature, count)
            if want[4][0] > 1e-5 and want[4][1] > 1e-12:
                assert tokens[s].tolist() == want[0].tolist() and int(accepted[s]) == want[1]
        lengths = [n + a + 1 for n, a in zip(lengths, accepted.tolist())]
        assert eager.pool.lengths.tolist() == lengths == captured.pool.lengths.tolist()
        stayed += int(accepted.sum())
    assert stayed < 20 * 3 * 9 and (stayed > 0 or temperature == 0)  # heads that learnt nothing do not hit the arg max
    assert kernels.device_status() == 0  # no write was refused: no draft was withdrawn over a block's end
    for a, b in zip(eager.caches, captured.caches):
        for name in ("key_code", "key_scale", "value_code", "value_scale", "key_low", "key_high"):
            assert torch.equal(getattr(a, name), getattr(b, name))
    # every sequence has its rows, and its blocks are its own but for the prompt's complete ones
    used = [-(-n // 64) for n in lengths]
    assert all(h >= u for h, u in zip(eager.pool.held.tolist(), used))
    shared = [n // 64 for n in SHAPE["prompts"]]
    assert sorted(eager.pool.references.tolist(), reverse=True)[:sum(shared) + 1] == [3] * sum(shared) + [1]


def test_attention_goes_on_after_sequences_end():
    need_gpu()
    kernels.device_status()
    model = DraftDecode("cuda", **SHAPE)
    for step in range(6):
        renew(model, seed=step)
        model.step()
    query = torch.randn(9, 8, 64, device="cuda").to(torch.bfloat16)
    before, _ = check_attention(model.caches[1], query, model.pool.lengths.tolist())
    model.finish(torch.tensor([0, 4, 8], dtype=torch.int32, device="cuda"))
    lengths = model.pool.lengths.tolist()
    assert [n == 0 for n in lengths] == [i in (0, 4, 8) for i in range(9)]
    live = int((model.pool.references > 0).sum())
    assert (model.pool.references[:live] > 0).all() and model.pool.free_blocks() == model.pool.num_blocks - live
    after, _ = check_attention(model.caches[1], query, lengths)
    stay = [1, 2, 3, 5, 6, 7]
    assert torch.allclose(after[stay].float(), before[stay].float(), atol=2e-2) and (after[[0, 4, 8]] == 0).all()
    # the ended ones' places are taken by forks, which go on
    model.pool.fork(torch.tensor([1, 1, 7], dtype=torch.int32, device="cuda"), torch.tensor([0, 4, 8], dtype=torch.int32, device="cuda"))
    for step in range(6, 12):
        renew(model, seed=step)
        tokens, accepted, _ = model.step()
        assert (tokens[:, 0] >= 0).all()
    assert kernels.device_status() == 0


def test_forked_sequences_are_the_prompt_s():
    need_gpu()
    model = DraftDecode("cuda", **SHAPE)
    query = torch.randn(3, 8, 64, device="cuda").to(torch.bfloat16)
    for cache in model.caches:
        out, _ = cache.attention(query.repeat(3, 1, 1))
        check_attention(cache, query.repeat(3, 1, 1), SHAPE["prompts"] * 3)
        # the same rows: sums in another order at most
        for i in (1, 2):
            assert torch.allclose(out[3 * i:3 * i + 3].float(), out[:3].float(), atol=1e-2)
