"""The decode workload over 8-bit block caches: eager and captured steps agree, and a layer's attention is
the oracle's over the cache that the steps wrote."""

from __future__ import annotations

import pytest
import torch

from unicache_b200 import kernels
from unicache_b200.workloads import Int8BlockDecode

from .gpu_util import need_gpu
from .test_block8_gpu import check_attention

pytestmark = pytest.mark.gpu

SHAPE = dict(prompts=[700, 1, 64, 1290], new_tokens=80, layers=2, hidden=512, q_heads=14, kv_heads=2, seed=3)


@pytest.mark.parametrize("count", [None, 8])
def test_captured_steps_equal_eager_ones(count):
    need_gpu()
    eager, captured = (Int8BlockDecode("cuda", **SHAPE, count=count) for _ in range(2))
    first = [m.step().clone() for m in (eager, captured)]
    assert torch.equal(*first)
    captured.capture()
    for _ in range(70):  # across block ends of every sequence
        assert torch.equal(eager.step(), captured.replay())
    assert torch.isfinite(eager.x.float()).all()
    lengths = [n + 71 for n in SHAPE["prompts"]]
    for model in (eager, captured):
        assert all(c.lengths.tolist() == lengths for c in model.caches)
    for name in ("key_code", "key_scale", "value_code", "value_scale", "key_low", "key_high"):
        for a, b in zip(eager.caches, captured.caches):
            assert torch.equal(getattr(a, name), getattr(b, name))
    # the last layer's attention of the last step
    query, cache = eager.query, eager.caches[-1]
    blocks = None if count is None else cache.select(query, count=count)
    out, _ = check_attention(cache, query, lengths, blocks=blocks)
    assert torch.equal(out, eager.attended)
    assert kernels.device_status() == 0


def test_enough_blocks_make_sparse_steps_dense_ones():
    need_gpu()
    dense = Int8BlockDecode("cuda", **SHAPE)
    sparse = Int8BlockDecode("cuda", **SHAPE, count=22)  # 1370 tokens are 22 blocks
    for _ in range(3):
        a, b = dense.step(), sparse.step()
    # the same sums in another order, through two layers: bf16 roundings that fall the other way
    assert torch.allclose(a.float(), b.float(), atol=0.05, rtol=0.02)
