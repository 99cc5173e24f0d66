"""Pools whose free blocks are ranked by several CTAs, beside kernels of another stream that keep the multiprocessors busy, so that
the CTAs of a call do not begin together."""

from __future__ import annotations

import random

import pytest
import torch

from oracle.block_pool import Pool
from unicache_b200 import BlockPool, kernels

from .gpu_util import need_gpu
from .test_block_pool_gpu import ints, same_state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("blocks", [16385, 40000, 131073])
def test_calls_beside_a_busy_stream(blocks):
    need_gpu()
    seqs, width, block = 16, blocks // 20, 16
    pool, oracle = BlockPool.allocate(seqs, width * block, blocks, block_size=block), Pool(seqs, width, blocks, block)
    pool.cache(num_kv_heads=1, head_dim=64)
    kernels.device_status()
    rng, busy = random.Random(blocks), torch.cuda.Stream()
    x = torch.randn(2048, 2048, device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    for _ in range(8):
        tokens = [rng.randint(0, min(40 * block, width * block - n)) for n in oracle.lengths]
        ends = [rng.randrange(seqs) for _ in range(3)]
        with torch.cuda.stream(busy):
            for _ in range(20):
                x @ x
        pool.advance(ints(tokens))
        live = pool.compact()
        pool.release(ints(ends))
        again = pool.compact()
        oracle.advance(tokens)
        assert live.tolist() == [oracle.compact()]
        oracle.release(ends)
        assert again.tolist() == [oracle.compact()]
        same_state(pool, oracle)
    torch.cuda.synchronize()
