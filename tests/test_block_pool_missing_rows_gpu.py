"""Rows that a full pool had no block for: once there is one, the block's later rows are refused rather than put behind rows of an
earlier sequence or of drafts that were withdrawn; and a step that was taken back is made again."""

from __future__ import annotations

import pytest
import torch

from unicache_b200 import BlockPool, kernels

from .gpu_util import need_gpu
from .test_block_pool_gpu import BAD, CONTENTS, ints, same_bits
from .test_block_pool_records_gpu import Layers, joined

pytestmark = pytest.mark.gpu

KINDS = [(16, 64, torch.bfloat16), (64, 128, torch.float16), (128, 128, torch.bfloat16)]


def full(block, dim, dtype, seed, blocks=6):
    """Layers over a pool that sequence 2 can fill."""

    layers = Layers(block, dim, dtype, seed)
    layers.pool = BlockPool.allocate(3, 6 * block, blocks, block_size=block)
    layers.caches = [layers.pool.cache(num_kv_heads=2, head_dim=dim, dtype=dtype) for _ in range(2)]
    return layers


def refused(layers, sequence, n):
    page = layers.pool.block_table[sequence][layers.pool.block_table[sequence] >= 0].long()
    was = [{name: getattr(c, name)[page].clone() for name in CONTENTS} for c in layers.caches]
    assert kernels.device_status() == 0
    layers.append(sequence, n, 4.0)
    assert kernels.device_status() & BAD
    for cache, old in zip(layers.caches, was):
        for name, x in old.items():
            same_bits(getattr(cache, name)[page], x)


@pytest.mark.parametrize("block,dim,dtype", KINDS)
def test_an_earlier_sequences_rows_are_not_taken(block, dim, dtype):
    need_gpu()
    layers = full(block, dim, dtype, 1)
    layers.append(0, 10, 1.0)
    layers.pool.release(ints([0]))
    layers.append(2, 6 * block, 1.0)  # the whole pool
    assert kernels.device_status() == 0
    layers.append(0, 5, 1.0)
    assert kernels.device_status() & BAD and layers.pool.held.tolist() == [0, 0, 6]
    layers.pool.release(ints([2]))
    layers.pool.advance(ints([0, 0, 0]))  # a block for the five rows, which are lost
    assert layers.pool.held.tolist() == [1, 0, 0]
    refused(layers, 0, 1)
    layers.back(0, 6)
    layers.check(0, layers.append(0, block + 3, 1.0))
    assert kernels.device_status() == 0


@pytest.mark.parametrize("block,dim,dtype", KINDS)
def test_rows_withdrawn_before_are_not_taken(block, dim, dtype):
    need_gpu()
    layers = full(block, dim, dtype, 2)
    prompt = layers.append(0, 2 * block, 1.0)
    layers.pool.fork(ints([0]), ints([1]))
    layers.append(2, 4 * block, 1.0)
    layers.back(0, block)
    assert kernels.device_status() == 0
    layers.append(0, 5, 1.0)  # gives the shared block back; there is no other
    assert kernels.device_status() & BAD and layers.pool.held.tolist() == [1, 2, 4]
    layers.check(1, prompt)
    layers.pool.release(ints([2]))
    layers.pool.advance(0)
    assert layers.pool.held.tolist() == [2, 2, 0]
    refused(layers, 0, 1)
    layers.check(1, prompt)
    layers.back(0, 6)
    layers.check(0, joined([x[:block] for x in prompt], layers.append(0, 9, 2.0)))
    layers.check(1, prompt)
    assert kernels.device_status() == 0


@pytest.mark.parametrize("block,dim,dtype", KINDS)
@pytest.mark.parametrize("more", [1, 7])
def test_a_step_from_a_blocks_end_that_was_taken_back_is_made_again(block, dim, dtype, more):
    """And rows of the block in front may be withdrawn, which are there still."""

    need_gpu()
    layers = full(block, dim, dtype, 3 + more)
    rows = joined(layers.append(0, 2 * block - 1, 1.0), layers.append(0, 1, 3.0))
    layers.append(2, 4 * block, 1.0)
    assert kernels.device_status() == 0
    layers.append(0, more, 2.0)
    assert kernels.device_status() & BAD
    layers.back(0, more)
    layers.pool.release(ints([2]))
    layers.back(0, 3)
    rows = joined([x[:-3] for x in rows], layers.append(0, 3 + more, 4.0))
    layers.check(0, rows)
    assert kernels.device_status() == 0


@pytest.mark.parametrize("block,dim,dtype", KINDS)
@pytest.mark.parametrize("inside,more", [(1, 1), (4, 2), (9, 5), (4, 12)])
def test_a_step_from_inside_a_block_that_was_taken_back_is_made_again(block, dim, dtype, inside, more):
    """The step fills a block and needs another one that is not there."""

    need_gpu()
    layers = full(block, dim, dtype, inside)
    rows = [x[:2 * block - inside] for x in layers.append(0, 2 * block - 1, 1.0)]
    layers.back(0, inside - 1)
    layers.append(2, 4 * block, 1.0)
    assert kernels.device_status() == 0
    layers.append(0, inside + more, 2.0)
    assert kernels.device_status() & BAD
    layers.back(0, inside + more)
    layers.pool.release(ints([2]))
    rows = joined(rows, layers.append(0, inside + more, 4.0))
    layers.check(0, rows)
    # a step over several blocks, of which the last is missing
    layers.append(2, 2 * block, 1.0)
    rows = joined(rows, layers.append(0, block - more - 1, 0.5))
    assert kernels.device_status() == 0
    layers.append(0, block + 3, 8.0)
    assert kernels.device_status() & BAD and layers.pool.held.tolist() == [4, 0, 2]
    layers.back(0, block + 3)
    layers.pool.release(ints([2]))
    rows = joined(rows, layers.append(0, block + 3, 0.7))
    layers.check(0, rows)
    assert kernels.device_status() == 0
