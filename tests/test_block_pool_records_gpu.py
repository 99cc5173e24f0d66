"""A fork at a block's end leaves neither parent nor child the block's unquantised rows: a write into its middle is refused,
whatever the child was before, and everything else is written."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from unicache_b200 import BlockPool, kernels, verify_drafts

from .gpu_util import host, need_gpu
from .test_block_pool_gpu import BAD, CONTENTS, ints, same_bits
from .test_block_pool_serving_gpu import restored

pytestmark = pytest.mark.gpu

HEADS = 2


class Layers:
    def __init__(self, block, dim, dtype, seed):
        self.block, self.dim, self.dtype = block, dim, dtype
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.pool = BlockPool.allocate(3, 6 * block, 18, block_size=block)
        self.caches = [self.pool.cache(num_kv_heads=HEADS, head_dim=dim, dtype=dtype) for _ in range(2)]
        kernels.device_status()

    def append(self, sequence, n, size):
        """Rows of both layers to one sequence: key and value of each."""

        counts = [n if s == sequence else 0 for s in range(3)]
        self.pool.advance(ints(counts))
        rows = [(size * torch.randn(n, HEADS, self.dim, generator=self.gen, device="cuda")).to(self.dtype) for _ in range(4)]
        for i, cache in enumerate(self.caches):
            cache.write(rows[2 * i], rows[2 * i + 1], starts=ints([0, *np.cumsum(counts).tolist()]))
        return rows

    def back(self, sequence, n):
        self.pool.advance(ints([-n if s == sequence else 0 for s in range(3)]))

    def check(self, sequence, rows, begin=0):
        """The sequence's rows from `begin` (a block's start) on are the quantisation of those."""

        lengths = self.pool.lengths.tolist()
        starts = ints([0, *np.cumsum([n if s == sequence else 0 for s, n in enumerate(lengths)]).tolist()])
        for i, cache in enumerate(self.caches):
            for got, want in zip(cache.read(lengths[sequence], starts=starts), rows[2 * i:2 * i + 2]):
                assert len(want) == lengths[sequence]
                assert torch.equal(got.cpu()[begin:], restored(host(want), self.block, self.dtype)[begin:])


def joined(*parts):
    return [torch.cat(x) for x in zip(*parts)]


@pytest.mark.parametrize("block,dim,dtype", [(16, 64, torch.bfloat16), (64, 128, torch.float16), (128, 64, torch.bfloat16), (32, 128, torch.bfloat16)])
@pytest.mark.parametrize("earlier", ["none", "same block", "same block, complete", "later block", "fewer rows"])
@pytest.mark.parametrize("back", [1, 7, 15])
def test_a_write_into_the_middle_of_the_childs_last_block_is_refused(block, dim, dtype, earlier, back):
    need_gpu()
    layers = Layers(block, dim, dtype, block + back)
    if earlier != "none":  # the child's slot has had another life, whose record and rows lie there still
        size = {"same block": 2 * block - 1, "same block, complete": 2 * block, "later block": 2 * block + 5, "fewer rows": block + 1}[earlier]
        layers.append(1, size, 0.5)
        layers.pool.release(ints([1]))
    prompt = layers.append(0, 2 * block, 1.0)
    layers.pool.fork(ints([0]), ints([1]))
    assert layers.pool.held.tolist() == [2, 2, 0]
    layers.pool.release(ints([0]))  # the child's alone from now on
    layers.back(1, back)
    assert layers.pool.lengths.tolist() == [0, 2 * block - back, 0] and kernels.device_status() == 0
    page = int(layers.pool.block_table[1, 1])
    was = [{n: getattr(c, n)[page].clone() for n in CONTENTS} for c in layers.caches]
    more = layers.append(1, back + block + 3, 4.0)
    assert kernels.device_status() & BAD
    for cache, old in zip(layers.caches, was):
        for name, x in old.items():
            same_bits(getattr(cache, name)[page], x)
    # the blocks behind are written, and go on
    rows = joined([x[:2 * block - back] for x in prompt], more)
    layers.check(1, rows, 2 * block)
    rows = joined(rows, layers.append(1, 2, 8.0))
    layers.check(1, rows, 2 * block)
    # from the block's start there is a way forward
    layers.back(1, 2 * block + 5)
    rows = joined([x[:block] for x in rows], layers.append(1, 5, 2.0))
    layers.check(1, rows)
    layers.back(1, 2)
    rows = joined([x[:-2] for x in rows], layers.append(1, block, 3.0))
    layers.check(1, rows)
    assert kernels.device_status() == 0


@pytest.mark.parametrize("who", [0, 1, 2])
@pytest.mark.parametrize("verified", [False, True])
def test_nobody_writes_into_the_middle_of_a_block_shared_at_its_end(who, verified):
    """Drafts up to a block's end, forked before they are verified: the lengths go back into the shared block without the pool."""

    need_gpu()
    layers = Layers(16, 64, torch.bfloat16, who)
    rows = layers.append(0, 32, 1.0)
    layers.pool.fork(ints([0, 0]), ints([1, 2]))
    page = int(layers.pool.block_table[0, 1])
    was = [{n: getattr(c, n)[page].clone() for n in CONTENTS} for c in layers.caches]
    if verified:  # all greedy drafts fall
        logits = torch.zeros(3, 4, 50, device="cuda")
        logits[:, :, 7] = 1.0
        _, accepted, _ = verify_drafts(logits, ints([[1, 2, 3]] * 3), torch.rand(3, 4, device="cuda"), temperature=0.0,
                                       lengths=layers.pool.lengths)
        assert accepted.tolist() == [0, 0, 0]
    else:
        layers.pool.lengths.sub_(3)
    assert layers.pool.lengths.tolist() == [29] * 3 and kernels.device_status() == 0
    layers.append(who, 1, 5.0)
    assert kernels.device_status() & BAD
    for cache, old in zip(layers.caches, was):
        for name, x in old.items():
            same_bits(getattr(cache, name)[page], x)
    layers.back(who, 14)  # to the block's start
    mine = joined([x[:16] for x in rows], layers.append(who, 20, 5.0))
    assert layers.pool.held.tolist() == [2 + (s == who) for s in range(3)]
    layers.check(who, mine)
    for cache, old in zip(layers.caches, was):
        for name, x in old.items():
            same_bits(getattr(cache, name)[page], x)
    assert kernels.device_status() == 0


def test_a_parent_goes_on_behind_a_fork():
    """Rows, drafts taken back and further ones, as if it had not been forked."""

    need_gpu()
    layers = Layers(16, 64, torch.bfloat16, 1)
    rows = layers.append(0, 32, 1.0)
    layers.pool.fork(ints([0]), ints([2]))
    rows = joined(rows, layers.append(0, 6, 1.0))
    layers.back(0, 3)
    rows = joined([x[:35] for x in rows], layers.append(0, 9, 4.0))
    layers.check(0, rows)
    assert kernels.device_status() == 0


def test_a_child_of_a_child():
    need_gpu()
    layers = Layers(16, 128, torch.float16, 2)
    prompt = layers.append(0, 32, 1.0)
    layers.pool.fork(ints([0]), ints([1]))
    layers.pool.fork(ints([1]), ints([2]))
    layers.pool.release(ints([0, 1]))
    layers.back(2, 3)
    layers.append(2, 2, 4.0)
    assert kernels.device_status() & BAD
    layers.back(2, 31)
    layers.check(2, [x[:0] for x in prompt])
    layers.check(2, layers.append(2, 20, 1.0))
    assert kernels.device_status() == 0
