"""Sequences that are taken back behind blocks that they share, and grow again: no other sequence's rows change."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from oracle.block_pool import Pool
from unicache_b200 import BlockPool, kernels

from .gpu_util import host, need_gpu
from .test_block_pool_gpu import fill, ints, same_contents, same_state, snapshot
from .test_block_pool_serving_gpu import restored

pytestmark = pytest.mark.gpu


class Served:
    """A pool with the oracle beside it and the rows that each sequence was given."""

    def __init__(self, seqs, width, blocks, block, *, heads=2, dim=64, dtype=torch.bfloat16, layers=2, seed=0):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.block, self.dtype, self.shape = block, dtype, (heads, dim)
        self.pool, self.shadow = BlockPool.allocate(seqs, width * block, blocks, block_size=block), Pool(seqs, width, blocks, block)
        self.layers = [self.pool.cache(num_kv_heads=heads, head_dim=dim, dtype=dtype) for _ in range(layers)]
        self.rows = [[torch.empty(0, heads, dim, dtype=dtype) for _ in range(2 * layers)] for _ in range(seqs)]
        self.old_scale = [False] * seqs  # rows were withdrawn from the last block and none written since
        kernels.device_status()

    def lengths(self):
        return [len(r[0]) for r in self.rows]

    def append(self, counts, size=1.0):
        starts = ints([0, *np.cumsum(counts).tolist()])
        self.advance(counts)
        new = [(size * torch.randn(sum(counts), *self.shape, generator=self.gen, device="cuda")).to(self.dtype)
               for _ in range(2 * len(self.layers))]
        for i, layer in enumerate(self.layers):
            layer.write(new[2 * i], new[2 * i + 1], starts=starts)
        at = 0
        for s, n in enumerate(counts):
            if n:
                self.rows[s] = [torch.cat((old, x[at:at + n].cpu())) for old, x in zip(self.rows[s], new)]
                self.old_scale[s] = False
            at += n

    def advance(self, counts):
        self.pool.advance(ints(counts))
        self.shadow.advance(counts)

    def back(self, counts):
        self.advance([-n for n in counts])
        for s, n in enumerate(counts):
            self.rows[s] = [x[:len(x) - n] for x in self.rows[s]]
            self.old_scale[s] |= n > 0

    def fork(self, parent, child):
        self.pool.fork(ints([parent]), ints([child]))
        self.shadow.fork([parent], [child])
        self.rows[child], self.old_scale[child] = list(self.rows[parent]), self.old_scale[parent]

    def release(self, s):
        self.pool.release(ints([s]))
        self.shadow.release([s])
        self.rows[s], self.old_scale[s] = [x[:0] for x in self.rows[s]], False

    def check(self):
        assert not self.shadow.refused
        same_state(self.pool, self.shadow)
        lengths = self.lengths()
        assert lengths == self.shadow.lengths
        if not sum(lengths):
            return
        starts = ints([0, *np.cumsum(lengths).tolist()])
        settled = torch.cat([torch.arange(n) < (n // self.block * self.block if old else n) for n, old in zip(lengths, self.old_scale)])
        for i, layer in enumerate(self.layers):
            for got, x in zip(layer.read(sum(lengths), starts=starts), (2 * i, 2 * i + 1)):
                want = torch.cat([restored(host(r[x]), self.block, self.dtype) for r in self.rows if len(r[0])])
                assert torch.equal(got.cpu()[settled], want[settled])


@pytest.mark.parametrize("block,dim,dtype", [(16, 64, torch.float16), (64, 128, torch.bfloat16), (128, 64, torch.bfloat16)])
@pytest.mark.parametrize("who", [0, 1])
@pytest.mark.parametrize("whole,inside,kept", [(2, 0, 1), (2, 0, 0), (1, 36, 0), (3, 5, 2), (3, 5, 0), (1, 0, 0)])
def test_the_other_sequence_keeps_its_rows(block, dim, dtype, who, whole, inside, kept):
    """A prompt of `whole` blocks and `inside` 64ths of one, forked; one of the two goes back to `kept` blocks and on from there with
    larger rows, one at a time, then many."""

    need_gpu()
    served = Served(3, 8, 20, block, dim=dim, dtype=dtype)
    prompt = whole * block + inside * block // 64
    served.append([prompt, 0, 0])
    served.fork(0, 1)
    served.check()
    back = [0, 0, 0]
    back[who] = prompt - kept * block
    served.back(back)
    served.check()
    one, many = [0, 0, 0], [0, 0, 0]
    one[who], many[who] = 1, block + 3
    served.append(one, 4.0)
    served.check()
    served.append(one, 2.0)
    served.append(many, 8.0)
    served.check()
    served.append([1, 1, 0], 3.0)  # and both
    served.check()


def test_both_go_back_and_grow_in_one_call():
    need_gpu()
    served = Served(4, 6, 30, 16)
    served.append([48, 0, 20, 0])
    served.fork(0, 1)
    served.fork(0, 3)
    served.back([32, 32, 0, 48])
    served.append([7, 20, 1, 33], 4.0)
    served.check()
    served.release(2)
    served.append([1, 1, 40, 1], 2.0)
    served.check()


@pytest.mark.parametrize("block,dim,dtype,seed", [(16, 64, torch.bfloat16, 0), (32, 128, torch.float16, 1), (16, 128, torch.bfloat16, 2),
                                                  (64, 64, torch.bfloat16, 3)])
def test_any_order_with_lengths_taken_back_to_earlier_blocks(block, dim, dtype, seed):
    """As a serving loop, and sequences go back to any block's end or to nothing, shared or not."""

    need_gpu()
    rng = random.Random(seed)
    seqs, width = 6, 6
    served = Served(seqs, width, 40, block, dim=dim, dtype=dtype, seed=seed)
    given_back = 0
    for step in range(120):
        kind = rng.choice(["append", "append", "prompts", "back", "back", "fork", "release", "compact"])
        lengths = served.lengths()
        if kind in ("append", "prompts"):
            most = 1 if kind == "append" else 2 * block
            held = [len(r) for r in served.shadow.rows]
            counts = [rng.randint(0, min(most, width * block - n)) * rng.randint(0, 1) for n in lengths]
            served.append(counts, rng.choice([0.3, 1.0, 3.0]))
            given_back += sum(n % block == 0 and c > 0 and n // block < h for n, c, h in zip(lengths, counts, held))
        elif kind == "back":
            served.back([rng.choice([0, 0, n % block, n % block + block * rng.randint(0, n // block), n]) for n in lengths])
        elif kind == "fork":
            served.fork(*rng.sample(range(seqs), 2))
        elif kind == "release" and rng.random() < 0.5:
            served.release(rng.randrange(seqs))
        else:
            assert served.pool.compact().tolist() == [served.shadow.compact()]
        if step % 2 == 0:
            served.check()
    served.check()
    assert given_back > 0


@pytest.mark.parametrize("seqs,blocks", [(40, 500), (4096, 20000), (300, 70001)])
def test_many_sequences_give_back_at_once(seqs, blocks):
    """One prompt shared by all, who go back and grow in the same calls; pools of one and of several CTAs."""

    need_gpu()
    block, width = 16, 4
    pool, oracle = BlockPool.allocate(seqs, width * block, blocks, block_size=block), Pool(seqs, width, blocks, block)
    cache = pool.cache(num_kv_heads=1, head_dim=64)
    fill(cache, 7)
    kernels.device_status()
    rng = random.Random(seqs)
    before = snapshot([cache])

    def both(tokens):
        pool.advance(ints(tokens))
        oracle.advance(tokens)
        same_state(pool, oracle)

    both([3 * block] + [0] * (seqs - 1))
    children = list(range(1, seqs))
    pool.fork(ints([0] * len(children)), ints(children))
    oracle.fork([0] * len(children), children)
    same_state(pool, oracle)
    for _ in range(3):
        both([-block * rng.randint(0, n // block) if n % block == 0 else 0 for n in oracle.lengths])
        both([rng.randint(0, 2 * block) if n <= 2 * block else 0 for n in oracle.lengths])
    assert not oracle.refused
    same_contents([cache], before, oracle)
