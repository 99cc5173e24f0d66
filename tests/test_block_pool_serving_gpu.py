"""A serving loop over a block pool against the rows themselves: after any order of prompts, appended tokens, withdrawn drafts, forks, ends
and compactions, every sequence's restored rows are the quantisation of the rows that it was given."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from oracle import block8 as oracle
from oracle.block_pool import Pool
from unicache_b200 import BlockPool, kernels

from .gpu_util import host, need_gpu

pytestmark = pytest.mark.gpu


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def restored(rows, block, dtype):
    """Rows [n, H, D] (float32) block by block in 8 bits and back, as the cache restores them."""

    out = np.empty_like(rows)
    for at in range(0, len(rows), block):
        part = rows[at:at + block]
        for h in range(rows.shape[1]):
            codes, scale = oracle.quantise(part[:, h])
            out[at:at + block, h] = codes.astype(np.float32) * scale
    return torch.from_numpy(out).to(dtype)


@pytest.mark.parametrize("block,dim,dtype,seed", [(16, 64, torch.bfloat16, 0), (32, 128, torch.float16, 1), (16, 128, torch.bfloat16, 2)])
def test_any_order_of_serving_calls(block, dim, dtype, seed):
    need_gpu()
    kernels.device_status()
    rng, gen = random.Random(seed), torch.Generator(device="cuda").manual_seed(seed)
    seqs, width, blocks, heads = 6, 6, 40, 2
    pool, shadow = BlockPool.allocate(seqs, width * block, blocks, block_size=block), Pool(seqs, width, blocks, block)
    layers = [pool.cache(num_kv_heads=heads, head_dim=dim, dtype=dtype) for _ in range(2)]
    rows = [[torch.empty(0, heads, dim, dtype=dtype) for _ in range(4)] for _ in range(seqs)]  # keys and values of both layers
    lowest = [0] * seqs  # how far a sequence may be taken back
    old_scale = [False] * seqs  # rows were withdrawn from the last block and none written since: it has its old scale still

    def append(counts):
        starts = ints([0, *np.cumsum(counts).tolist()])
        pool.advance(ints(counts))
        shadow.advance(counts)
        new = [(torch.randn(sum(counts), heads, dim, generator=gen, device="cuda") * rng.choice([0.3, 1.0, 3.0])).to(dtype) for _ in range(4)]
        for i, layer in enumerate(layers):
            layer.write(new[2 * i], new[2 * i + 1], starts=starts)
        at = 0
        for s, n in enumerate(counts):
            if n:
                for x in range(4):
                    rows[s][x] = torch.cat((rows[s][x], new[x][at:at + n].cpu()))
                lowest[s], old_scale[s] = (len(rows[s][0]) - 1) // block * block, False
            at += n

    for step in range(120):
        kind = rng.choice(["append", "append", "prompts", "withdraw", "fork", "release", "compact"])
        lengths = [len(r[0]) for r in rows]
        room = [width * block - n for n in lengths]
        if kind == "append":
            append([min(1, r) * rng.randint(0, 1) for r in room])
        elif kind == "prompts":
            append([rng.randint(0, min(r, 2 * block)) if rng.random() < 0.3 else 0 for r in room])
        elif kind == "withdraw":
            back = [-rng.randint(0, max(0, n - low)) for n, low in zip(lengths, lowest)]
            pool.advance(ints(back))
            shadow.advance(back)
            for s, n in enumerate(back):
                rows[s], old_scale[s] = [x[:len(x) + n] for x in rows[s]], old_scale[s] or n < 0
        elif kind == "fork":
            children = rng.sample(range(seqs), rng.randint(1, 3))
            parents = [rng.choice([s for s in range(seqs) if s not in children]) for _ in children]
            pool.fork(ints(parents), ints(children))
            shadow.fork(parents, children)
            for p, c in zip(parents, children):
                rows[c], old_scale[c] = list(rows[p]), old_scale[p]
                # complete blocks are shared from now on: neither goes back into them
                whole = len(rows[p][0]) // block * block
                lowest[p], lowest[c] = max(lowest[p], whole), whole
        elif kind == "release":
            ends = [s for s in range(seqs) if rng.random() < 0.3]
            pool.release(ints(ends))
            shadow.release(ends)
            for s in ends:
                rows[s], lowest[s], old_scale[s] = [x[:0] for x in rows[s]], 0, False
        else:
            assert pool.compact().tolist() == [shadow.compact()]
        assert not shadow.refused and kernels.device_status() == 0
        assert pool.block_table.tolist() == shadow.table() and pool.references.tolist() == shadow.references()
        total = sum(len(r[0]) for r in rows)
        if total and step % 3 == 0:
            starts = ints([0, *np.cumsum([len(r[0]) for r in rows]).tolist()])
            settled = torch.cat([torch.arange(len(r[0])) < (len(r[0]) // block * block if old else len(r[0])) for r, old in zip(rows, old_scale)])
            for i, layer in enumerate(layers):
                for got, x in zip(layer.read(total, starts=starts), (2 * i, 2 * i + 1)):
                    want = torch.cat([restored(host(r[x]), block, dtype) for r in rows if len(r[0])])
                    assert torch.equal(got.cpu()[settled], want[settled]), (step, kind)
    assert sum(len(r[0]) for r in rows) > 0
