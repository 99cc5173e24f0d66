"""The block pool against plain Python: table, lengths, references and contents after every call, bit for bit."""

from __future__ import annotations

import random

import pytest
import torch

from oracle.block_pool import Pool
from unicache_b200 import BlockPool, Int8BlockCache, int8_block_decode, kernels

from .gpu_util import need_gpu

pytestmark = pytest.mark.gpu

CONTENTS = ("key_code", "value_code", "key_scale", "value_scale", "key_low", "key_high")
BAD = 2  # the device error bit


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def fill(cache, seed):
    """Random contents, bit patterns rather than numbers where they are copied as they are."""

    gen = torch.Generator(device="cuda").manual_seed(seed)
    for name in ("key_code", "value_code", "key_low", "key_high"):
        x = getattr(cache, name)
        x.copy_(torch.randint(-128, 128, x.shape, generator=gen, device="cuda", dtype=torch.int8))
    for name in ("key_scale", "value_scale"):
        getattr(cache, name).uniform_(generator=gen)
    for name in ("pending_key", "pending_value"):
        x = getattr(cache, name)
        x.view(torch.int16).copy_(torch.randint(-32768, 32768, x.shape, generator=gen, device="cuda", dtype=torch.int16))


def snapshot(caches):
    return [{n: getattr(c, n).clone() for n in (*CONTENTS, "pending_key", "pending_value")} for c in caches]


def same_state(pool, oracle):
    assert pool.block_table.tolist() == oracle.table()
    assert pool.lengths.tolist() == oracle.lengths
    assert pool.references.tolist() == oracle.references()
    assert pool.held.tolist() == [len(r) for r in oracle.rows]
    assert bool(kernels.device_status() & BAD) == oracle.refused
    oracle.refused = False


def same_bits(a, b):
    as_ints = {1: torch.int8, 2: torch.int16, 4: torch.int32}[a.element_size()]
    assert torch.equal(a.view(as_ints), b.view(as_ints))


def same_contents(caches, before, oracle, forked=False, compacted=False):
    for cache, old in zip(caches, before):
        if forked:
            for source, target, parent, child, rows in oracle.copies:
                for name in ("key", "value"):
                    old[name + "_code"][target, :, :rows] = old[name + "_code"][source, :, :rows]
                    old[name + "_scale"][target] = old[name + "_scale"][source]
                    old["pending_" + name][child, :, :rows] = old["pending_" + name][parent, :, :rows]
                old["pending_key"][child, :, -1] = old["pending_key"][parent, :, -1]
                for name in ("key_low", "key_high"):
                    old[name][target] = old[name][source]
        if compacted:
            for name in CONTENTS:
                for source, target in oracle.moves.items():
                    old[name][target] = old[name][source]
        for name, x in old.items():
            same_bits(getattr(cache, name), x)


LAYERS = [dict(num_kv_heads=4, head_dim=128), dict(num_kv_heads=1, head_dim=64), dict(num_kv_heads=3, head_dim=64, dtype=torch.float16)]


@pytest.mark.parametrize("seqs,width,blocks,block,seed", [(1, 1, 1, 16, 0), (2, 3, 5, 128, 1), (7, 5, 23, 32, 2), (40, 9, 200, 16, 3),
                                                          (33, 6, 111, 64, 4), (5, 40, 201, 32, 5)])
def test_calls_in_any_order(seqs, width, blocks, block, seed):
    need_gpu()
    rng = random.Random(seed)
    pool, oracle = BlockPool.allocate(seqs, width * block - rng.randrange(block), blocks, block_size=block), Pool(seqs, width, blocks, block)
    caches = [pool.cache(**kind) for kind in LAYERS]
    for i, cache in enumerate(caches):
        fill(cache, seed * 10 + i)
    kernels.device_status()
    for step in range(60):
        before = snapshot(caches)
        kind = rng.choice(["advance", "advance", "release", "fork", "fork", "compact"])
        if kind == "advance" and rng.random() < 0.5:
            n = rng.choice([1, 1, 3, block, 0, -1])
            pool.advance(n)
            oracle.advance([n] * seqs)
        elif kind == "advance":
            room = [width * block - t for t in oracle.lengths]
            tokens = [rng.choice([0, 1, block, rng.randint(0, max(0, r)), -min(oracle.lengths[s], rng.randint(0, block))])
                      for s, r in enumerate(room)]
            pool.advance(ints(tokens))
            oracle.advance(tokens)
        elif kind == "release":
            ends = [rng.randrange(seqs) for _ in range(rng.randint(0, seqs))]  # some of them twice
            pool.release(ints(ends))
            oracle.release(ends)
        elif kind == "fork":
            n = rng.randint(0, seqs)
            parents, children = [rng.randrange(seqs) for _ in range(n)], rng.sample(range(seqs), n)
            if rng.random() < 0.5:  # well-formed pairs
                parents = [rng.choice([s for s in range(seqs) if s not in children] or [0]) for _ in children]
            pool.fork(ints(parents), ints(children))
            oracle.fork(parents, children)
        else:
            assert pool.compact().tolist() == [oracle.compact()]
        same_state(pool, oracle)
        same_contents(caches, before, oracle, forked=kind == "fork", compacted=kind == "compact")
    assert pool.free_blocks() == len(oracle.free())


@pytest.mark.parametrize("blocks", [32767, 32769, 70001, 300007])
def test_pools_of_more_blocks_than_one_cta_ranks(blocks):
    """Taken, shared and free blocks all over pools of 1 to 8 CTAs and of several rounds."""

    need_gpu()
    seqs, width, block = 24, blocks // 20, 16
    pool, oracle = BlockPool.allocate(seqs, width * block, blocks, block_size=block), Pool(seqs, width, blocks, block)
    cache = pool.cache(num_kv_heads=1, head_dim=64)
    fill(cache, 1)
    kernels.device_status()
    rng = random.Random(blocks)

    def check(kind=None):
        same_state(pool, oracle)
        same_contents([cache], before, oracle, kind == "fork", False)

    before = snapshot([cache])
    tokens = [rng.randint(0, width * block) for _ in range(seqs)]
    pool.advance(ints(tokens))
    oracle.advance(tokens)
    check()
    ends = [1, 4, 9, 17, 22]
    pool.release(ints(ends))
    oracle.release(ends)
    check()
    pool.advance(17)
    oracle.advance([17] * seqs)
    check()
    before = snapshot([cache])
    pool.fork(ints([0, 2, 0]), ints([1, 4, 9]))
    oracle.fork([0, 2, 0], [1, 4, 9])
    check("fork")
    pool.release(ints([3, 5]))
    oracle.release([3, 5])
    before = snapshot([cache])
    assert pool.compact().tolist() == [oracle.compact()]
    same_state(pool, oracle)
    for name in CONTENTS:
        old = before[0][name]
        source, target = (torch.tensor(list(x), device="cuda", dtype=torch.long) for x in (oracle.moves.keys(), oracle.moves.values()))
        old[target] = old[source]
        same_bits(getattr(cache, name), old)


def test_a_full_pool_leaves_entries_empty_and_recovers():
    need_gpu()
    pool, oracle = BlockPool.allocate(3, 64, 5, block_size=16), Pool(3, 4, 5, 16)
    cache = pool.cache(num_kv_heads=2, head_dim=64)
    kernels.device_status()
    for tokens in ([33, 20, 0], [16, 16, 10], [-16, -16, -10], [0, 0, 10]):
        pool.advance(ints(tokens))
        oracle.advance(tokens)
        same_state(pool, oracle)
    assert oracle.lengths == [33, 20, 10] and pool.block_table[2].tolist() == [-1] * 4
    pool.fork(ints([1]), ints([2]))  # no room for the incomplete block: the child is left empty
    oracle.fork([1], [2])
    assert oracle.refused and oracle.lengths[2] == 0
    same_state(pool, oracle)
    pool.advance(ints([-100, 0, 0]))  # below nothing
    oracle.advance([-100, 0, 0])
    assert oracle.refused and oracle.lengths[0] == 0
    same_state(pool, oracle)
    pool.advance(ints([65, 0, 0]))  # past the table
    oracle.advance([65, 0, 0])
    same_state(pool, oracle)
    pool.release(ints([0, 7, -1]))
    oracle.release([0, 7, -1])
    same_state(pool, oracle)
    pool.fork(ints([1, 9, 1]), ints([2, 0, -3]))
    oracle.fork([1, 9, 1], [2, 0, -3])
    assert oracle.refused and oracle.lengths == [0, 20, 20]
    same_state(pool, oracle)
    assert cache.num_seqs == 3


def test_no_length_goes_back_into_a_shared_block():
    need_gpu()
    pool, oracle = BlockPool.allocate(4, 64, 20, block_size=16), Pool(4, 4, 20, 16)
    pool.cache(num_kv_heads=2, head_dim=64)
    kernels.device_status()

    def both(tokens):
        pool.advance(ints(tokens))
        oracle.advance(tokens)
        same_state(pool, oracle)

    both([32, 40, 32, 0])
    pool.fork(ints([0, 1]), ints([3, 2]))  # at a block's end, and inside one
    oracle.fork([0, 1], [3, 2])
    both([-1, -1, -1, -1])  # 0 and 3 stay at 32, the others go back in blocks of their own
    assert oracle.lengths == [32, 39, 39, 32]
    both([-16, -9, 0, 5])  # to blocks' ends and further rows: 16 and 30 are refused or not by whom the block belongs to
    assert oracle.lengths == [16, 39, 39, 37]
    both([0, 0, 0, -3])
    assert oracle.lengths[3] == 34
    both([0, 0, 0, -4])  # 30: shared with sequence 0, which holds the block still
    assert oracle.lengths[3] == 34
    pool.release(ints([0, 2]))
    oracle.release([0, 2])
    both([0, -9, 0, -4])  # nobody shares them any more
    assert oracle.lengths == [0, 30, 0, 30]


def test_the_most_sequences():
    need_gpu()
    seqs, block = 4096, 16
    pool, oracle = BlockPool.allocate(seqs, 48, 9000, block_size=block), Pool(seqs, 3, 9000, block)
    cache = pool.cache(num_kv_heads=1, head_dim=64)
    fill(cache, 3)
    kernels.device_status()
    tokens = [(i * 37) % 40 for i in range(seqs)]
    pool.advance(ints(tokens))
    oracle.advance(tokens)
    same_state(pool, oracle)
    parents, children = [i % 1365 for i in range(2731)], list(range(1365, 4096))
    before = snapshot([cache])
    pool.fork(ints(parents), ints(children))
    oracle.fork(parents, children)
    same_state(pool, oracle)
    # targets and children are distinct: the copies of all pairs at once
    old = before[0]
    copies = torch.tensor(oracle.copies, device="cuda")
    rows = torch.arange(block, device="cuda")[None, None, :, None] < copies[:, 4, None, None, None]
    source, target, parent, child = (copies[:, i] for i in range(4))
    for name in ("key", "value"):
        codes, pending = old[name + "_code"], old["pending_" + name]
        codes[target] = torch.where(rows, codes[source], codes[target])
        kept = rows.clone()
        kept[:, :, -1] |= name == "key"
        pending[child] = torch.where(kept, pending[parent], pending[child])
        old[name + "_scale"][target] = old[name + "_scale"][source]
    for name in ("key_low", "key_high"):
        old[name][target] = old[name][source]
    for name, x in old.items():
        same_bits(getattr(cache, name), x)
    pool.release(torch.arange(seqs, device="cuda", dtype=torch.int32))
    assert pool.free_blocks() == 9000 and (pool.block_table == -1).all() and kernels.device_status() == 0


@pytest.mark.parametrize("block,dtype", [(16, torch.float16), (64, torch.bfloat16), (128, torch.bfloat16)])
def test_forked_sequences_go_on_as_their_own(block, dtype):
    """A forked sequence that is written to is bit for bit the one that was written alone, and its parent is unchanged."""

    need_gpu()
    heads, dim, prompt, more = 2, 64, 2 * block + 5, block
    gen = torch.Generator(device="cuda").manual_seed(block)

    def rows(n, size=1.0):
        return [(size * torch.randn(n, heads, dim, generator=gen, device="cuda")).to(dtype) for _ in range(2)]

    first, then = rows(prompt), [rows(1, 1.0 + 0.3 * i) for i in range(2 * more)]
    pool = BlockPool.allocate(3, 8 * block, 20, block_size=block)
    cache = pool.cache(num_kv_heads=heads, head_dim=dim, dtype=dtype)
    alone = Int8BlockCache.allocate(2, 8 * block, num_kv_heads=heads, head_dim=dim, block_size=block, dtype=dtype)
    pool.advance(ints([prompt, 0, 0]))
    cache.write(*first, starts=ints([0, prompt, prompt, prompt]))
    alone.advance(ints([prompt, prompt]))
    alone.write(torch.cat([first[0]] * 2), torch.cat([first[1]] * 2), starts=ints([0, prompt, 2 * prompt]))
    pool.fork(ints([0, 0]), ints([2, 1]))
    pool.release(ints([1]))  # and one that ends at once
    assert pool.references.tolist()[:4] == [2, 2, 1, 1]
    for i in range(more):
        a, b = then[2 * i], then[2 * i + 1]
        pool.advance(ints([1, 0, 1]))
        cache.write(torch.cat((a[0], b[0])), torch.cat((a[1], b[1])), starts=ints([0, 1, 1, 2]))
        alone.advance(1)
        alone.write(torch.cat((a[0], b[0])), torch.cat((a[1], b[1])))
        if i == more // 2:  # drafts withdrawn inside the block
            pool.advance(ints([0, 0, -2]))
            alone.advance(ints([0, -2]))
    total = alone.lengths.tolist()
    assert pool.lengths.tolist() == [total[0], 0, total[1]]
    got = cache.read(sum(total), starts=ints([0, total[0], total[0], sum(total)]))
    want = alone.read(sum(total), starts=ints([0, total[0], sum(total)]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    query = torch.randn(3, 4, dim, generator=gen, device="cuda").to(dtype)
    out, lse = int8_block_decode(query, cache)
    plain, plain_lse = int8_block_decode(query[[0, 2]].contiguous(), alone)
    assert torch.equal(out[[0, 2]], plain) and torch.equal(lse[[0, 2]], plain_lse)
    pool.compact()
    again, _ = int8_block_decode(query, cache)
    assert torch.equal(again, out) and kernels.device_status() == 0


def test_captured_calls_replay_on_the_state_of_their_time():
    need_gpu()
    seqs, width, blocks, block = 6, 8, 40, 16
    pool, oracle = BlockPool.allocate(seqs, width * block, blocks, block_size=block), Pool(seqs, width, blocks, block)
    caches = [pool.cache(num_kv_heads=2, head_dim=64) for _ in range(2)]
    for i, cache in enumerate(caches):
        fill(cache, i)
    ends, parents, children, tokens = ints([0]), ints([1]), ints([2]), ints([5] * seqs)
    kernels.device_status()

    def step():
        pool.advance(tokens)
        pool.fork(parents, children)
        pool.release(ends)
        return pool.compact()

    step()
    for calls in [(oracle.advance, [5] * seqs), (oracle.fork, [1], [2]), (oracle.release, [0]), (oracle.compact,)]:
        calls[0](*calls[1:])
    same_state(pool, oracle)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        live = step()
    torch.cuda.current_stream().wait_stream(stream)
    rng = random.Random(0)
    for _ in range(12):
        p, c, e = rng.sample(range(seqs), 3)
        t = [rng.randint(0, 9) for _ in range(seqs)]
        for x, v in ((ends, [e]), (parents, [p]), (children, [c]), (tokens, t)):
            x.copy_(ints(v))
        before = snapshot(caches)
        graph.replay()
        oracle.advance(t)
        oracle.fork([p], [c])
        oracle.release([e])
        assert live.tolist() == [oracle.compact()]
        same_state(pool, oracle)
        same_contents(caches, before, oracle, forked=True, compacted=True)


def test_a_captured_fork_outlives_a_later_attachment():
    need_gpu()
    pool, oracle = BlockPool.allocate(4, 64, 20, block_size=16), Pool(4, 4, 20, 16)
    cache = pool.cache(num_kv_heads=2, head_dim=64)
    fill(cache, 1)
    kernels.device_status()
    parents, children = ints([0]), ints([3])
    pool.advance(21)
    oracle.advance([21] * 4)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        pool.fork(parents, children)
    torch.cuda.current_stream().wait_stream(stream)
    later = pool.cache(num_kv_heads=4, head_dim=128)
    assert [torch.full((112 * i,), 255, device="cuda", dtype=torch.uint8).sum() for i in range(1, 40)]  # reuse what is free
    fill(later, 2)
    before = snapshot([cache, later])
    graph.replay()
    oracle.fork([0], [3])
    same_state(pool, oracle)
    same_contents([cache], before[:1], oracle, forked=True)
    oracle.copies = []
    same_contents([later], before[1:], oracle, forked=True)  # not of its time
    before = snapshot([cache, later])
    pool.fork(parents, children)
    oracle.fork([0], [3])
    same_state(pool, oracle)
    same_contents([cache, later], before, oracle, forked=True)


def test_another_stream():
    need_gpu()
    pool, oracle = BlockPool.allocate(4, 64, 20, block_size=16), Pool(4, 4, 20, 16)
    pool.cache(num_kv_heads=2, head_dim=64)
    kernels.device_status()
    parents, children = ints([0]), ints([3])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(5):
            pool.advance(7)
            pool.fork(parents, children)
    torch.cuda.current_stream().wait_stream(stream)
    for _ in range(5):
        oracle.advance([7] * 4)
        oracle.fork([0], [3])
    same_state(pool, oracle)


def test_bad_calls_are_refused():
    need_gpu()
    pool = BlockPool.allocate(4, 64, 20, block_size=16)
    with pytest.raises(ValueError, match="no caches"):
        pool.compact()
    with pytest.raises(ValueError, match="no caches"):
        pool.fork(ints([0]), ints([1]))
    cache = pool.cache(num_kv_heads=2, head_dim=64)
    for call in (lambda: pool.attach([cache]),
                 lambda: pool.attach([Int8BlockCache.allocate(4, 64, num_kv_heads=2, block_size=16)]),
                 lambda: pool.release([1]), lambda: pool.release(ints([1]).long()), lambda: pool.release(ints([[1]])),
                 lambda: pool.release(ints([1, 2, 3, 4])[::2]), lambda: pool.release(torch.zeros(1, dtype=torch.int32)),
                 lambda: pool.advance(ints([1, 2, 3])), lambda: pool.advance(1 << 31),
                 lambda: pool.fork(ints([0]), ints([1, 2])), lambda: pool.fork(ints([0] * 5), ints([1] * 5)),
                 lambda: BlockPool.allocate(0, 64, 20), lambda: BlockPool.allocate(4, 64, 20, block_size=48),
                 lambda: BlockPool.allocate(4097, 64, 20),
                 lambda: BlockPool(block_table=pool.block_table, lengths=pool.lengths[:3], references=pool.references, block_size=16),
                 lambda: BlockPool(block_table=pool.block_table.long(), lengths=pool.lengths, references=pool.references, block_size=16),
                 lambda: BlockPool(block_table=pool.block_table, lengths=pool.lengths, references=pool.references[1:], block_size=16)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        BlockPool(block_table=pool.block_table.cpu(), lengths=pool.lengths, references=pool.references, block_size=16)
    empty = ints([])
    pool.release(empty), pool.fork(empty, empty)  # nothing to do
    assert kernels.device_status() == 0 and pool.free_blocks() == 20
