"""Attention over the 8-bit block cache where the work is split over the whole chip: tables of more tokens than
one block of threads takes alone, so that pairs cross warps and blocks of threads and their states are merged.
Every element type, head size, number of query rows and block size, against the float64 oracle."""

from __future__ import annotations

import pytest
import torch

from unicache_b200 import Int8BlockCache, kernels, sparse_int8_block_decode

from .gpu_util import need_gpu
from .test_block8_gpu import check_attention, check_select, filled, make_cache, make_query, make_rows, starts_of

pytestmark = pytest.mark.gpu

CAPACITY = 4500  # tokens of a sequence that the tables here have room for
EDGES = [0, 1, 15, 16, 17, 64, 65, 127, 129, 1000, 4500, 333, 2047]


def wide(block):
    return -(-CAPACITY // block)


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("hq,heads,dim", [(28, 4, 128), (40, 2, 128), (8, 8, 64), (24, 2, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_single_tokens_over_ragged_lengths(block, hq, heads, dim, dtype):
    need_gpu()
    cache, _, _, gen = filled(EDGES, heads=heads, dim=dim, block=block, dtype=dtype, seed=block + hq, width=wide(block))
    check_attention(cache, make_query(gen, (len(EDGES), hq, dim), dtype), EDGES)


@pytest.mark.parametrize("queries", [2, 5, 16])
@pytest.mark.parametrize("hq,heads,dim,block,dtype", [(28, 4, 128, 64, torch.float16), (4, 4, 64, 32, torch.bfloat16),
                                                      (16, 1, 128, 16, torch.bfloat16), (6, 2, 64, 16, torch.float16)])
def test_several_tokens_are_causal_and_may_see_none(queries, hq, heads, dim, block, dtype):
    need_gpu()
    lengths = [0, 1, 2, 5, 16, 17, 64, 70, 300, 1300, 2500]
    cache, _, _, gen = filled(lengths, heads=heads, dim=dim, block=block, dtype=dtype, seed=queries, width=wide(block))
    check_attention(cache, make_query(gen, (len(lengths), queries, hq, dim), dtype), lengths)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_strided_queries_and_scales(dtype):
    need_gpu()
    lengths = [100, 3257]
    cache, _, _, gen = filled(lengths, seed=8, dtype=dtype)
    q = make_query(gen, (2, 3, 36, 131), dtype)
    check_attention(cache, q[:, :, 4:32, 1:129], lengths)
    check_attention(cache, q[:, 1, 4:32, :128].transpose(0, 1).contiguous().transpose(0, 1), lengths)
    for scale in (0.31, 0.0, -0.1):
        check_attention(cache, q[:, 1, 4:32, 3:], lengths, scale=scale)
    check_attention(cache, q[:, 2, 4:32, :128] * 60, lengths)
    check_attention(cache, torch.zeros_like(q[:, 2, 4:32, :128]), lengths)
    if dtype is torch.bfloat16:
        check_attention(cache, q[:, 2, 4:32, :128] * 1e-30, lengths)
        check_attention(cache, q[:, 2, 4:32, :128] * 1e30, lengths, scale=1e-31)


@pytest.mark.parametrize("hq,dim,block", [(14, 128, 64), (32, 128, 16), (14, 64, 32), (32, 64, 32)])
def test_block_scales_of_very_different_size(hq, dim, block):
    need_gpu()
    lengths = [6400, 1]
    cache, gen = make_cache(lengths, heads=2, dim=dim, block=block)
    key, value = (make_rows(gen, lengths, 2, dim, torch.bfloat16) for _ in range(2))
    factors = torch.tensor([1e-6, 1e4, 1.0, 0.0, 1e-3, 1e6, 1e-9, 30.0, 0.0, 1e2], device="cuda").repeat(10)
    factors = torch.cat([factors.repeat_interleave(64), factors[:1]])[:, None, None]
    value = (value.float() * factors).to(torch.bfloat16)
    key = (key.float() * factors.clamp(1e-3, 2.0)).to(torch.bfloat16)
    cache.advance(torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    cache.write(key, value, starts=starts_of(lengths))
    check_attention(cache, make_query(gen, (2, hq, dim), torch.bfloat16), lengths)


@pytest.mark.parametrize("queries", [1, 4])
@pytest.mark.parametrize("dim,block,dtype", [(128, 64, torch.bfloat16), (64, 32, torch.float16), (128, 16, torch.float16)])
def test_selected_blocks_only(queries, dim, block, dtype):
    need_gpu()
    lengths = [4480, 64, 1, 0, 2000]
    cache, _, _, gen = filled(lengths, dim=dim, block=block, dtype=dtype, seed=9, width=wide(block))
    count = 1536 // block
    blocks = torch.full((5, 4, count), -1, dtype=torch.int32, device="cuda")
    for s, n in enumerate(lengths):
        for h in range(4):
            held = -(-n // block)
            some = torch.randperm(held, generator=gen, device="cuda")[:count - h].to(torch.int32)  # any order
            at = torch.randperm(count, generator=gen, device="cuda")[:some.numel()]                # gaps
            blocks[s, h, at] = some
    blocks[1, 3] = 64 // block + 1  # past the end: no tokens
    query = make_query(gen, (5, queries, 28, dim), dtype)
    check_attention(cache, query, lengths, blocks=blocks)
    check_attention(cache, query, lengths, blocks=torch.full_like(blocks, -1))


@pytest.mark.parametrize("dim,dtype", [(128, torch.bfloat16), (64, torch.float16)])
def test_sparse_decode_is_selection_then_attention(dim, dtype):
    need_gpu()
    lengths = [4400, 900, 10]
    cache, _, _, gen = filled(lengths, dim=dim, dtype=dtype, seed=14)
    query = make_query(gen, (3, 28, dim), dtype)
    blocks, out, lse = sparse_int8_block_decode(query, cache, count=33)
    assert torch.equal(blocks, cache.select(query, count=33))
    expect = cache.attention(query, blocks=blocks)
    assert torch.equal(out, expect[0]) and torch.equal(lse, expect[1])
    check_attention(cache, query, lengths, blocks=blocks)


@pytest.mark.parametrize("dim,block,dtype", [(128, 64, torch.bfloat16), (64, 32, torch.float16)])
@pytest.mark.parametrize("queries", [1, 3])
def test_poison_comes_through_the_merges(queries, dim, block, dtype):
    """A NaN and infinities in single blocks of a sequence whose heads are split over many blocks of threads show
    in the heads that see them and in no other."""

    need_gpu()
    lengths = [15000, 300, 7000]
    cache, gen = make_cache(lengths, dim=dim, block=block, dtype=dtype)
    key, value = (make_rows(gen, lengths, 4, dim, dtype) for _ in range(2))
    key[9000, 1, 5] = float("nan")       # sequence 0
    value[14999, 2, 3] = float("inf")    # its last token
    value[15310, 0, 3] = float("nan")    # sequence 2, first block
    key[20000, 3, 0] = float("inf")
    cache.advance(torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    cache.write(key, value, starts=starts_of(lengths))
    query = make_query(gen, (3, queries, 28, dim), dtype)
    out, lse = cache.attention(query)
    bad = out.isnan().any(-1).view(3, queries, 4, 7)
    # whether a row of several sees the poisoned last block goes by the tokens that it sees
    last = [n for n in range(queries) if lengths[0] - queries + 1 + n > (lengths[0] - 1) // block * block]
    expect = torch.zeros_like(bad)
    expect[0, :, 1] = True
    expect[0, last, 2] = True
    expect[2, :, 0] = True
    expect[2, :, 3] = True
    assert torch.equal(bad, expect)
    nan_lse = lse.isnan().view(3, queries, 4, 7)
    keys = torch.zeros_like(bad)
    keys[0, :, 1] = True
    keys[2, :, 3] = True
    assert torch.equal(nan_lse, keys) and not lse.isinf().any()
    assert kernels.device_status() == 0


def test_many_sequences_of_one_block_and_a_long_one():
    need_gpu()
    lengths = [(i * 37) % 91 for i in range(700)]
    lengths[333] = 4400
    cache, _, _, gen = filled(lengths, heads=2, dim=64, block=32, seed=6, dtype=torch.float16)
    check_attention(cache, make_query(gen, (700, 6, 64), torch.float16), lengths)


def test_code_offsets_past_32_bits():
    need_gpu()
    heads, dim, block = 8, 128, 128
    blocks, width, lengths = (1 << 31) // (heads * dim * block) + 40, 12, [1400, 1536]

    def empty(*shape, dtype):
        return torch.empty(shape, device="cuda", dtype=dtype)

    table = torch.arange(blocks - 2 * width, blocks, device="cuda", dtype=torch.int32).flip(0).view(2, width).contiguous()
    table[0, 1], table[1, 3], table[1, 11] = 0, blocks // 2, 5
    cache = Int8BlockCache(
        key_code=empty(blocks, heads, block, dim, dtype=torch.int8), key_scale=empty(blocks, heads, dtype=torch.float32),
        key_low=empty(blocks, heads, dim, dtype=torch.int8), key_high=empty(blocks, heads, dim, dtype=torch.int8),
        value_code=empty(blocks, heads, block, dim, dtype=torch.int8),
        value_scale=empty(blocks, heads, dtype=torch.float32),
        pending_key=torch.zeros(2, heads, block, dim, device="cuda", dtype=torch.bfloat16),
        pending_value=torch.zeros(2, heads, block, dim, device="cuda", dtype=torch.bfloat16), block_table=table,
        lengths=torch.zeros(2, device="cuda", dtype=torch.int32))
    small, gen = make_cache([width * block] * 2, heads=heads, dim=dim, block=block)
    key, value = (make_rows(gen, lengths, heads, dim, torch.bfloat16) for _ in range(2))
    query = make_query(gen, (2, 16, 128), torch.bfloat16)
    results = []
    for c in (cache, small):
        c.advance(torch.tensor(lengths, dtype=torch.int32, device="cuda"))
        c.write(key, value, starts=starts_of(lengths))
        results.append((*c.read(sum(lengths), starts=starts_of(lengths)), *c.attention(query),
                        *sparse_int8_block_decode(query, c, count=9, recent=1)))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    check_attention(small, query, lengths)


@pytest.mark.parametrize("hq,heads,dtype", [(28, 4, torch.bfloat16), (20, 1, torch.float16)])
@pytest.mark.parametrize("blocks,count", [(300, 40), (5000, 1000)])
def test_selection_by_clusters_at_128_channels(blocks, count, hq, heads, dtype):
    """One to eight blocks of threads a pair, one pass over the heads or three."""

    need_gpu()
    for distinct in (False, True):
        lengths = [16 * blocks - 7, 16 * (blocks // 3), 16 * count + 1]
        cache, gen = make_cache([16 * blocks] * 3, heads=heads, dim=128, block=16, dtype=dtype, seed=count)
        cache.lengths.copy_(torch.tensor(lengths))
        shape = cache.key_low.shape
        pick = torch.randint(0, 128 if distinct else 3, shape if distinct else (*shape[:2], 1), generator=gen, device="cuda")
        cache.key_high.copy_(pick.expand(shape))
        cache.key_low.copy_((-pick.flip(0)).expand(shape))
        cache.key_scale.copy_(torch.rand(shape[:2], generator=gen, device="cuda") if distinct
                              else torch.full(shape[:2], 0.5))
        check_select(cache, make_query(gen, (3, hq, 128), dtype), lengths, count=count)
