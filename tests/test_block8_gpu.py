"""The 8-bit block cache: writes and restored rows bit for bit, selections exactly, and
attention within derived bounds of the float64 oracle."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import block8 as oracle
from unicache_b200 import (Int8BlockCache, int8_block_decode, kernels, merge_attention_summaries,
                           sparse_int8_block_decode)

from .gpu_util import host, need_gpu

pytestmark = pytest.mark.gpu

# attention: the output's rounding (half a unit in the last place), then the weights, held in fp16
# where they multiply the values: a relative 2^-11 of each term, so of the weighted mean magnitude of
# the values, doubled for weights below the fp16 normal range and for fp32 sums.
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make_cache(lengths, *, heads=4, dim=128, block=64, dtype=torch.bfloat16, seed=0, spare=3, width=None):
    """A cache with shuffled blocks whose unused rows, scales and bounds are garbage."""

    gen = torch.Generator(device="cuda").manual_seed(seed)
    width = width or max(1, -(-max(lengths) // block))
    seqs, blocks = len(lengths), len(lengths) * width + spare

    def codes(*shape):
        return torch.randint(-127, 128, shape, generator=gen, device="cuda").to(torch.int8)

    table = torch.randperm(blocks, generator=gen, device="cuda")[:seqs * width].to(torch.int32).view(seqs, width)
    cache = Int8BlockCache(
        key_code=codes(blocks, heads, block, dim), key_scale=torch.full((blocks, heads), float("nan"), device="cuda"),
        key_low=codes(blocks, heads, dim), key_high=codes(blocks, heads, dim),
        value_code=codes(blocks, heads, block, dim), value_scale=torch.full((blocks, heads), float("nan"), device="cuda"),
        pending_key=torch.full((seqs, heads, block, dim), float("nan"), device="cuda", dtype=dtype),
        pending_value=torch.full((seqs, heads, block, dim), float("nan"), device="cuda", dtype=dtype),
        block_table=table, lengths=torch.zeros(seqs, device="cuda", dtype=torch.int32))
    return cache, gen


def starts_of(counts):
    return torch.tensor([0, *np.cumsum(counts)], dtype=torch.int32, device="cuda")


def make_rows(gen, counts, heads, dim, dtype, spread=0.8):
    rows = torch.randn(sum(counts), heads, dim, generator=gen, device="cuda")
    block_means = torch.randn(sum(counts) // 16 + 1, heads, dim, generator=gen, device="cuda")
    return (rows + spread * block_means.repeat_interleave(16, 0)[:sum(counts)]).to(dtype)


def filled(lengths, *, heads=4, dim=128, block=64, dtype=torch.bfloat16, seed=0, **more):
    cache, gen = make_cache(lengths, heads=heads, dim=dim, block=block, dtype=dtype, seed=seed, **more)
    key, value = (make_rows(gen, lengths, heads, dim, dtype) for _ in range(2))
    cache.advance(torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    cache.write(key, value, starts=starts_of(lengths))
    return cache, key, value, gen


def check_contents(cache, lengths, keys, values):
    """Codes, scales, bounds and pending rows against the oracle, from all rows of every sequence."""

    block = cache.block_size
    fields = {n: host(getattr(cache, n)) for n in ("key_code", "key_scale", "key_low", "key_high", "value_code",
                                                  "value_scale", "pending_key", "pending_value")}
    table = host(cache.block_table)
    for s, n in enumerate(lengths):
        for j in range(-(-n // block)):
            page = table[s, j]
            for h in range(cache.num_kv_heads):
                for name, rows in (("key", keys[s]), ("value", values[s])):
                    part = rows[j * block:min(n, (j + 1) * block), h]
                    codes, scale = oracle.quantise(part)
                    np.testing.assert_array_equal(fields[name + "_scale"][page, h], scale)
                    np.testing.assert_array_equal(fields[name + "_code"][page, h, :len(part)], codes)
                    if name == "key":
                        np.testing.assert_array_equal(fields["key_low"][page, h], codes.min(0))
                        np.testing.assert_array_equal(fields["key_high"][page, h], codes.max(0))
                    if len(part) < block:
                        np.testing.assert_array_equal(fields["pending_" + name][s, h, :len(part)], part)


def split(rows, counts):
    at = np.cumsum([0, *counts])
    return [host(rows[a:b]) for a, b in zip(at, at[1:])]


# ---------------------------------------------------------------- writing and reading
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,dim,dtype", [(4, 128, torch.bfloat16), (3, 64, torch.float16), (1, 128, torch.float16)])
def test_prompts_then_single_tokens_then_chunks(block, heads, dim, dtype):
    """Ragged prompts (empty ones too), then rows one at a time across block ends, then ragged chunks:
    always the quantisation of all rows so far."""

    need_gpu()
    counts = [0, 1, block - 1, block, block + 1, 3 * block + 5]
    cache, gen = make_cache([c + 8 * block for c in counts], heads=heads, dim=dim, block=block, dtype=dtype, seed=block)
    held = {"key": [np.zeros((0, heads, dim), np.float32) for _ in counts],
            "value": [np.zeros((0, heads, dim), np.float32) for _ in counts]}
    lengths = np.zeros(len(counts), int)

    def add(n, use_starts=True):
        nonlocal lengths
        rows = {name: make_rows(gen, n, heads, dim, dtype) * torch.rand((), generator=gen, device="cuda") * 3
                for name in held}
        rows = {name: r.to(dtype) for name, r in rows.items()}
        cache.advance(torch.tensor(n, dtype=torch.int32, device="cuda"))
        cache.write(rows["key"], rows["value"], starts=starts_of(n) if use_starts else None)
        for name in held:
            held[name] = [np.concatenate([a, b]) for a, b in zip(held[name], split(rows[name], n))]
        lengths = lengths + np.array(n)

    add(counts)
    check_contents(cache, lengths, held["key"], held["value"])
    for _ in range(block // 4 + 2):
        add([1] * len(counts), use_starts=False)
    check_contents(cache, lengths, held["key"], held["value"])
    add([block + 3, 0, 2 * block, 1, block - 1, 5])
    check_contents(cache, lengths, held["key"], held["value"])
    back = [int(n) for n in lengths]
    key, value = cache.read(sum(back), starts=starts_of(back))
    for got, rows in ((key, held["key"]), (value, held["value"])):
        at = 0
        for s, n in enumerate(back):
            expect = np.zeros((n, heads, dim), np.float32)
            for j in range(0, n, block):
                for h in range(heads):
                    codes, scale = oracle.quantise(rows[s][j:j + block, h])
                    expect[j:j + block, h] = codes.astype(np.float32) * scale
            expect = torch.from_numpy(expect).to(dtype)
            assert torch.equal(got[at:at + n].cpu(), expect)
            at += n
    few = [min(n, 3) for n in back]
    part, _ = cache.read(sum(few), starts=starts_of(few))
    at, to = np.cumsum([0, *few]), np.cumsum(back)
    for s, n in enumerate(few):
        assert torch.equal(part[at[s]:at[s] + n], key[to[s] - n:to[s]])
    assert kernels.device_status() == 0


def test_strided_and_unaligned_rows():
    need_gpu()
    lengths = [70, 129]
    cache, gen = make_cache(lengths)
    flat = torch.randn(199 * 9 * 131 + 1, generator=gen, device="cuda").to(torch.bfloat16)
    wide = flat[1:].view(199, 9, 131)
    key, value = wide[:, 1:5, :128], wide[:, 5:9, 3:]
    cache.advance(torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    cache.write(key, value, starts=starts_of(lengths))
    check_contents(cache, lengths, split(key, lengths), split(value, lengths))
    other, _ = make_cache(lengths)
    other.advance(torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    major = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (key, value)]
    other.write(*major, starts=starts_of(lengths))
    check_contents(other, lengths, split(key, lengths), split(value, lengths))


def test_values_at_the_edges_of_the_codes():
    """Ties between codes, zeros, the smallest and the largest numbers, infinities and NaN."""

    need_gpu()
    lengths = [64] * 6
    cache, gen = make_cache(lengths, heads=1)
    rows = torch.randn(6, 64, 1, 128, generator=gen, device="cuda")
    rows[0] = torch.randint(-254, 255, (64, 1, 128), generator=gen, device="cuda") / 2.0  # halves: ties
    rows[0, 0, 0, 0] = 127.0
    rows[1] = 0
    rows[2] *= 1e-38
    rows[3] *= 5e37
    rows[4, 3, 0, 7] = float("inf")
    rows[5, 60, 0, 1] = float("nan")
    rows = rows.to(torch.bfloat16).flatten(0, 1)
    cache.advance(64)
    cache.write(rows, rows, starts=starts_of(lengths))
    check_contents(cache, lengths, split(rows, lengths), split(rows, lengths))
    key, _ = cache.read(384, starts=starts_of(lengths))
    assert key[256:].isnan().all() and not key[:256].isnan().any()
    # row by row, the same
    other, _ = make_cache(lengths, heads=1)
    for t in range(64):
        other.advance(1)
        row = rows.view(6, 64, 1, 128)[:, t]
        other.write(row, row)
    check_contents(other, lengths, split(rows, lengths), split(rows, lengths))


def test_from_dense_and_shared_tables():
    need_gpu()
    gen = torch.Generator(device="cuda").manual_seed(3)
    lengths = [100, 0, 64]
    keys = [make_rows(gen, [n], 2, 64, torch.float16) for n in lengths]
    values = [make_rows(gen, [n], 2, 64, torch.float16) for n in lengths]
    cache = Int8BlockCache.from_dense(keys, values, max_tokens=200, block_size=32)
    assert cache.max_tokens == 224 and cache.resident_bytes > cache.key_code.numel() * 2
    check_contents(cache, lengths, [host(k) for k in keys], [host(v) for v in values])
    layer = Int8BlockCache.allocate(3, 200, num_kv_heads=2, head_dim=64, block_size=32, dtype=torch.float16,
                                    block_table=cache.block_table, num_blocks=21, lengths=cache.lengths)
    cache.advance(1)  # counts for both
    rows = make_rows(gen, [3], 2, 64, torch.float16)
    cache.write(rows, rows)
    layer.write(rows, rows)
    assert cache.lengths.tolist() == [101, 1, 65] == layer.lengths.tolist()


def test_bad_tables_lengths_and_starts_are_flagged_and_write_nothing():
    need_gpu()
    for breakage in ("table", "table high", "length", "starts", "old"):
        cache, _, _, gen = filled([70, 70, 70], width=2)
        before = {n: getattr(cache, n).clone() for n in ("key_code", "value_code", "pending_key", "key_low")}
        rows = make_rows(gen, [3], 4, 128, torch.bfloat16)
        starts = starts_of([1, 1, 1])
        cache.advance(1)
        if breakage.startswith("table"):
            cache.block_table[1, 1] = -1 if breakage == "table" else cache.key_code.shape[0]
        elif breakage == "length":
            cache.lengths[1] = 129
        elif breakage == "starts":
            starts[1] = 4
        else:
            cache.lengths[1] = 0
        assert kernels.device_status() == 0
        cache.write(rows, rows, starts=starts)
        assert kernels.device_status() & 2, breakage
        table = cache.block_table.long()
        touched = [] if breakage == "starts" else [0, 2]  # the broken range spoils its neighbours too
        for name, was in before.items():
            now = getattr(cache, name)
            index = [1] if name.startswith("pending") else \
                [p for p in range(now.shape[0]) if p not in {int(table[s, 1]) for s in touched}]
            if breakage != "starts":
                assert torch.equal(now[index].view(torch.int8), was[index].view(torch.int8)), (breakage, name)
        cache.lengths.fill_(70)
        if breakage in ("table", "table high"):
            query = torch.randn(3, 28, 128, generator=gen, device="cuda").to(torch.bfloat16)
            cache.attention(query)
            assert kernels.device_status() & 2
            cache.select(query, count=4)
            assert kernels.device_status() & 2
            key, value = cache.read(3)
            assert kernels.device_status() & 2
            assert key[1].isnan().all() and value[1].isnan().all() and key[[0, 2]].isfinite().all()
    assert kernels.device_status() == 0


# ---------------------------------------------------------------- attention
def expect_attention(cache, query, lengths, blocks=None, scale=None):
    """float64 attention, and the bounds of the output and of the LSE."""

    q = host(query).astype(np.float64)
    q = q[:, None] if q.ndim == 3 else q
    seqs, n, hq, dim = q.shape
    scale = 1 / math.sqrt(dim) if scale is None else scale
    size, heads = cache.block_size, cache.num_kv_heads
    codes = {m: host(getattr(cache, m + "_code")) for m in ("key", "value")}
    scales = {m: host(getattr(cache, m + "_scale")).astype(np.float64) for m in ("key", "value")}
    table = host(cache.block_table)
    result = []
    for s, length in enumerate(lengths):
        keys, values, visible = [], [], []
        for h in range(heads):
            if blocks is None:
                chosen = np.arange(-(-length // size))
            else:
                chosen = np.array([b for b in host(blocks)[s, h] if 0 <= b < -(-length // size)], int)
            token = (chosen[:, None] * size + np.arange(size)).reshape(-1)
            inside = token < length
            pages = table[s, chosen]
            for m, into in (("key", keys), ("value", values)):
                into.append((codes[m][pages, h].astype(np.float64) * scales[m][pages, h][:, None, None]).reshape(-1, dim)[inside])
            visible.append(token[inside][None] < (length - n + 1 + np.arange(n))[:, None])
        out, lse, mean = oracle.attention(q[s], keys, values, scale, visible)
        # fp32 logits: a sum of D products off by D * 2^-24 of the sum of their magnitudes, and the
        # exponentials and sums by 2^-20; errors of the logits change the weights by as much
        group = hq // heads
        worst = np.zeros((n, hq))
        for h in range(hq):
            if len(keys[h // group]):
                worst[:, h] = (np.abs(q[s][:, h]) @ np.abs(keys[h // group]).T).max(-1) * abs(scale)
        lse_bound = (dim + 8) * 2.0 ** -24 * worst + 2.0 ** -20
        bound = np.abs(out) * HALF_ULP[query.dtype] * 1.01 + mean * (2.0 ** -10 + 2 * lse_bound[..., None]) + 2.0 ** -25
        result.append((out, lse, bound, lse_bound))
    result = tuple(np.stack(x) for x in zip(*result))
    return tuple(x[:, 0] for x in result) if query.dim() == 3 else result


def check_attention(cache, query, lengths, blocks=None, scale=None):
    out, lse = cache.attention(query, blocks=blocks, softmax_scale=scale)
    assert out.shape == query.shape and out.dtype == query.dtype and lse.shape == query.shape[:-1]
    eo, el, bound, lse_bound = expect_attention(cache, query, lengths, blocks, scale)
    got = host(out).astype(np.float64)
    assert np.isfinite(got).all()
    off = np.abs(got - eo) - bound
    assert (off <= 0).all(), f"output off by {off.max():.3e} more than its bound"
    gl = host(lse).astype(np.float64)
    empty = np.isneginf(el)
    assert np.array_equal(np.isneginf(gl), empty)
    assert (got[empty] == 0).all()
    off = np.abs(gl[~empty] - el[~empty]) - lse_bound[~empty] - np.abs(el[~empty]) * 2.0 ** -23
    assert off.size == 0 or (off <= 0).all(), f"LSE off by {off.max():.3e} more than its bound"
    assert kernels.device_status() == 0
    return out, lse


def make_query(gen, shape, dtype):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("hq,heads,dim,dtype", [(28, 4, 128, torch.bfloat16), (8, 8, 64, torch.float16),
                                                (5, 1, 128, torch.float16), (24, 2, 64, torch.bfloat16),
                                                (40, 2, 128, torch.bfloat16)])
def test_single_tokens_over_ragged_lengths(block, hq, heads, dim, dtype):
    need_gpu()
    lengths = [0, 1, 15, 16, 17, 63, 64, 65, 200, 1000, 127, 128, 129, 333]
    cache, _, _, gen = filled(lengths, heads=heads, dim=dim, block=block, dtype=dtype, seed=block + hq)
    check_attention(cache, make_query(gen, (len(lengths), hq, dim), dtype), lengths)


@pytest.mark.parametrize("queries", [1, 2, 3, 8, 16])
@pytest.mark.parametrize("hq,heads,dim", [(28, 4, 128), (4, 4, 64), (16, 1, 128)])
def test_several_tokens_are_causal_and_may_see_none(queries, hq, heads, dim):
    need_gpu()
    lengths = [0, 1, 2, 5, 16, 17, 64, 70, 300]  # shorter than the queries: their first rows see nothing
    cache, _, _, gen = filled(lengths, heads=heads, dim=dim, seed=queries)
    check_attention(cache, make_query(gen, (len(lengths), queries, hq, dim), torch.bfloat16), lengths)


def test_one_long_sequence_and_many_short_ones():
    need_gpu()
    cache, _, _, gen = filled([20011], seed=5)
    check_attention(cache, make_query(gen, (1, 28, 128), torch.bfloat16), [20011])
    lengths = [(i * 37) % 91 for i in range(600)]
    cache, _, _, gen = filled(lengths, heads=2, dim=64, block=16, seed=6)
    check_attention(cache, make_query(gen, (600, 6, 64), torch.bfloat16), lengths)
    lengths = [3000 if i == 7 else 2 for i in range(40)]
    cache, _, _, gen = filled(lengths, heads=8, dim=128, block=32, seed=7)
    check_attention(cache, make_query(gen, (40, 8, 128), torch.bfloat16), lengths)


def test_strided_queries_and_scales():
    need_gpu()
    lengths = [100, 257]
    cache, _, _, gen = filled(lengths, seed=8)
    wide = make_query(gen, (2, 3, 36, 131), torch.bfloat16)
    check_attention(cache, wide[:, :, 4:32, 1:129], lengths)
    flat = make_query(gen, (2 * 28 * 128 + 1,), torch.bfloat16)
    check_attention(cache, flat[1:].view(2, 28, 128), lengths)
    check_attention(cache, wide[:, 1, 4:32, :128].transpose(0, 1).contiguous().transpose(0, 1), lengths)
    check_attention(cache, wide[:, 1, 4:32, 3:], lengths, scale=0.31)
    check_attention(cache, wide[:, 1, 4:32, :128], lengths, scale=0.0)
    check_attention(cache, wide[:, 1, 4:32, :128], lengths, scale=-0.1)
    check_attention(cache, wide[:, 2, 4:32, :128] * 60, lengths)  # one token takes nearly all the weight
    check_attention(cache, wide[:, 2, 4:32, :128] * 1e-30, lengths)
    check_attention(cache, torch.zeros_like(wide[:, 2, 4:32, :128]), lengths)
    check_attention(cache, wide[:, 2, 4:32, :128] * 1e30, lengths, scale=1e-31)  # beyond fp16 and back


def test_block_scales_of_very_different_size():
    need_gpu()
    lengths = [640]
    cache, gen = make_cache(lengths, heads=2)
    key, value = (make_rows(gen, lengths, 2, 128, torch.bfloat16) for _ in range(2))
    factors = torch.tensor([1e-6, 1e4, 1.0, 0.0, 1e-3, 1e6, 1e-9, 30.0, 0.0, 1e2], device="cuda")
    value = (value.float() * factors.repeat_interleave(64)[:, None, None]).to(torch.bfloat16)
    key = (key.float() * factors.clamp(1e-3, 2.0).repeat_interleave(64)[:, None, None]).to(torch.bfloat16)
    cache.advance(640)
    cache.write(key, value, starts=starts_of(lengths))
    check_attention(cache, make_query(gen, (1, 14, 128), torch.bfloat16), lengths)


@pytest.mark.parametrize("queries", [1, 4])
def test_selected_blocks_only(queries):
    need_gpu()
    lengths = [1000, 64, 1, 0, 500]
    cache, _, _, gen = filled(lengths, seed=9)
    full = torch.full((5, 4, 7), -1, dtype=torch.int32)
    full[0, :, :7] = torch.tensor([0, 3, 4, 9, 11, 14, 15])
    full[0, 1, :7] = torch.tensor([15, -1, 2, -1, 7, 0, -1])  # any order, gaps
    full[1, 0, 6] = 0
    full[1, 1, 0] = 0
    full[2, :, 0] = 0
    full[4, 0] = torch.tensor([7, 6, 5, 4, 3, 2, 1])
    full[4, 2, 0] = 7
    full[4, 3, 0] = 14  # past the end: no tokens
    query = make_query(gen, (5, queries, 28, 128), torch.bfloat16)
    check_attention(cache, query, lengths, blocks=full.cuda())
    check_attention(cache, query, lengths, blocks=torch.full((5, 4, 1), -1, dtype=torch.int32, device="cuda"))
    every = torch.arange(16, dtype=torch.int32, device="cuda").expand(5, 4, 16).contiguous()
    out, lse = cache.attention(query, blocks=every)
    whole, whole_lse = cache.attention(query)
    check_attention(cache, query, lengths, blocks=every)
    assert torch.allclose(lse, whole_lse, rtol=1e-6, atol=1e-6)


def test_poisoned_blocks_show_and_stale_rows_do_not():
    need_gpu()
    lengths = [200, 200, 200]
    cache, gen = make_cache(lengths)
    rows = make_rows(gen, lengths, 4, 128, torch.bfloat16)
    key, value = rows.clone(), rows.clone()
    key[210, 1, 5] = float("nan")      # sequence 1, block 0, head 1
    value[430, 2, 3] = float("inf")    # sequence 2, block 0, head 2
    cache.advance(200)
    cache.write(key, value, starts=starts_of(lengths))
    query = make_query(gen, (3, 28, 128), torch.bfloat16)
    out, lse = cache.attention(query)
    bad = out.isnan().any(-1)
    assert not bad[0].any() and bad[1, 7:14].all() and not bad[1, :7].any() and not bad[1, 14:].any()
    assert bad[2, 14:21].all() and not bad[2, :14].any() and not bad[2, 21:].any()
    assert lse[2].isfinite().all() and lse[1, 7:14].isnan().all()
    assert out[0].isfinite().all()  # unused rows, blocks and scales are garbage (make_cache)


def test_poison_of_later_tokens_stays_out_of_earlier_rows():
    """Four tokens written at once, the last alone in its block with a NaN and an infinity: the rows
    before it do not see that block."""

    need_gpu()
    for block in (16, 64):
        lengths = [block * 3 + 1]
        cache, gen = make_cache(lengths, block=block)
        key, value = (make_rows(gen, lengths, 4, 128, torch.bfloat16) for _ in range(2))
        key[-1, 0, 3], value[-1, 1, 2], value[-1, 2, 9] = float("nan"), float("nan"), float("inf")
        cache.advance(lengths[0])
        cache.write(key, value, starts=starts_of(lengths))
        query = make_query(gen, (1, 4, 28, 128), torch.bfloat16)
        out, lse = cache.attention(query)
        clean, _, _, _ = filled([block * 3], block=block)
        clean.write(key[:-1], value[:-1], starts=starts_of([block * 3]))
        expect, expect_lse = clean.attention(query[:, :3])
        assert torch.allclose(out[:, :3].float(), expect.float(), atol=2e-2) and torch.allclose(lse[:, :3], expect_lse)
        assert out[0, 3, :21].isnan().any(-1).all() and out[0, 3, 21:].isfinite().all()


def test_code_offsets_past_32_bits():
    need_gpu()
    heads, dim, block = 8, 128, 128
    blocks = (1 << 31) // (heads * dim * block) + 40

    def empty(*shape, dtype):
        return torch.empty(shape, device="cuda", dtype=dtype)

    table = torch.tensor([[blocks - 1, 0, blocks - 7], [blocks // 2, blocks - 3, 5]], device="cuda", dtype=torch.int32)
    cache = Int8BlockCache(
        key_code=empty(blocks, heads, block, dim, dtype=torch.int8), key_scale=empty(blocks, heads, dtype=torch.float32),
        key_low=empty(blocks, heads, dim, dtype=torch.int8), key_high=empty(blocks, heads, dim, dtype=torch.int8),
        value_code=empty(blocks, heads, block, dim, dtype=torch.int8),
        value_scale=empty(blocks, heads, dtype=torch.float32),
        pending_key=empty(2, heads, block, dim, dtype=torch.bfloat16),
        pending_value=empty(2, heads, block, dim, dtype=torch.bfloat16), block_table=table,
        lengths=torch.zeros(2, device="cuda", dtype=torch.int32))
    small, gen = make_cache([300, 384], heads=heads, dim=dim, block=block)
    lengths = [300, 384]
    key, value = (make_rows(gen, lengths, heads, dim, torch.bfloat16) for _ in range(2))
    query = make_query(gen, (2, 16, 128), torch.bfloat16)
    results = []
    for c in (cache, small):
        c.advance(torch.tensor(lengths, dtype=torch.int32, device="cuda"))
        c.write(key, value, starts=starts_of(lengths))
        results.append((*c.read(684, starts=starts_of(lengths)), *c.attention(query), c.select(query, count=2, recent=1)))
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_summaries_merge_with_a_dense_part():
    """The cache's (out, lse) of one token combine with another part's through the framework's merge."""

    need_gpu()
    cache, key, value, gen = filled([300], seed=11)
    query = make_query(gen, (1, 28, 128), torch.bfloat16)
    front = torch.arange(3, dtype=torch.int32, device="cuda").expand(1, 4, 3).contiguous()
    back = torch.arange(3, 5, dtype=torch.int32, device="cuda").expand(1, 4, 2).contiguous()
    parts = [cache.attention(query, blocks=b) for b in (front, back)]
    merged, lse = merge_attention_summaries([(o, l.transpose(0, 1)) for o, l in parts])
    whole, whole_lse = int8_block_decode(query, cache)
    assert torch.allclose(lse.transpose(0, 1), whole_lse, atol=1e-5)
    assert torch.allclose(merged.float(), whole.float(), atol=2e-2)


# ---------------------------------------------------------------- selection
def check_select(cache, query, lengths, **how):
    got = host(cache.select(query, **how))
    fields = {n: host(getattr(cache, n)) for n in ("key_low", "key_high", "key_scale", "block_table")}
    for s, n in enumerate(lengths):
        pages = fields["block_table"][s, :-(-n // cache.block_size)]
        heads = range(cache.num_kv_heads)
        expect = oracle.select(host(query[s]), [fields["key_low"][pages, h] for h in heads],
                               [fields["key_high"][pages, h] for h in heads],
                               [fields["key_scale"][pages, h] for h in heads], how["count"], how.get("first", 1),
                               how.get("recent", 2))
        np.testing.assert_array_equal(got[s], expect)


@pytest.mark.parametrize("hq,heads,dim,block,dtype", [(28, 4, 128, 64, torch.bfloat16), (8, 8, 64, 16, torch.float16),
                                                      (32, 1, 128, 32, torch.bfloat16), (6, 2, 64, 128, torch.bfloat16)])
@pytest.mark.parametrize("count,first,recent", [(3, 1, 2), (8, 1, 2), (1, 0, 0), (4, 0, 4), (4, 4, 0), (40, 2, 3)])
def test_selection_is_exact(hq, heads, dim, block, dtype, count, first, recent):
    need_gpu()
    lengths = [0, 1, block, 3 * block, 3 * block + 1, 9 * block - 3, 33 * block + 5, 70 * block]
    cache, _, _, gen = filled(lengths, heads=heads, dim=dim, block=block, dtype=dtype, seed=count + hq)
    query = make_query(gen, (len(lengths), hq, dim), dtype)
    check_select(cache, query, lengths, count=count, first=first, recent=recent)


@pytest.mark.parametrize("blocks,count", [(1500, 64), (5000, 1000), (5000, 4096), (33000, 17)])
def test_selection_among_many_blocks(blocks, count):
    """Scores and bounds made directly; with few distinct values most scores are equal."""

    need_gpu()
    for distinct in (False, True):
        lengths = [16 * blocks - 7, 16 * (blocks // 3)]
        cache, gen = make_cache([16 * blocks] * 2, heads=2, dim=64, block=16, seed=count)
        cache.lengths.copy_(torch.tensor(lengths))
        shape = cache.key_low.shape
        if distinct:
            cache.key_high.copy_(torch.randint(0, 128, shape, generator=gen, device="cuda"))
            cache.key_low.copy_(-torch.randint(0, 128, shape, generator=gen, device="cuda"))
            cache.key_scale.copy_(torch.rand(shape[:2], generator=gen, device="cuda"))
        else:
            pick = torch.randint(0, 3, shape[:2], generator=gen, device="cuda")[..., None]
            cache.key_high.copy_((pick * 10).expand(shape))
            cache.key_low.copy_((-pick * 10).expand(shape))
            cache.key_scale.fill_(0.5)
        check_select(cache, make_query(gen, (2, 8, 64), torch.bfloat16), lengths, count=count)


def test_selection_of_more_blocks_than_shared_memory_holds():
    need_gpu()
    blocks = 60000
    cache, gen = make_cache([16 * blocks], heads=1, dim=64, block=16, seed=1)
    cache.lengths.fill_(16 * blocks - 3)
    shape = cache.key_low.shape
    cache.key_high.copy_(torch.randint(0, 128, shape, generator=gen, device="cuda"))
    cache.key_low.copy_(-torch.randint(0, 128, shape, generator=gen, device="cuda"))
    cache.key_scale.copy_(torch.rand(shape[:2], generator=gen, device="cuda"))
    check_select(cache, make_query(gen, (1, 20, 64), torch.bfloat16), [16 * blocks - 3], count=300)


def test_selection_with_zeros_negatives_and_poison():
    need_gpu()
    lengths = [64 * 20] * 4
    cache, _, _, gen = filled(lengths, seed=13)
    query = make_query(gen, (4, 28, 128), torch.bfloat16)
    query[0] = 0  # every score is 0: the lowest blocks
    page = cache.block_table[1].long()
    cache.key_high[page] = -cache.key_high[page].abs()  # bounds below zero
    cache.key_low[page] = -127
    cache.key_scale[cache.block_table[2, 7].long(), 1] = float("nan")
    cache.key_scale[cache.block_table[2, 9].long()] = float("inf")
    query[3, 5, 0] = float("nan")
    check_select(cache, query, lengths, count=6)
    got = cache.select(query, count=6)
    assert 7 in got[2, 1].tolist() and 9 in got[2, 0].tolist()
    strided = torch.empty(4, 30, 130, device="cuda", dtype=torch.bfloat16)
    strided[:, 2:, 1:129] = query
    assert torch.equal(cache.select(strided[:, 2:, 1:129], count=6), got)


def test_sparse_decode_is_selection_then_attention():
    need_gpu()
    lengths = [3000, 900, 10]
    cache, _, _, gen = filled(lengths, seed=14)
    query = make_query(gen, (3, 28, 128), torch.bfloat16)
    blocks, out, lse = sparse_int8_block_decode(query, cache, count=9)
    assert torch.equal(blocks, cache.select(query, count=9))
    expect = cache.attention(query, blocks=blocks)
    assert torch.equal(out, expect[0]) and torch.equal(lse, expect[1])
    check_attention(cache, query, lengths, blocks=blocks)


# ---------------------------------------------------------------- streams, graphs, refusals
def test_another_stream_and_repeated_calls_agree():
    need_gpu()
    lengths = [5000, 77, 0, 1234]
    cache, _, _, gen = filled(lengths, seed=15)
    query = make_query(gen, (4, 28, 128), torch.bfloat16)
    first = (*cache.attention(query), cache.select(query, count=12))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        results = [(*cache.attention(query), cache.select(query, count=12)) for _ in range(20)]
    stream.synchronize()
    for r in results:
        for a, b in zip(first, r):
            assert torch.equal(a, b)


def test_a_captured_step_follows_the_lengths():
    """advance, write, select and attend as one CUDA graph, replayed across a block end."""

    need_gpu()
    lengths = [60, 130, 0]
    cache, _, _, gen = filled(lengths, seed=16, width=8)
    twin, _, _, _ = filled(lengths, seed=16, width=8)
    rows = [make_rows(gen, [3], 4, 128, torch.bfloat16) for _ in range(8)]
    queries = [make_query(gen, (3, 28, 128), torch.bfloat16) for _ in range(8)]
    key, value, query = rows[0].clone(), rows[0].clone(), queries[0].clone()

    def step(c, k, v, q):
        c.advance(1)
        c.write(k, v)
        return (*c.attention(q), *sparse_int8_block_decode(q, c, count=3))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        captured = step(cache, key, value, query)
    torch.cuda.current_stream().wait_stream(side)
    for k, q in zip(rows, queries):
        key.copy_(k), value.copy_(k * 2), query.copy_(q)
        graph.replay()
        for a, b in zip(captured, step(twin, k, k * 2, q)):
            assert torch.equal(a, b)
    assert cache.lengths.tolist() == [68, 138, 8] and kernels.device_status() == 0


def test_refusals():
    need_gpu()
    cache, _, _, gen = filled([100, 100], seed=17)
    query = make_query(gen, (2, 28, 128), torch.bfloat16)
    rows = make_rows(gen, [2], 4, 128, torch.bfloat16)
    for bad in (query[:1], query.half(), query[:, :27], query[..., :64], query.cpu(), query[:, None].expand(2, 17, 28, 128),
                query[0], query.transpose(1, 2).contiguous().transpose(1, 2)):
        with pytest.raises(ValueError):
            cache.attention(bad)
    for bad in (query[:, None], query.half(), query[:1]):
        with pytest.raises(ValueError):
            cache.select(bad, count=4)
    for how in ({"count": 0}, {"count": 2}, {"count": 4097}, {"count": 4, "first": -1}, {"count": 4, "recent": 4}):
        with pytest.raises(ValueError):
            cache.select(query, **how)
    for bad in (torch.zeros(2, 4, 3, device="cuda"), torch.zeros(2, 3, 3, device="cuda", dtype=torch.int32),
                torch.zeros(2, 4, 0, device="cuda", dtype=torch.int32), torch.zeros(2, 4, 3, dtype=torch.int32)):
        with pytest.raises(ValueError):
            cache.attention(query, blocks=bad)
    for k, v in ((rows[:1], rows[:1]), (rows, rows[:1]), (rows.half(), rows), (rows[:, :3], rows), (rows.cpu(), rows),
                 (rows[..., :64], rows)):
        with pytest.raises(ValueError):
            cache.write(k, v)
    with pytest.raises(ValueError):
        cache.write(rows, rows, starts=starts_of([1, 1]).long())
    with pytest.raises(ValueError):
        cache.read(5)
    with pytest.raises(AttributeError):
        cache.lengths = cache.lengths
    fields = {n: getattr(cache, n) for n in ("key_code", "key_scale", "key_low", "key_high", "value_code", "value_scale",
                                             "pending_key", "pending_value", "block_table", "lengths")}
    for name, bad in (("key_code", fields["key_code"][..., :96]), ("key_scale", fields["key_scale"].half()),
                      ("value_code", fields["value_code"][:1]), ("pending_key", fields["pending_key"].float()),
                      ("block_table", fields["block_table"].long()), ("lengths", fields["lengths"][:1]),
                      ("key_low", fields["key_low"].cpu())):
        with pytest.raises(ValueError):
            Int8BlockCache(**{**fields, name: bad})
    with pytest.raises(RuntimeError):
        Int8BlockCache(**{**fields, "key_code": fields["key_code"].cpu()})
    odd = torch.empty(fields["key_code"].numel() + 8, device="cuda", dtype=torch.int8)[8:].view(fields["key_code"].shape)
    with pytest.raises(ValueError, match="aligned"):
        Int8BlockCache(**{**fields, "key_code": odd})
    for how in ({"block_size": 48}, {"head_dim": 96}, {"num_blocks": 1}, {"dtype": torch.float32}):
        with pytest.raises(ValueError):
            Int8BlockCache.allocate(2, 100, **{"num_kv_heads": 4, **how})
    with pytest.raises(RuntimeError):
        Int8BlockCache.allocate(2, 100, num_kv_heads=4, device="cpu")
    with pytest.raises(ValueError):
        Int8BlockCache.from_dense([], [])
    assert cache.read(0, starts=starts_of([0, 0]))[0].shape == (0, 4, 128)
    cache.write(rows[:0], rows[:0], starts=starts_of([0, 0]))
    assert kernels.device_status() == 0
