"""What a refused write of the 8-bit block cache leaves out, and that it writes the rest."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import block8 as oracle
from unicache_b200 import kernels

from .gpu_util import host, need_gpu
from .test_block8_gpu import check_contents, filled, make_rows, split, starts_of

pytestmark = pytest.mark.gpu

FIELDS = ("key_code", "value_code", "key_scale", "value_scale", "key_low", "key_high")


def same(a, b):
    return torch.equal(a.view(torch.int8), b.view(torch.int8))


def check_block(cache, page, rows, name):
    """The first rows of one pool block against the oracle."""

    for h in range(cache.num_kv_heads):
        codes, scale = oracle.quantise(rows[:, h])
        np.testing.assert_array_equal(host(getattr(cache, name + "_scale"))[page, h], scale)
        np.testing.assert_array_equal(host(getattr(cache, name + "_code"))[page, h, :len(rows)], codes)


@pytest.mark.parametrize("broken", [0, 2, 4])
@pytest.mark.parametrize("entry", [-1, 1 << 30])
def test_a_block_outside_the_pool_is_skipped_and_the_others_written(broken, entry):
    """A write of the sequence's blocks 0 to 4, one of them nowhere."""

    need_gpu()
    block, before, counts = 16, [5, 9], [4 * 16, 70]
    cache, key0, value0, gen = filled(before, block=block, heads=2, width=6)
    rows = {m: make_rows(gen, counts, 2, 128, torch.bfloat16) for m in ("key", "value")}
    whole = {m: [np.concatenate(p) for p in zip(split(old, before), split(rows[m], counts))]
             for m, old in (("key", key0), ("value", value0))}
    page = int(cache.block_table[0, broken])
    was = {n: getattr(cache, n)[page].clone() for n in FIELDS}
    table = host(cache.block_table).copy()
    cache.block_table[0, broken] = entry
    cache.advance(torch.tensor(counts, dtype=torch.int32, device="cuda"))
    assert kernels.device_status() == 0
    cache.write(rows["key"], rows["value"], starts=starts_of(counts))
    assert kernels.device_status() & 2
    for n in FIELDS:
        assert same(getattr(cache, n)[page], was[n]), n
    for m in whole:
        for j in range(5):
            if j != broken:
                check_block(cache, table[0, j], whole[m][0][j * block:(j + 1) * block], m)
    # the other sequence as a whole
    cache.lengths[0] = 0
    check_contents(cache, [0, sum((before[1], counts[1]))], whole["key"], whole["value"])


@pytest.mark.parametrize("starts,written", [([0, 4, 2, 3], [2]), ([-1, 1, 2, 3], [1, 2]), ([0, 1, 2, 4], [0, 1]),
                                            ([2, 1, 2, 3], [1, 2])])
def test_a_malformed_range_skips_its_sequence(starts, written):
    need_gpu()
    lengths = [70, 70, 70]
    cache, key, value, gen = filled(lengths, width=2)
    old = {"key": split(key, lengths), "value": split(value, lengths)}
    rows = {m: make_rows(gen, [3], 4, 128, torch.bfloat16) for m in old}
    was = {n: getattr(cache, n).clone() for n in (*FIELDS, "pending_key", "pending_value")}
    begin = torch.tensor(starts, dtype=torch.int32, device="cuda")
    cache.advance(1)
    assert kernels.device_status() == 0
    cache.write(rows["key"], rows["value"], starts=begin)
    assert kernels.device_status() & 2
    table = cache.block_table.long()
    for s in range(3):
        if s in written:
            new = {m: np.concatenate([old[m][s], host(rows[m][starts[s]:starts[s + 1]])]) for m in old}
            for m in new:
                check_block(cache, int(table[s, 1]), new[m][64:], m)
        else:
            for n in FIELDS:
                assert same(getattr(cache, n)[table[s]], was[n][table[s]]), (s, n)
            for n in ("pending_key", "pending_value"):
                assert same(getattr(cache, n)[s], was[n][s]), (s, n)


@pytest.mark.parametrize("length", [129, 1 << 30, 0, -5])
def test_a_length_that_cannot_be_skips_its_sequence(length):
    need_gpu()
    lengths = [70, 70, 70]
    cache, key, value, gen = filled(lengths, width=2)
    old = {"key": split(key, lengths), "value": split(value, lengths)}
    rows = {m: make_rows(gen, [3], 4, 128, torch.bfloat16) for m in old}
    was = {n: getattr(cache, n).clone() for n in (*FIELDS, "pending_key", "pending_value")}
    cache.advance(1)
    cache.lengths[1] = length
    cache.write(rows["key"], rows["value"])
    assert kernels.device_status() & 2
    table = cache.block_table.long()
    for n in FIELDS:
        assert same(getattr(cache, n)[table[1]], was[n][table[1]]), n
    for n in ("pending_key", "pending_value"):
        assert same(getattr(cache, n)[1], was[n][1]), n
    for s in (0, 2):
        for m in old:
            check_block(cache, int(table[s, 1]), np.concatenate([old[m][s], host(rows[m][s:s + 1])])[64:], m)


def test_a_block_without_its_earlier_rows_is_skipped_and_the_later_ones_written():
    need_gpu()
    block = 16
    cache, key, value, gen = filled([14], block=block, heads=2, width=6)
    draft = make_rows(gen, [5], 2, 128, torch.bfloat16)
    cache.advance(5)
    cache.write(draft, draft, starts=starts_of([5]))
    cache.advance(-4)  # 15 rows: the block before the last one written
    page = int(cache.block_table[0, 0])
    was = {n: getattr(cache, n)[page].clone() for n in FIELDS}
    rows = make_rows(gen, [40], 2, 128, torch.bfloat16)
    cache.advance(40)
    assert kernels.device_status() == 0
    cache.write(rows, rows, starts=starts_of([40]))
    assert kernels.device_status() & 2
    for n in FIELDS:
        assert same(getattr(cache, n)[page], was[n]), n
    new = host(rows)
    for j in (1, 2, 3):
        for m in ("key", "value"):
            check_block(cache, int(cache.block_table[0, j]), new[16 * j - 15:min(40, 16 * j + 1)], m)
    more = make_rows(gen, [1], 2, 128, torch.bfloat16)
    cache.advance(1)
    cache.write(more, more)
    check_block(cache, int(cache.block_table[0, 3]), np.concatenate([new[33:], host(more)]), "key")
    assert kernels.device_status() == 0
