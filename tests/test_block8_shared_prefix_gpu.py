"""Sequences of the 8-bit block cache that have their first blocks in common, forked at a block's end and inside a block."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from unicache_b200 import kernels

from .gpu_util import host, need_gpu
from .test_block8_gpu import check_attention, check_contents, make_cache, make_query, make_rows, starts_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prefix", [128, 150])
def test_forks_share_complete_blocks_and_copy_the_last(prefix):
    need_gpu()
    block, spare = 64, 5
    cache, gen = make_cache([320, 320, 320], block=block, heads=2, spare=spare)
    sides = ("key", "value")
    first = {m: make_rows(gen, [prefix], 2, 128, torch.bfloat16) for m in sides}
    count = torch.tensor([prefix, 0, 0], dtype=torch.int32, device="cuda")
    cache.advance(count)
    cache.write(first["key"], first["value"], starts=starts_of([prefix, 0, 0]))
    # sequences 1 and 2 go on from sequence 0's tokens
    whole = prefix // block
    cache.block_table[1:, :whole] = cache.block_table[0, :whole]
    if prefix % block:
        page = cache.block_table[0, whole].long()
        for s in (1, 2):
            for n in ("key_code", "key_scale", "key_low", "key_high", "value_code", "value_scale"):
                tensor = getattr(cache, n)
                tensor[cache.block_table[s, whole].long()] = tensor[page]
            cache.pending_key[s], cache.pending_value[s] = cache.pending_key[0], cache.pending_value[0]
    cache.lengths.fill_(prefix)
    held = {m: [host(first[m])] * 3 for m in sides}
    lengths = [prefix] * 3
    for counts in ([1, 1, 1], [3, 80, 0], [1, 1, 1], [70, 2, 5]):
        rows = {m: make_rows(gen, counts, 2, 128, torch.bfloat16) * 2 for m in sides}
        cache.advance(torch.tensor(counts, dtype=torch.int32, device="cuda"))
        cache.write(rows["key"], rows["value"], starts=starts_of(counts))
        at = np.cumsum([0, *counts])
        held = {m: [np.concatenate([h, host(rows[m][a:b])]) for h, a, b in zip(held[m], at, at[1:])] for m in sides}
        lengths = [n + c for n, c in zip(lengths, counts)]
        check_contents(cache, lengths, held["key"], held["value"])
    check_attention(cache, make_query(gen, (3, 14, 128), torch.bfloat16), lengths)
    assert kernels.device_status() == 0
