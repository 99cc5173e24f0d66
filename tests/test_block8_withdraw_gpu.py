"""Rows taken back from the 8-bit block cache (drafted tokens that were rejected): after the next
write the cache is the quantisation of the rows that count, as if the others had never come."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from unicache_b200 import kernels

from .gpu_util import host, need_gpu
from .test_block8_gpu import check_attention, check_contents, make_cache, make_query, make_rows, starts_of

pytestmark = pytest.mark.gpu


class Sequences:
    """A cache and, on the host, the rows that count of each of its sequences."""

    def __init__(self, seqs, *, block, heads=2, dim=128, dtype=torch.bfloat16, width=6, seed=0):
        self.cache, self.gen = make_cache([width * block] * seqs, heads=heads, dim=dim, block=block, dtype=dtype, seed=seed)
        self.shape, self.dtype = (heads, dim), dtype
        self.rows = {m: [np.zeros((0, heads, dim), np.float32) for _ in range(seqs)] for m in ("key", "value")}

    @property
    def lengths(self):
        return [len(r) for r in self.rows["key"]]

    def write(self, counts, factor=1.0, poison=(), count_them=True, one_each=False):
        new = {m: (make_rows(self.gen, counts, *self.shape, self.dtype).float() * factor).to(self.dtype) for m in self.rows}
        at = np.cumsum([0, *counts])
        for s in poison:
            new["key"][at[s] + counts[s] - 1, 0, 3] = float("nan")
            new["value"][at[s] + counts[s] - 1, 0, 5] = float("inf")
        self.cache.advance(torch.tensor(counts, dtype=torch.int32, device="cuda"))
        self.cache.write(new["key"], new["value"], starts=None if one_each else starts_of(counts))
        if count_them:
            for m in self.rows:
                self.rows[m] = [np.concatenate([r, host(new[m][a:b])]) for r, a, b in zip(self.rows[m], at, at[1:])]

    def withdraw(self, counts):
        self.cache.advance(-torch.tensor(counts, dtype=torch.int32, device="cuda"))

    def keep(self, lengths):
        for m in self.rows:
            self.rows[m] = [r[:n] for r, n in zip(self.rows[m], lengths)]

    def check(self):
        assert self.cache.lengths.tolist() == self.lengths
        check_contents(self.cache, self.lengths, self.rows["key"], self.rows["value"])


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,dim,dtype", [(2, 128, torch.bfloat16), (3, 64, torch.float16)])
def test_rejected_rows_leave_no_trace(block, heads, dim, dtype):
    """Drafts of larger rows, and of NaN and infinities, inside a block, up to its very end and from a block end
    on; part of them or all are taken back and others come."""

    need_gpu()
    held = [3, 5, block - 6, block - 5, 2 * block - 8, block, 2 * block, block + 1, 0]
    draft = [4, 4, 4, 5, 8, 4, 7, 5, 6]
    back = [3, 4, 4, 2, 5, 1, 7, 5, 2]
    q = Sequences(len(held), block=block, heads=heads, dim=dim, dtype=dtype, seed=block)
    q.write(held)
    q.check()
    q.write(draft, factor=8.0, poison=(1, 4, 7))  # their last rows, which go again
    kept = [h + d - b for h, d, b in zip(held, draft, back)]
    q.withdraw(back)
    q.keep(kept)
    q.write([1] * len(held), one_each=True)
    q.check()
    q.write([2] * len(held), factor=3.0)
    q.check()
    # and again, the drafts small
    small = [3, 3, 3, 3, 2, 3, 3, 3, 3]
    q.write(small, factor=0.1, count_them=False)
    q.withdraw(small)
    q.write([5, 1, 0, 2, block, 2 * block, 1, 3, 1], factor=0.5)
    q.write([1] * len(held), one_each=True)  # the sequence without rows in the last write has its block made again here
    q.check()
    assert kernels.device_status() == 0
    query = make_query(q.gen, (len(held), 4 * heads, dim), dtype)
    check_attention(q.cache, query, q.lengths)


def test_a_warm_up_step_taken_back():
    """A warm-up step whose lengths are put back, then the same step for good, across a block end."""

    need_gpu()
    q = Sequences(3, block=16, seed=5)
    q.write([15, 16, 7])
    for _ in range(20):
        q.write([1, 1, 1], factor=5.0, count_them=False, one_each=True)
        q.withdraw([1, 1, 1])
        q.write([1, 1, 1], one_each=True)
        q.check()
    assert kernels.device_status() == 0


def test_a_sequence_may_start_again_or_fall_back_to_a_block_end():
    need_gpu()
    block = 32
    q = Sequences(3, block=block, seed=6)
    q.write([100, 70, 45])
    q.withdraw([100, 6, 13])  # to nothing, and to block ends
    q.keep([0, 64, 32])
    q.write([40, 3, 1])
    q.check()
    q.write([1, 1, 1], one_each=True)
    q.check()
    assert kernels.device_status() == 0


def test_rows_that_are_gone_are_not_made_up():
    """Taken back over a block end into the middle of the block before: its unquantised rows
    are gone, so a write there is refused and the block stays as it is."""

    need_gpu()
    block = 16
    for one_each in (True, False):
        q = Sequences(3, block=block, seed=7)
        q.write([14, 14, 3])
        q.write([4, 2, 4])  # the first one two rows into its second block, the next one to the block's end
        q.withdraw([3, 1, 1])
        q.keep([15, 15, 6])
        assert kernels.device_status() == 0
        before = {n: getattr(q.cache, n).clone() for n in ("key_code", "value_code", "key_scale", "value_scale", "key_low",
                                                          "key_high")}
        q.write([1, 1, 1], factor=20.0, one_each=one_each)
        assert kernels.device_status() & 2
        page = q.cache.block_table[0].long()
        for name, was in before.items():
            a, b = getattr(q.cache, name)[page], was[page]
            assert torch.equal(a.view(torch.int8), b.view(torch.int8)), name
        # the other sequences have what they were given
        fields = {m: q.rows[m] for m in q.rows}
        lengths = q.lengths
        check_contents(q.cache, [0, *lengths[1:]], fields["key"], fields["value"])
        # refused until the block is left, at its start or its end
        q.write([1, 1, 1], one_each=one_each)  # first row of the second block
        assert kernels.device_status() == 0
        q.cache.lengths[0] = 0
        q.rows = {m: [r[0][:0], r[1], r[2]] for m, r in q.rows.items()}
        q.write([20, 1, 1])
        q.check()
        assert kernels.device_status() == 0


def test_rows_that_never_came_are_not_made_up():
    """Lengths advanced without a write: the block would have rows that no one gave."""

    need_gpu()
    q = Sequences(2, block=16, seed=8)
    q.write([5, 5])
    q.cache.advance(torch.tensor([1, 0], dtype=torch.int32, device="cuda"))
    page = q.cache.block_table[0].long()
    before = q.cache.key_code[page].clone()
    q.write([1, 1], one_each=True)
    assert kernels.device_status() & 2
    assert torch.equal(q.cache.key_code[page], before)
    check_contents(q.cache, [0, 6], q.rows["key"], q.rows["value"])
    assert kernels.device_status() == 0
