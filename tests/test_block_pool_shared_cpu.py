"""Withdrawn lengths over shared blocks, in the block pool's oracle: whatever is called, no new row goes into a block that two entries name."""

from __future__ import annotations

import random

import pytest

from oracle.block_pool import Pool


@pytest.mark.parametrize("seed", range(20))
def test_rows_go_into_blocks_of_one_sequence(seed):
    rng = random.Random(seed)
    seqs, width, block = 6, 6, 16
    pool = Pool(seqs, width, 40, block)
    grown = 0
    for _ in range(400):
        kind = rng.choice(["grow", "grow", "back", "fork", "release", "compact"])
        before = list(pool.lengths)
        if kind == "grow":
            pool.advance([min(rng.choice([0, 1, 5, block, 2 * block]), width * block - n) for n in before])
            references = pool.references()
            for s, (old, new) in enumerate(zip(before, pool.lengths)):
                written = pool.rows[s][old // block:-(-new // block)] if new > old else []
                assert all(references[b] == 1 for b in written), (s, old, new)
                grown += len(written)
        elif kind == "back":  # to blocks' ends, to nothing, and into blocks
            pool.advance([-rng.choice([0, n, n % block, n % block + block, rng.randint(0, n)]) for n in before])
        elif kind == "fork":
            pair = rng.sample(range(seqs), 2)
            pool.fork(pair[:1], pair[1:])
        elif kind == "release" and rng.random() < 0.3:
            pool.release([rng.randrange(seqs)])
        else:
            pool.compact()
        counts = pool.references()
        # only leading blocks are shared: along a row the references do not grow
        assert all(counts[a] >= counts[b] for row in pool.rows for a, b in zip(row, row[1:]))
    assert grown > 100


def test_blocks_are_given_back_when_a_sequence_grows_from_their_start():
    pool = Pool(3, 4, 8, 16)
    pool.advance([40, 0, 0])
    pool.fork([0], [1])
    assert pool.rows == [[0, 1, 2], [0, 1, 3], []]
    pool.advance([0, -24, 0])
    assert pool.lengths == [40, 16, 0] and pool.rows[1] == [0, 1, 3]
    pool.advance([0, 1, 0])
    assert pool.rows == [[0, 1, 2], [0, 3], []] and pool.lengths == [40, 17, 0]
    pool.advance([-40, 0, 0])
    pool.advance([10, 0, 20])  # block 0 is shared, 1 and 2 were sequence 0's alone: all three are given back
    assert pool.rows == [[1], [0, 3], [2, 4]] and not pool.refused
    pool.fork([1], [2])
    pool.advance([0, -17, -17])
    pool.advance([0, 1, 1])  # each sees block 0 shared as the call begins
    assert pool.rows == [[1], [0], [2]] and pool.lengths == [10, 1, 1] and not pool.refused
