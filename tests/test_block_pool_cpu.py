"""CPU checks of the block pool's C boundary (layout, refusals before the GPU is touched) and of its oracle."""

from __future__ import annotations

import ctypes
import random

import pytest

from oracle.block_pool import Pool
from unicache_b200 import BlockPool, _capi

from .test_block8_cpu import header_fields


def test_descriptor_follows_the_header():
    kinds = {ctypes.c_void_p: "Q", ctypes.c_int64: "q", ctypes.c_int32: "i"}
    assert "".join(kinds[k] for _, k in _capi.UcbBlockPool._fields_) == header_fields("ucb_block_pool")
    assert ctypes.sizeof(_capi.UcbBlockPool) == 56


def descriptor(**changes):
    fields = dict(block_table=4096, lengths=4096, held=4096, references=4096, num_blocks=8, num_seqs=4, max_blocks=4, block_tokens=64)
    return _capi.UcbBlockPool(**{**fields, **changes})


@pytest.mark.parametrize("changes,message", [
    ({"block_table": None}, "null pointer"), ({"held": None}, "null pointer"), ({"references": None}, "null pointer"),
    ({"references": 4104}, "aligned"), ({"num_seqs": 0}, "bad shape"), ({"num_seqs": 4097}, "4096 sequences"),
    ({"num_blocks": 0}, "bad shape"), ({"num_blocks": 1 << 31}, "2^31"), ({"block_tokens": 48}, "block_tokens"),
    ({"max_blocks": 1 << 30}, "2^31")])
def test_bad_pools_are_refused_by_every_entry(changes, message):
    lib, one = _capi.load(), ctypes.c_void_p(4096)
    pool = ctypes.addressof(struct := descriptor(**changes))
    for call in (lambda: lib.ucb_block_pool_advance(pool, None, 1, None), lambda: lib.ucb_block_pool_release(pool, one, 1, None),
                 lambda: lib.ucb_block_pool_fork(pool, one, one, 1, one, 1, 4, one, None),
                 lambda: lib.ucb_block_pool_compact(pool, one, 1, 4, one, one, None)):
        assert call() in (_capi.UCB_ERR_INVALID, _capi.UCB_ERR_UNSUPPORTED) and message in lib.ucb_last_error().decode()
    assert lib.ucb_block_pool_compact_workspace_bytes(pool) == -1
    assert struct is not None


def test_bad_calls_are_refused():
    lib, one = _capi.load(), ctypes.c_void_p(4096)
    pool = ctypes.addressof(struct := descriptor())
    for call, message in (
            (lambda: lib.ucb_block_pool_release(pool, None, 1, None), "null pointer"), (lambda: lib.ucb_block_pool_release(pool, one, -1, None), "count"),
            (lambda: lib.ucb_block_pool_fork(pool, one, one, 5, one, 1, 4, one, None), "one pair"),
            (lambda: lib.ucb_block_pool_fork(pool, None, one, 1, one, 1, 4, one, None), "null pointer"),
            (lambda: lib.ucb_block_pool_fork(pool, one, one, 1, None, 1, 4, one, None), "no caches"),
            (lambda: lib.ucb_block_pool_fork(pool, one, one, 1, one, 0, 4, one, None), "no caches"),
            (lambda: lib.ucb_block_pool_fork(pool, one, one, 1, one, 32768, 4, one, None), "32767"),
            (lambda: lib.ucb_block_pool_fork(pool, one, one, 1, one, 1, 4, ctypes.c_void_p(4104), None), "aligned"),
            (lambda: lib.ucb_block_pool_compact(pool, one, 1, 4, None, one, None), "null pointer"),
            (lambda: lib.ucb_block_pool_compact(pool, None, 1, 4, one, one, None), "no caches"),
            (lambda: lib.ucb_block_pool_compact(pool, one, 1, 4, one, ctypes.c_void_p(4098), None), "aligned")):
        assert call() in (_capi.UCB_ERR_INVALID, _capi.UCB_ERR_UNSUPPORTED) and message in lib.ucb_last_error().decode()
    assert lib.ucb_block_pool_release(pool, None, 0, None) == _capi.UCB_OK  # nothing to do
    assert lib.ucb_block_pool_fork(pool, None, None, 0, one, 1, 4, None, None) == _capi.UCB_OK
    assert lib.ucb_block_pool_fork_workspace_bytes(3) == 48 and lib.ucb_block_pool_compact_workspace_bytes(pool) == 80
    assert struct is not None


def test_there_is_no_cpu_path():
    with pytest.raises(RuntimeError):
        BlockPool.allocate(4, 64, 20, device="cpu")


def test_oracle_keeps_its_invariants():
    rng, pool = random.Random(0), Pool(9, 6, 30, 16)
    for _ in range(300):
        rng.choice([lambda: pool.advance([rng.choice([0, 1, 16, -1]) for _ in range(9)]), lambda: pool.release([rng.randrange(9)]),
                    lambda: pool.fork([rng.randrange(9)], [rng.randrange(9)]), pool.compact])()
        counts = pool.references()
        assert sum(counts) == sum(len(r) for r in pool.rows) and all(len(set(r)) == len(r) for r in pool.rows)
        assert all(len(r) <= pool.width for r in pool.rows)
    live = pool.compact()
    assert all(n > 0 for n in pool.references()[:live]) and not any(pool.references()[live:])
