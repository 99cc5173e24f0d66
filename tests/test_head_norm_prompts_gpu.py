"""Head norm with rotation for as many rows as prompts have: several rows of a token at once, and from token to token."""

from __future__ import annotations

import pytest
import torch

from unicache_b200 import head_norm_rope, kernels

from .gpu_util import need_gpu
from .test_head_norm_gpu import _check, _inputs

pytestmark = pytest.mark.gpu

# Head counts that four does not divide, tokens that make no equal turns.  One row a lane goes up to 303,104 lanes
# (tokens * heads * dim / 8), four rows of one token up to 2,424,832, and longer ones go from token to token.
CASES = [
    # tokens, q heads, kv heads, dim, rotary, interleaved, dtype
    (1501, 9, 5, 128, 128, False, torch.bfloat16),
    (4999, 16, 2, 64, 32, True, torch.float16),
    (2503, 15, 6, 256, 64, False, torch.float32),
    (1999, 12, 3, 128, 96, True, torch.float32),
    (9001, 3, 0, 128, 128, False, torch.float16),
    (9001, 13, 7, 128, 128, False, torch.bfloat16),
    (5003, 13, 4, 256, 256, True, torch.bfloat16),
    (5003, 15, 3, 256, 128, False, torch.float32),
    (20011, 10, 7, 64, 64, False, torch.float16),
    (16001, 0, 11, 128, 0, False, torch.bfloat16),
]


@pytest.mark.parametrize("tokens,hq,hk,dim,rotary,interleaved,dtype", CASES)
@pytest.mark.parametrize("weighted", [True, False])
def test_norm_and_rotation(tokens, hq, hk, dim, rotary, interleaved, dtype, weighted):
    need_gpu()
    query, key, weights, tables, positions = _inputs(tokens, hq, hk, dim, rotary, dtype)
    if not weighted:
        weights = [None, None]
    got = head_norm_rope(query, key, *weights, *tables, positions, eps=1e-5, interleaved=interleaved)
    for out, x, w in zip(got, (query, key), weights):
        if x is None:
            assert out is None
        else:
            _check(out, x, w, *tables, positions, 1e-5, interleaved)
    assert kernels.device_status() == 0


@pytest.mark.parametrize("tokens", [1501, 9001])
@pytest.mark.parametrize("interleaved", [False, True])
def test_outputs_may_be_the_inputs(tokens, interleaved):
    need_gpu()
    query, key, weights, tables, positions = _inputs(tokens, 14, 6, 128, 128, torch.bfloat16)
    how = dict(interleaved=interleaved)
    plain = head_norm_rope(query, key, *weights, *tables, positions, **how)
    narrow = head_norm_rope(query, key, *weights, *tables, positions.int(), **how)
    inside = head_norm_rope(query, key, *weights, *tables, positions, query_out=query, key_out=key, **how)
    for a, b, c in zip(plain, narrow, inside):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("tokens", [1501, 9001, 18001])
def test_positions_outside_the_tables_are_flagged(tokens):
    """In the first tokens, the last ones and between: their rows are NaN, the others untouched."""

    need_gpu()
    query, key, weights, tables, positions = _inputs(tokens, 14, 6, 128, 128, torch.bfloat16)
    good = head_norm_rope(query, key, *weights, *tables, positions)
    assert kernels.device_status() == 0
    wrong = [0, 1, tokens // 2, tokens - 2, tokens - 1]
    for value in (70000, -1, 1 << 40):
        moved = positions.clone()
        moved[wrong] = value
        got = head_norm_rope(query, key, *weights, *tables, moved)
        assert kernels.device_status() & 2
        rest = torch.ones(tokens, dtype=torch.bool, device="cuda")
        rest[wrong] = False
        for a, b in zip(got, good):
            assert a[wrong].isnan().all() and torch.equal(a[rest], b[rest])
    # in the last token alone
    moved = positions.clone()
    moved[-1] = 70000
    head_norm_rope(query, key, *weights, *tables, moved)
    assert kernels.device_status() & 2


def test_head_major_rows_and_a_gap_between_tokens():
    need_gpu()
    _, _, weights, tables, positions = _inputs(8000, 1, 1, 128, 128, torch.float16)
    major = torch.randn(22, 8000, 128, device="cuda").to(torch.float16).transpose(0, 1)
    gaps = torch.randn(8000, 22, 132, device="cuda").to(torch.float16)[:, :, 4:]
    for x in (major, gaps):
        got = head_norm_rope(x[:, :15], x[:, 15:], *weights, *tables, positions)
        _check(got[0], x[:, :15], weights[0], *tables, positions, 1e-6, False)
        _check(got[1], x[:, 15:], weights[1], *tables, positions, 1e-6, False)
