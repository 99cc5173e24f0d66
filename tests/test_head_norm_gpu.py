"""Head norm with rotation against the float64 oracle."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import block8 as oracle
from unicache_b200 import head_norm_rope, kernels, rope_table

from .gpu_util import host, need_gpu

pytestmark = pytest.mark.gpu

# One rounding to the rows' type (half a unit in the last place, relative to the result), and fp32
# arithmetic before it: the sum of squares and the root cost a relative (D / 32 + 10) * 2^-24 < 2^-19
# of each normalised channel; the rotation adds two such products whose difference may be small, so that
# part is relative to their magnitudes.
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SMALLEST = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}


def _check(got, x, weight, cos, sin, positions, eps, interleaved):
    args = [None if t is None else host(t) for t in (weight, cos, sin, positions)]
    expect = oracle.head_norm_rope(host(x), *args, eps, interleaved)
    plain = np.abs(oracle.head_norm_rope(host(x), args[0], None, None, None, eps, interleaved))
    size = plain.max(-1, keepdims=True) * 2 if cos is not None else plain
    bound = HALF_ULP[x.dtype] * np.abs(expect) * 1.01 + SMALLEST[x.dtype] + 2.0 ** -19 * size
    err = np.abs(host(got).astype(np.float64) - expect)
    assert (err <= bound).all(), float((err - bound).max())


CASES = [
    # tokens, q heads, kv heads, dim, rotary, interleaved, dtype
    (1, 28, 4, 128, 128, False, torch.bfloat16),
    (33, 28, 4, 128, 128, False, torch.bfloat16),
    (300, 32, 8, 128, 128, True, torch.float16),
    (77, 16, 2, 64, 32, True, torch.float16),
    (77, 16, 2, 64, 32, False, torch.bfloat16),
    (5, 3, 1, 80, 40, False, torch.bfloat16),
    (5, 3, 1, 80, 24, True, torch.float32),
    (9, 4, 4, 256, 256, False, torch.bfloat16),
    (9, 4, 4, 256, 64, False, torch.float32),
    (13, 7, 7, 96, 0, False, torch.bfloat16),
    (13, 1, 1, 2, 2, True, torch.float32),
    (65, 5, 3, 64, 64, False, torch.float32),
    (1000, 9, 5, 128, 20, False, torch.bfloat16),
    (130, 6, 2, 33, 32, False, torch.bfloat16),
    (130, 12, 0, 128, 128, False, torch.bfloat16),
    (130, 0, 4, 128, 128, False, torch.bfloat16),
]


def _inputs(tokens, hq, hk, dim, rotary, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    qkv = (3 * torch.randn(tokens, hq + 2 * hk + 1, dim, generator=gen, device="cuda")).to(dtype)
    query = qkv[:, :hq] if hq else None
    key = qkv[:, hq:hq + hk] if hk else None
    weights = [(1 + 0.3 * torch.randn(dim, generator=gen, device="cuda")).to(dtype) for _ in range(2)]
    tables = rope_table(70000, rotary, theta=1e6) if rotary else (None, None)
    positions = torch.randint(0, 70000, (tokens,), generator=gen, device="cuda") if rotary else None
    return query, key, weights, tables, positions


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


def test_position_types_and_in_place_outputs():
    need_gpu()
    query, key, weights, tables, positions = _inputs(50, 28, 4, 128, 128, torch.bfloat16)
    plain = head_norm_rope(query, key, *weights, *tables, positions)
    narrow = head_norm_rope(query, key, *weights, *tables, positions.int())
    assert torch.equal(plain[0], narrow[0]) and torch.equal(plain[1], narrow[1])
    inside = head_norm_rope(query, key, *weights, *tables, positions, query_out=query, key_out=key)
    assert inside[0] is query and torch.equal(query, plain[0]) and torch.equal(key, plain[1])


@pytest.mark.parametrize("dim,rotary", [(128, 128), (64, 32), (80, 80)])
def test_unaligned_and_head_major_rows(dim, rotary):
    need_gpu()
    for interleaved in (False, True):
        _, _, weights, tables, positions = _inputs(37, 4, 2, dim, rotary, torch.bfloat16)
        flat = torch.randn(37 * 6 * (dim + 3) + 1, device="cuda").to(torch.bfloat16)
        odd = flat[1:].view(37, 6, dim + 3)[:, :, 1:dim + 1]
        major = torch.randn(6, 37, dim, device="cuda").to(torch.bfloat16).transpose(0, 1)
        for x in (odd, major):
            got = head_norm_rope(x[:, :4], x[:, 4:], *weights, *tables, positions, interleaved=interleaved)
            _check(got[0], x[:, :4], weights[0], *tables, positions, 1e-6, interleaved)
            _check(got[1], x[:, 4:], weights[1], *tables, positions, 1e-6, interleaved)


def test_large_small_and_broken_rows():
    """Squares that overflow fp32 are not representable (the row becomes 0, as the formula in fp32 gives);
    tiny rows are carried by eps; a NaN stays in its row."""

    need_gpu()
    x = torch.ones(4, 2, 128, device="cuda", dtype=torch.bfloat16)
    x[1] = 1e-20
    x[2, 0, 5] = float("nan")
    x[3] = 1e18
    got, _ = head_norm_rope(x, None)
    assert torch.equal(got[0], x[0])
    assert torch.allclose(got[1].float(), torch.full((2, 128), 1e-17, device="cuda"), rtol=2.0 ** -8, atol=0)
    assert got[2, 0].isnan().all() and torch.equal(got[2, 1], x[0, 0])
    assert torch.equal(got[3], x[0])


def test_positions_outside_the_tables_are_flagged():
    need_gpu()
    query, key, weights, tables, positions = _inputs(20, 4, 2, 128, 128, torch.bfloat16)
    good = head_norm_rope(query, key, *weights, *tables, positions)
    positions = positions.clone()
    positions[3], positions[7] = 70000, -1
    got = head_norm_rope(query, key, *weights, *tables, positions)
    assert kernels.device_status() & 2
    rest = [t for t in range(20) if t not in (3, 7)]
    for a, b in zip(got, good):
        assert a[3].isnan().all() and a[7].isnan().all() and torch.equal(a[rest], b[rest])
    assert kernels.device_status() == 0


def test_empty_and_refused_inputs():
    need_gpu()
    query, key, weights, tables, positions = _inputs(6, 4, 2, 128, 128, torch.bfloat16)
    out = head_norm_rope(query[:0], key[:0], *weights, *tables, positions[:0])
    assert out[0].shape == (0, 4, 128) and out[1].shape == (0, 2, 128)
    with pytest.raises(ValueError):
        head_norm_rope(None, None)
    with pytest.raises(RuntimeError):
        head_norm_rope(query.cpu(), None)
    with pytest.raises(ValueError):
        head_norm_rope(query, key.float(), *weights, *tables, positions)
    with pytest.raises(ValueError):
        head_norm_rope(query, key[:5], *weights, *tables, positions)
    with pytest.raises(ValueError):
        head_norm_rope(query.double(), None)
    with pytest.raises(ValueError):
        head_norm_rope(query[..., ::2], None)
    with pytest.raises(ValueError):
        head_norm_rope(query, key, weights[0][:64], None)
    with pytest.raises(ValueError):
        head_norm_rope(query, key, *weights, tables[0], None, positions)
    with pytest.raises(ValueError):
        head_norm_rope(query, key, *weights, *tables, positions[:5])
    with pytest.raises(ValueError):
        head_norm_rope(query, key, *weights, *rope_table(8, 130), positions)
    with pytest.raises(ValueError):
        head_norm_rope(query, key, query_out=key)
    with pytest.raises(ValueError):
        rope_table(8, 3)
