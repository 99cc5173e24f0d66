"""Head norm with rotation by positions of several axes, against the float64 oracle with every pair's own angle."""

from __future__ import annotations

import pytest
import torch

from unicache_b200 import head_norm_rope, kernels, rope_axes

from .gpu_util import need_gpu
from .test_head_norm_gpu import _check, _inputs

pytestmark = pytest.mark.gpu

BAD = 2  # the device error bit


def sections(half, count, fours):
    """Unequal sections of `half` pairs: by whole fours, so that a lane's pairs share an axis, or not."""

    step = 4 if fours else 1
    first = [max(0, half // (count + 1) // step * step)] * (count - 1)
    return [*first, half - sum(first)]


def own_tables(tables, positions, axes):
    """Tables of one row a token that hold each pair's own angle."""

    at = positions.long()[torch.tensor(axes, device="cuda")].t()
    return [t.gather(0, at) for t in tables]


def call_and_check(tokens, hq, hk, dim, rotary, interleaved, dtype, count, axes, weighted=True, wide=False):
    query, key, weights, tables, _ = _inputs(tokens, hq, hk, dim, rotary, dtype)
    if not weighted:
        weights = [None, None]
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    positions = torch.randint(0, 70000, (count, tokens), generator=gen, device="cuda", dtype=torch.int64 if wide else torch.int32)
    got = head_norm_rope(query, key, *weights, *tables, positions, eps=1e-5, interleaved=interleaved, axes=axes)
    own, each = own_tables(tables, positions, axes), torch.arange(tokens, device="cuda")
    for out, x, w in zip(got, (query, key), weights):
        if x is None:
            assert out is None
        else:
            _check(out, x, w, *own, each, 1e-5, interleaved)
    assert kernels.device_status() == 0


CASES = [
    # tokens, q heads, kv heads, dim, rotary, interleaved, dtype
    (1, 28, 4, 128, 128, False, torch.bfloat16),
    (33, 28, 4, 128, 128, True, torch.bfloat16),
    (77, 16, 2, 64, 32, True, torch.float16),
    (5, 3, 1, 80, 40, False, torch.bfloat16),  # one warp a row from here
    (5, 3, 1, 80, 24, True, torch.float32),
    (13, 1, 1, 2, 2, True, torch.float32),
    (130, 6, 2, 33, 32, False, torch.bfloat16),
    (1000, 9, 5, 128, 20, False, torch.bfloat16),
    (9, 4, 4, 256, 256, False, torch.bfloat16),  # and lanes again, up to the longest
    (9, 4, 0, 256, 64, True, torch.float32),
    (1501, 9, 5, 128, 128, False, torch.bfloat16),
    (4999, 16, 2, 64, 32, True, torch.float16),
    (9001, 13, 7, 128, 128, False, torch.bfloat16),
    (9001, 0, 15, 128, 96, True, torch.float16),
    (5003, 15, 3, 256, 128, False, torch.float32),
    (20011, 10, 7, 64, 64, False, torch.float16),
]


@pytest.mark.parametrize("tokens,hq,hk,dim,rotary,interleaved,dtype", CASES)
@pytest.mark.parametrize("count,kind", [(3, "fours"), (3, "odd"), (2, "turns"), (4, "turns"), (4, "fours"), (1, "fours")])
def test_norm_and_rotation(tokens, hq, hk, dim, rotary, interleaved, dtype, count, kind):
    need_gpu()
    lengths = sections(rotary // 2, count, kind == "fours")
    axes = rope_axes(lengths, alternating=kind == "turns")
    assert len(axes) == rotary // 2
    call_and_check(tokens, hq, hk, dim, rotary, interleaved, dtype, count, axes, weighted=tokens % 2 == 1, wide=tokens % 3 == 0)


@pytest.mark.parametrize("tokens", [3, 1501, 9001])
@pytest.mark.parametrize("interleaved", [False, True])
def test_equal_positions_are_the_one_axis_call_bit_for_bit(tokens, interleaved):
    need_gpu()
    query, key, weights, tables, positions = _inputs(tokens, 14, 6, 128, 128, torch.bfloat16)
    plain = head_norm_rope(query, key, *weights, *tables, positions, interleaved=interleaved)
    every = positions.int().expand(3, tokens)  # an axis stride of 0
    spaced = torch.zeros(4, tokens + 5, device="cuda", dtype=torch.int64)
    spaced[:, 2:tokens + 2] = positions
    for axes in (rope_axes([16, 24, 24]), rope_axes([24, 20, 20], alternating=True), (0,) * 64, (2,) * 64):
        for where in (every, spaced[:, 2:tokens + 2]):
            got = head_norm_rope(query, key, *weights, *tables, where, interleaved=interleaved, axes=axes)
            assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])
    inside = head_norm_rope(query, key, *weights, *tables, every, interleaved=interleaved, axes=rope_axes([16, 24, 24]),
                            query_out=query, key_out=key)
    assert torch.equal(inside[0], plain[0]) and torch.equal(inside[1], plain[1])


@pytest.mark.parametrize("dim,rotary,tokens", [(128, 128, 37), (64, 32, 37), (256, 128, 37), (80, 40, 37), (128, 64, 9001), (128, 40, 9001)])
@pytest.mark.parametrize("kind", ["fours", "odd", "turns"])
def test_a_position_outside_on_any_axis_makes_its_rows_nan(dim, rotary, tokens, kind):
    need_gpu()
    query, key, weights, tables, _ = _inputs(tokens, 5, 3, dim, rotary, torch.bfloat16)
    axes = rope_axes(sections(rotary // 2, 3, kind == "fours"), alternating=kind == "turns")
    for wide in (torch.int32, torch.int64):
        positions = torch.randint(0, 70000, (4, tokens), device="cuda", dtype=wide)
        whole = head_norm_rope(query, key, *weights, *tables, positions, axes=axes)
        assert kernels.device_status() == 0
        positions[0, 5], positions[1, 9], positions[2, 20], positions[2, tokens - 1] = -1, 70000, (1 << 31) - 1, -(1 << 31)
        positions[3] = -7  # an axis that no pair turns by is not looked at
        if wide is torch.int64:
            positions[1, 9] = 1 << 40  # 32 bits of it would be a row of the table
        got = head_norm_rope(query, key, *weights, *tables, positions, axes=axes)
        assert kernels.device_status() == BAD
        bad = torch.zeros(tokens, dtype=torch.bool, device="cuda")
        bad[[5, 9, 20, tokens - 1]] = True
        for a, b in zip(got, whole):
            assert a[bad].isnan().all() and torch.equal(a[~bad], b[~bad])


def test_rows_of_any_alignment():
    need_gpu()
    tokens, dim = 50, 128
    base = torch.randn(tokens, 9, dim + 3, device="cuda").to(torch.bfloat16)
    _, _, weights, tables, _ = _inputs(tokens, 4, 4, dim, dim, torch.bfloat16)
    positions, axes = torch.randint(0, 70000, (3, tokens), device="cuda", dtype=torch.int32), rope_axes([16, 24, 24])
    query, key = base[:, :5, 1:dim + 1], base[:, 5:, 1:dim + 1]
    got = head_norm_rope(query, key, *weights, *tables, positions, axes=axes)
    own, each = own_tables(tables, positions, axes), torch.arange(tokens, device="cuda")
    for out, x, w in zip(got, (query, key), weights):
        _check(out, x, w, *own, each, 1e-6, False)


def test_captured_and_on_another_stream():
    need_gpu()
    query, key, weights, tables, _ = _inputs(64, 28, 4, 128, 128, torch.bfloat16)
    positions, axes = torch.randint(0, 70000, (3, 64), device="cuda", dtype=torch.int32), rope_axes([16, 24, 24])
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        head_norm_rope(query, key, *weights, *tables, positions, axes=axes)
        with torch.cuda.graph(graph, stream=stream):
            captured = head_norm_rope(query, key, *weights, *tables, positions, axes=axes)
    torch.cuda.current_stream().wait_stream(stream)
    for _ in range(3):
        positions.random_(0, 70000)
        graph.replay()
        want = head_norm_rope(query, key, *weights, *tables, positions, axes=axes)
        assert torch.equal(captured[0], want[0]) and torch.equal(captured[1], want[1])


def test_bad_calls_are_refused():
    need_gpu()
    query, key, weights, tables, positions = _inputs(8, 4, 2, 64, 32, torch.bfloat16)
    where, axes = positions.expand(3, 8), rope_axes([4, 6, 6])
    for change in (dict(positions=positions), dict(positions=where[:, :7]), dict(positions=where.float()),
                   dict(positions=torch.zeros(8, 3, device="cuda", dtype=torch.int32).t()), dict(positions=where.cpu()),
                   dict(axes=axes[:-1]), dict(axes=(3,) * 16), dict(axes=(-1,) * 16), dict(axes=()),
                   dict(positions=positions.expand(5, 8)), dict(positions=where[:0]), dict(positions=None, cos=None, sin=None)):
        args = {"cos": tables[0], "sin": tables[1], "positions": where, "axes": axes, **change}
        with pytest.raises(ValueError):
            head_norm_rope(query, key, *weights, args["cos"], args["sin"], args["positions"], axes=args["axes"])
    none = head_norm_rope(query[:0], key[:0], *weights, *tables, where[:, :0], axes=axes)
    assert none[0].shape == (0, 4, 64) and kernels.device_status() == 0
