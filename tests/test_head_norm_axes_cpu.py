"""CPU checks of the rotation by several axes: the record, its refusals and the helper for sections."""

from __future__ import annotations

import struct

import pytest

from unicache_b200 import _capi, kernels, rope_axes

VALUES = [4096] * 9 + [4608, 128, 4608, 128, 3584, 128, 512, 128, 100, 5, 28, 4, 128, 128, 0, 0, 0, 1e-6]


def test_record_follows_the_header():
    record = kernels._packed_axes(rope_axes([16, 24, 24]), 3, 77)
    stride, *rest = struct.unpack("=q8I2i", record)
    words, count = rest[:8], rest[8]
    assert len(record) == _capi.ROPE_AXES.size == 48 and (stride, count) == (77, 3)
    assert [words[i // 16] >> 2 * (i % 16) & 3 for i in range(64)] == [0] * 16 + [1] * 24 + [2] * 24


def test_sections():
    assert rope_axes([2, 3]) == (0, 0, 1, 1, 1)
    assert rope_axes([3, 2, 2], alternating=True) == (0, 1, 2, 0, 1, 2, 0)
    assert rope_axes([0, 1]) == (1,) == rope_axes([0, 1], alternating=True)
    for bad in ([], [-1, 2]):
        with pytest.raises(ValueError):
            rope_axes(bad)
    for axes, count in (((0, 3), 3), ((0, 1), 5), ((0, -1), 2), ((0,), 0)):
        with pytest.raises(ValueError):
            kernels._packed_axes(axes, count, 8)


@pytest.mark.parametrize("change,count,words,message", [
    ({0: 0}, 3, 0, "null pointer"), ({22: 0}, 3, 0, "no rotation"), ({}, 0, 0, "1 to 4 axes"), ({}, 5, 0, "1 to 4 axes"),
    ({}, 3, 3 << 10, "not among"), ({22: 130}, 3, 0, "rotary_dim"), ({17: 0}, 3, 0, "empty tables")])
def test_bad_calls_are_refused(change, count, words, message):
    values = list(VALUES)
    for k, v in change.items():
        values[k] = v
    lib = _capi.load()
    rc = lib.ucb_head_norm_rope_axes(_capi.HEAD_NORM_ARGS.pack(*values), _capi.ROPE_AXES.pack(5, words, *[0] * 7, count, 0), None)
    assert rc in (_capi.UCB_ERR_INVALID, _capi.UCB_ERR_UNSUPPORTED) and message in lib.ucb_last_error().decode()
    assert lib.ucb_head_norm_rope_axes(_capi.HEAD_NORM_ARGS.pack(*VALUES), None, None) == _capi.UCB_ERR_INVALID
