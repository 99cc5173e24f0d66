"""CPU checks of the block cache's and the head norm's C boundary: record layouts and refusals before the GPU
is touched."""

from __future__ import annotations

import ctypes
import re
import os

import pytest

from unicache_b200 import _capi, rope_table

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CODES = {"int64_t": "q", "int32_t": "i", "float": "f"}


def header_fields(name: str) -> str:
    """Format codes of a struct's fields, in order, from the header."""

    text = open(os.path.join(ROOT, "include", "unicache_b200.h")).read()
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
    codes = ""
    for line in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
        line = line.strip()
        if line:
            kind = "Q" if "*" in line else CODES[line.split()[0]]
            codes += kind * len(line.split(","))
    return codes


@pytest.mark.parametrize("name,packed", [("ucb_head_norm_args", _capi.HEAD_NORM_ARGS),
                                         ("ucb_block8_attention_args", _capi.BLOCK8_ATTENTION_ARGS)])
def test_packed_records_follow_the_header(name, packed):
    expand = re.sub(r"(\d+)([a-zQ])", lambda m: m.group(2) * int(m.group(1)), packed.format[1:])
    assert expand == header_fields(name)
    # no padding: eight-byte fields first, a whole number of eight bytes in all
    assert "iQ" not in expand and "iq" not in expand and "fQ" not in expand and packed.size % 8 == 0


def test_cache_descriptor_follows_the_header():
    kinds = {ctypes.c_void_p: "Q", ctypes.c_int64: "q", ctypes.c_int32: "i"}
    assert "".join(kinds[k] for _, k in _capi.UcbBlock8Cache._fields_) == header_fields("ucb_block8_cache")
    assert ctypes.sizeof(_capi.UcbBlock8Cache) == 112


def descriptor(**changes):
    fields = dict(key_code=4096, value_code=4096, key_scale=4096, value_scale=4096, key_low=4096, key_high=4096,
                  pending_key=4096, pending_value=4096, block_table=4096, lengths=4096, num_blocks=8, num_seqs=2,
                  max_blocks=4, kv_heads=4, head_dim=128, block_tokens=64, dtype=_capi.UCB_BF16)
    return _capi.UcbBlock8Cache(**{**fields, **changes})


@pytest.mark.parametrize("changes,message", [
    ({"key_code": None}, "null pointer"), ({"lengths": None}, "null pointer"), ({"num_seqs": 0}, "bad shape"),
    ({"num_seqs": 5000}, "4096 sequences"), ({"head_dim": 96}, "head_dim"), ({"block_tokens": 48}, "block_tokens"),
    ({"dtype": _capi.UCB_F32}, "dtype"), ({"value_code": 4104}, "aligned"), ({"max_blocks": 1 << 30}, "2^31"),
])
def test_bad_caches_are_refused_by_every_entry(changes, message):
    lib = _capi.load()
    cache = ctypes.addressof(struct := descriptor(**changes))
    one = ctypes.c_void_p(4096)
    args = _capi.BLOCK8_ATTENTION_ARGS.pack(4096, 0, 4096, 4096, 4096, 3584, 0, 128, 1, 28, 0, 0.1)
    for rc in (lib.ucb_block8_write(cache, one, 512, 128, one, 512, 128, 2, None, None),
               lib.ucb_block8_read(cache, 2, None, one, one, None),
               lib.ucb_block8_select(cache, one, 3584, 128, 28, 4, 1, 2, one, None, None),
               lib.ucb_block8_attention(cache, args, None),
               lib.ucb_block8_sparse_attention(cache, _capi.BLOCK8_ATTENTION_ARGS.pack(
                   4096, 4096, 4096, 4096, 4096, 3584, 0, 128, 1, 28, 4, 0.1), 1, 2, None, None)):
        assert rc in (_capi.UCB_ERR_INVALID, _capi.UCB_ERR_UNSUPPORTED)
        assert message in lib.ucb_last_error().decode()
    assert lib.ucb_block8_select_workspace_bytes(cache) == -1
    assert struct is not None


@pytest.mark.parametrize("change,message", [
    ({0: 0}, "null pointer"), ({2: 0}, "null pointer"), ({4: 0}, "null pointer"), ({4: 4100}, "aligned"),
    ({2: 4104}, "aligned"), ({0: 4098}, "8 bytes"), ({7: 130}, "8 bytes"), ({8: 0}, "16 query tokens"), ({8: 17}, "16 query tokens"), ({9: 27}, "divisible"),
    ({1: 4096, 10: 0}, "selection")])
def test_bad_attention_calls_are_refused(change, message):
    lib = _capi.load()
    values = [4096, 0, 4096, 4096, 4096, 3584, 0, 128, 1, 28, 0, 0.1]
    for k, v in change.items():
        values[k] = v
    struct = descriptor()
    rc = lib.ucb_block8_attention(ctypes.addressof(struct), _capi.BLOCK8_ATTENTION_ARGS.pack(*values), None)
    assert rc in (_capi.UCB_ERR_INVALID, _capi.UCB_ERR_UNSUPPORTED) and message in lib.ucb_last_error().decode()


def test_bad_selections_and_rows_are_refused():
    lib = _capi.load()
    struct = descriptor()
    cache, one = ctypes.addressof(struct), ctypes.c_void_p(4096)
    for q_heads, count, first, recent, message in ((27, 4, 1, 2, "divisible"), (28, 0, 0, 0, "count"),
                                                   (28, 4, 3, 2, "count"), (28, 4, -1, 2, "count"),
                                                   (28, 5000, 1, 2, "4096 blocks")):
        rc = lib.ucb_block8_select(cache, one, 3584, 128, q_heads, count, first, recent, one, None, None)
        assert rc in (_capi.UCB_ERR_INVALID, _capi.UCB_ERR_UNSUPPORTED) and message in lib.ucb_last_error().decode()
    for blocks, queries, count, message in ((0, 1, 4, "null pointer"), (4096, 2, 4, "one query"), (4096, 1, 2, "count")):
        args = _capi.BLOCK8_ATTENTION_ARGS.pack(4096, blocks, 4096, 4096, 4096, 3584, 0, 128, queries, 28, count, 0.1)
        rc = lib.ucb_block8_sparse_attention(cache, args, 1, 2, None, None)
        assert rc in (_capi.UCB_ERR_INVALID, _capi.UCB_ERR_UNSUPPORTED) and message in lib.ucb_last_error().decode()
    assert lib.ucb_block8_write(cache, one, 512, 128, one, 512, 128, 3, None, None) == _capi.UCB_ERR_INVALID
    assert lib.ucb_block8_write(cache, None, 512, 128, one, 512, 128, 2, None, None) == _capi.UCB_ERR_INVALID
    assert lib.ucb_block8_read(cache, 3, None, one, one, None) == _capi.UCB_ERR_INVALID
    assert lib.ucb_block8_read(cache, 2, None, one, ctypes.c_void_p(4104), None) == _capi.UCB_ERR_INVALID
    assert lib.ucb_block8_write(cache, None, 0, 0, None, 0, 0, 0, one, None) == _capi.UCB_OK  # nothing to do


@pytest.mark.parametrize("change,message", [
    ({0: 0}, "null pointer"), ({7: 0}, "null pointer"), ({4: 0}, "null pointer"), ({18: -1}, "bad shape"),
    ({19: 0, 20: 0}, "bad shape"), ({21: 1}, "head_dim"), ({21: 257}, "head_dim"), ({22: 3}, "rotary_dim"),
    ({22: 130}, "rotary_dim"), ({17: 0}, "empty tables")])
def test_bad_head_norms_are_refused(change, message):
    lib = _capi.load()
    values = [4096] * 9 + [4608, 128, 4608, 128, 3584, 128, 512, 128, 100, 5, 28, 4, 128, 128, 0, 0, 0, 1e-6]
    for k, v in change.items():
        values[k] = v
    rc = lib.ucb_head_norm_rope(_capi.HEAD_NORM_ARGS.pack(*values), None)
    assert rc in (_capi.UCB_ERR_INVALID, _capi.UCB_ERR_UNSUPPORTED) and message in lib.ucb_last_error().decode()


def test_rope_table_is_exact_at_far_positions():
    import math

    cos, sin = rope_table(131073, 128, theta=1e6, device="cpu")
    for pos in (1, 4097, 131072):
        for i in (0, 1, 63):
            angle = pos * 1e6 ** (-i / 64)
            assert abs(float(cos[pos, i]) - math.cos(angle)) < 1e-7
            assert abs(float(sin[pos, i]) - math.sin(angle)) < 1e-7
    with pytest.raises(ValueError):
        rope_table(8, 0)
