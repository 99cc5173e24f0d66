"""CPU checks of draft verification: the argument record, refusals before the GPU is touched, and the oracle."""

from __future__ import annotations

import ctypes
import re

import numpy as np
import pytest

from oracle.verify import verify
from unicache_b200 import _capi

from .test_block8_cpu import header_fields


def test_packed_record_follows_the_header():
    packed = _capi.VERIFY_ARGS
    expand = re.sub(r"(\d+)([a-zQ])", lambda m: m.group(2) * int(m.group(1)), packed.format[1:])
    assert expand == header_fields("ucb_verify_args")
    assert "iQ" not in expand and "iq" not in expand and packed.size % 8 == 0


@pytest.mark.parametrize("change,message", [
    ({0: 0}, "null pointer"), ({1: 0}, "null pointer"), ({3: 0}, "null pointer"), ({7: 0}, "null pointer"), ({10: 0}, "null pointer"),
    ({10: 4104}, "aligned"), ({17: -1}, "bad shape"), ({18: -1}, "bad shape"), ({18: 32}, "31 drafts"), ({19: 0}, "bad shape"),
    ({17: 1 << 25}, "too many"), ({19: (1 << 30) + 1}, "too many"), ({2: 4096, 21: 3}, "dtype"), ({24: -1.0}, "temperature"), ({24: float("nan")}, "temperature"),
    ({24: float("inf")}, "temperature")])
def test_bad_calls_are_refused(change, message):
    values = [4096, 4096, 0, 4096, 0, 0, 0, 4096, 4096, 4096, 4096, 300, 100, 200, 100, 2, 3, 5, 2, 100, 0, 0, 0, 0, 1.0]
    for k, v in change.items():
        values[k] = v
    lib = _capi.load()
    rc = lib.ucb_verify_drafts(_capi.VERIFY_ARGS.pack(*values), None)
    assert rc in (_capi.UCB_ERR_INVALID, _capi.UCB_ERR_UNSUPPORTED) and message in lib.ucb_last_error().decode()
    assert lib.ucb_verify_drafts(None, None) == _capi.UCB_ERR_INVALID
    values[17], values[18], values[19], values[24] = 0, 2, 100, 1.0
    assert lib.ucb_verify_drafts(_capi.VERIFY_ARGS.pack(*values), ctypes.c_void_p()) == _capi.UCB_OK or change.keys() & {2}  # nothing to do


def test_oracle_draws_from_the_target():
    rng = np.random.default_rng(0)
    logits, q = rng.normal(size=(2, 5)), np.exp(rng.normal(size=(1, 5)))
    q /= q.sum()
    p, seen, kept = np.exp(logits[0]) / np.exp(logits[0]).sum(), np.zeros(5), 0
    for _ in range(20000):
        tokens, accepted, _, _, _ = verify(logits, rng.choice(5, 1, p=q[0]), rng.random(2), q, 1.0, 1)
        seen[tokens[0]] += 1
        kept += accepted
    assert (np.abs(seen - 20000 * p) <= 5 * np.sqrt(20000 * p * (1 - p))).all()
    assert abs(kept - 20000 * np.minimum(p, q[0]).sum()) <= 5 * np.sqrt(5000)
