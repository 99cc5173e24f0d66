"""Axes that are no whole numbers are refused rather than rounded down."""

from __future__ import annotations

import pytest

from unicache_b200 import kernels


@pytest.mark.parametrize("axes", [(0.5, 1), (0, 1.25), (0, 1, float("nan"))])
def test_axes_that_are_no_whole_numbers(axes):
    with pytest.raises(ValueError):
        kernels._packed_axes(axes, 3, 8)


def test_whole_numbers_of_any_type_name_the_same_axes():
    assert kernels._packed_axes((0.0, True, 2), 3, 8) == kernels._packed_axes((0, 1, 2), 3, 8)
