"""Rows of more than 8192 columns, two chunks a lane, with more rows than the backward
has workgroups: sums over rows of a gate of channels and of each sequence."""

import pytest
import torch

from test_residual_gpu import TYPES, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("types", [TYPES[0], TYPES[1], TYPES[3]], ids=["fff", "bbb", "fbf"])
@pytest.mark.parametrize("shape,gate,post", [((3, 241, 8200), "channel", True), ((2, 300, 16384), "sequence", True),
                                             ((301, 2, 8193), "sequence", True), ((2, 7, 12289), "channel", False),
                                             ((5, 3, 9999), "full", True)],
                         ids=lambda v: str(v).replace(" ", ""))
def test_wide_rows_with_gates(shape, gate, post, types):
    a, dh, dy = make(shape, types, gate, post=post)
    check(a, dh, dy, types, p=0.1 if post else 0.0, seed=3, branch_scale=0.5)


@pytest.mark.parametrize("which", ["dh", "dy"])
def test_wide_rows_one_output_differentiated(which):
    a, dh, dy = make((4, 130, 8704), TYPES[1], "channel")
    check(a, dh, dy, TYPES[1], with_dh=which == "dh", with_dy=which == "dy")
