# SPDX-License-Identifier: Apache-2.0
"""Calls of the tree operators past what their kernels' counts and layouts hold: refused on the host, before
any device call, so no GPU is needed and the pointers are never read."""
from __future__ import annotations

import pytest

import k3kda
from test_tree_refusals import ATTENTION, call


def refused(name, defaults, subject, **changed):
    rc, msg = call(name, defaults, **changed)
    assert rc == k3kda.EINVAL and msg.startswith(name) and subject in msg, (rc, msg)


def test_attention_over_more_steps_than_two_of_which_fit_an_int():
    """40 sequences of up to 2^30 positions, 2^25 steps of 32 each: sums of two counts of steps would pass an int."""
    refused("k3hip_mla_tree_attention", ATTENTION, "40 sequences", B=40, page=1 << 10, max_pages=1 << 20)


@pytest.mark.parametrize("bad", [(65536, 1, 1, 512), (1, 64, 1 << 15, 512), (1, 64, (1 << 31) - 1, 512), (1, 1, 65535 * 16 + 1, 8)])
def test_workspace_of_calls_that_are_too_large(bad):
    """What the call refuses has no workspace (not the size of a count that passed an int)."""
    assert k3kda.lib().k3hip_mla_tree_workspace(*bad) == 0
