# SPDX-License-Identifier: Apache-2.0
"""Calls of the tree operators past what their kernels' counts and layouts hold: refused on the host, before
any device call, so no GPU is needed and the pointers are never read."""
from __future__ import annotations

import k3kda
from test_tree_refusals import ATTENTION, call


def refused(name, defaults, subject, **changed):
    rc, msg = call(name, defaults, **changed)
    assert rc == k3kda.EINVAL and msg.startswith(name) and subject in msg, (rc, msg)


def test_attention_over_more_steps_than_two_of_which_fit_an_int():
    """40 sequences of up to 2^30 positions, 2^25 steps of 32 each: sums of two counts of steps would pass an int."""
    refused("k3hip_mla_tree_attention", ATTENTION, "40 sequences", B=40, page=1 << 10, max_pages=1 << 20)
