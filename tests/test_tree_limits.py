# SPDX-License-Identifier: Apache-2.0
"""Calls of the tree operators past what their kernels' counts and layouts hold: refused on the host, before
any device call, so no GPU is needed and the pointers are never read."""
from __future__ import annotations

import ctypes as C

import pytest

import k3kda
from test_tree_refusals import APPEND, ATTENTION, A, call


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


A2 = C.c_void_p(1 << 24)


@pytest.mark.parametrize("B,N,H,ld,head", [
    (1, 4, 2, 64, 64),       # row n + 1's first head on row n's second
    (1, 4, 3, 100, 150),     # row 3 (300) on head 2 (300)
    (2, 3, 5, 128, 200),     # row 3 (384) ends inside head 2 (400)
    (1, 9, 2, 64, 500),      # head 1 inside the rows' range
])
def test_rotated_queries_whose_heads_overlap_rows(B, N, H, ld, head):
    refused("k3hip_latent_append", APPEND, "overlap", B=B, N=N, H=H, q_out=A2, q_out_ld=ld, q_out_head=head)


@pytest.mark.parametrize("B,N,H,ld,head", [
    (2, 9, 3, 192, 64), (2, 9, 3, 64, 18 * 64), (1, 4, 2, 1 << 20, 64), (1, 1, 5, 64, 64), (1, 9, 1, 64, 64),
    (1, 3, 3, 160, 224),     # rows at 0, 160, 320, heads at 0, 224, 448: between each other
])
def test_rotated_queries_that_do_not_overlap(B, N, H, ld, head):
    """Every layout in which no two heads of rows meet stands (no queries to rotate here: the check is all there is)."""
    starts = sorted(r * ld + h * head for r in range(B * N) for h in range(H))
    assert all(b - a >= 64 for a, b in zip(starts, starts[1:]))
    rc, msg = call("k3hip_latent_append", APPEND, B=B, N=N, H=H, q_out=A2, q_out_ld=ld, q_out_head=head, rows=None)
    assert rc == k3kda.EINVAL and "overlap" not in msg and "rows NULL" in msg


@pytest.mark.parametrize("changed", [dict(q_out_dtype=1), dict(q_out_ld=256), dict(q_out_head=72, q_out_ld=144)])
def test_queries_rotated_in_place_in_another_layout(changed):
    """A workgroup would write over what another has not read yet."""
    same = dict(q_out=A, q_out_dtype=0, q_out_ld=128, q_out_head=64)
    refused("k3hip_latent_append", APPEND, "in place", **{**same, **changed})


def test_rotated_queries_of_more_elements_a_row_than_an_int():
    refused("k3hip_latent_append", APPEND, "H=", H=(1 << 25), q_out=A2, q_out_ld=1 << 40, q_out_head=64)
