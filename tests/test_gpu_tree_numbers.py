# SPDX-License-Identifier: Apache-2.0
"""Attention over trees of drafted tokens where its numbers leave the ordinary: queries, nodes and whole
pages that are not finite, in every place a sequence can be cut into parts. Plain form and tolerances:
test_gpu_tree.py; what such a value does not reach is compared bit for bit with the call without it. And
finite rows of sizes near the ends of fp32, or far apart."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_tree import SEED, U, rounded, run_attention, within
from tree_form import Cache, attention, path_of, random_tree

pytestmark = pytest.mark.gpu
KL, R = 512, 64


def with_pages(cache: Cache, pages) -> Cache:
    """The same table over other pages."""
    c = Cache.__new__(Cache)
    c.page, c.table, c.pages = cache.page, cache.table, pages
    return c


def attend(gpu, q, cache, lens, parents, bf16, counts=None):
    return run_attention(gpu, q, cache, np.asarray(lens, np.int32), counts, parents, 0.05, KL, bf16, False)


def only_these(got, clean, hit, what):
    """Rows of `hit` [B, N, H] are NaN throughout, their lse too; all others have the clean call's bits."""
    o, lse = got
    assert hit.any() and np.isnan(o[hit]).all(), f"{what}: o of rows that see it"
    assert np.isnan(lse[hit]).all(), f"{what}: lse of rows that see it"
    assert np.array_equal(o[~hit], clean[0][~hit]) and np.array_equal(lse[~hit], clean[1][~hit]), f"{what}: other rows"


# 16 heads are merged by eight waves a row, 64 by one
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("H", [16, 64])
@pytest.mark.parametrize("ctx", [0, 20, 700])
def test_a_query_that_is_nan(gpu, ctx, H, bf16):
    """One element of one query row: in a sequence of one step, which is not cut, and of many parts."""
    rng = np.random.default_rng(SEED + 201 + ctx + H)
    B, N = 2, 9
    cache = Cache(rng, B, ctx + N, 16, KL + R)
    cache.pages = rounded(cache.pages, bf16)
    q = rounded(rng.standard_normal((B, N, H, KL + R)).astype(np.float32), bf16)
    lens, parents = [ctx, ctx // 2], random_tree(rng, B, N)
    clean = attend(gpu, q, cache, lens, parents, bf16)
    hit = np.zeros((B, N, H), bool)
    for b, n, h, c in ((0, 4, 3, 0), (1, 8, H - 1, KL + R - 1), (1, 0, 7, 300)):
        hit[b, n, h], q[b, n, h, c] = True, np.nan
    only_these(attend(gpu, q, cache, lens, parents, bf16), clean, hit, "query")


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("what", [np.nan, np.inf])
@pytest.mark.parametrize("ctx,N,H", [(64, 1, 16), (64, 3, 16), (96, 3, 8), (32, 5, 64), (0, 3, 8), (65, 40, 16)])
def test_a_node_that_is_not_finite(gpu, ctx, N, H, what, bf16):
    """Contexts that end with a step of 32 positions, so that the nodes are alone in a part, and a tree over several parts."""
    rng = np.random.default_rng(SEED + 211 + ctx + N)
    B = 2
    cache = Cache(rng, B, ctx + N, 16, KL + R)
    cache.pages = rounded(cache.pages, bf16)
    q = rounded(rng.standard_normal((B, N, H, KL + R)).astype(np.float32), bf16)
    lens, parents = [ctx, ctx], random_tree(rng, B, N)
    if N > 2:
        parents[0][:3] = [-1, -1, 1]
    bad = min(1, N - 1)
    pages = cache.pages.copy()
    cache.pages[cache.at(0, ctx + bad)] = 0
    clean = attend(gpu, q, cache, lens, parents, bf16)
    pages[cache.at(0, ctx + bad)][::3] = what
    hit = np.zeros((B, N, H), bool)
    for n in range(N):
        hit[0, n] = bad in path_of(parents[0], n)
    only_these(attend(gpu, q, with_pages(cache, pages), lens, parents, bf16), clean, hit, "node")


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("H", [16, 64])
@pytest.mark.parametrize("first,last", [(2, 2), (0, 0), (4, 5)])
def test_committed_pages_of_nan(gpu, first, last, H, bf16):
    """Pages of 32 positions that hold nothing but NaN, so that parts see nothing else: every row of the sequence."""
    rng = np.random.default_rng(SEED + 221 + first + H)
    B, N, ctx = 2, 5, 300
    cache = Cache(rng, B, ctx + N, 32, KL + R)
    cache.pages = rounded(cache.pages, bf16)
    q = rounded(rng.standard_normal((B, N, H, KL + R)).astype(np.float32), bf16)
    lens, parents = [ctx, ctx - 50], random_tree(rng, B, N)
    clean = attend(gpu, q, cache, lens, parents, bf16)
    pages = cache.pages.copy()
    pages[cache.table[0, first:last + 1]] = np.nan
    hit = np.zeros((B, N, H), bool)
    hit[0] = True
    only_these(attend(gpu, q, with_pages(cache, pages), lens, parents, bf16), clean, hit, "pages")


# ------------------------------------------------------ rows of any size (fp32) ----
def sized(gpu, rng, sizes, q_size, lens, N, H, scale, zeros=()):
    """Sequences whose positions' rows are of size 2^sizes[b](t) (None: zero), queries of 2^q_size[b]. The check
    is test_gpu_tree's bound without its floor, everything of a sequence times a power of two that makes its
    largest row's size 1."""
    B = len(sizes)
    cache = Cache(rng, B, max(lens) + N, 16, KL + R)
    q = rng.standard_normal((B, N, H, KL + R)).astype(np.float32)
    top = np.full(B, -200)
    for b in range(B):
        q[b] *= np.float32(2.0 ** q_size[b])
        for t in range(lens[b] + N):
            k = sizes[b](t)
            cache.pages[cache.at(b, t)] *= np.float32(0 if k is None else 2.0 ** k)
            top[b] = max(top[b], -200 if k is None else k)
    lens, parents = np.asarray(lens, np.int32), random_tree(rng, B, N)
    got, got_lse = run_attention(gpu, q, cache, lens, None, parents, scale, KL, False, False)
    o, lse, mag, dot = attention(q, cache, lens, np.full(B, N), parents, scale, KL)
    T = int(lens.max()) + N
    e = 2 * (KL + R + 4) * U * dot + (T + 16) * U
    unit = (2.0 ** -top.astype(np.float64))[:, None, None, None]
    within(got.astype(np.float64) * unit, o * unit, e[..., None] * mag * unit, "o")
    within(got_lse, lse, e + 8 * U * np.abs(lse), "lse")


@pytest.mark.parametrize("k", [-105, -90, -120, 110])
@pytest.mark.parametrize("ctx", [20, 500])
def test_rows_of_one_far_size(gpu, ctx, k):
    """All rows of one size near the ends of fp32, the queries of ordinary size or (scores over rows of 2^110) of 2^-110."""
    rng = np.random.default_rng(SEED + 231 + ctx - k)
    sized(gpu, rng, [lambda t: k, lambda t: k], [min(0, -k)] * 2, [ctx, ctx // 3], 3, 8, 0.05)


@pytest.mark.parametrize("big,small", [(75, -60), (100, -100), (120, 0)])
@pytest.mark.parametrize("ctx", [20, 700])
def test_rows_of_far_sizes_together(gpu, ctx, big, small):
    """Rows of size 2^big among rows of size 2^small, in turn, one half behind the other and zeros among them: scores are
    alike, so that every row counts in the sum of the weights, within a part and between parts."""
    rng = np.random.default_rng(SEED + 241 + ctx + big)
    half = ctx // 2
    sizes = [lambda t: big if t % 2 else small, lambda t: big if t < half else small, lambda t: small if t < half else big,
             lambda t: (big, small, None)[t % 3]]
    sized(gpu, rng, sizes, [-big] * 4, [ctx] * 4, 3, 8, 0.05)


@pytest.mark.parametrize("k", [0, -7, -10, -14, -40])
@pytest.mark.parametrize("ctx", [25, 100])
def test_zero_rows_among_small_ones(gpu, ctx, k):
    """Rows of one small size and one, some or nothing but zero rows: what the others add to o keeps its accuracy."""
    rng = np.random.default_rng(SEED + 251 + ctx - k)
    sizes = [lambda t: None if t == 3 else k, lambda t: None if t % 4 == 1 else k, lambda t: None if t > 1 else k, lambda t: None]
    sized(gpu, rng, sizes, [0] * 4, [ctx] * 4, 3, 5, 0.05)
