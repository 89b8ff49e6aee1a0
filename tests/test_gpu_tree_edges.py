# SPDX-License-Identifier: Apache-2.0
"""The operators on trees of drafted tokens at the ends of their ranges: more sequences than a wave has
lanes, more row tiles than the card has compute units, page pools past 4 GiB, rows of very different
sizes, unaligned inputs, captured graphs side by side. Plain forms and tolerances: test_gpu_tree.py;
what only moves or computes the same another way is compared bit for bit."""
from __future__ import annotations

import numpy as np
import pytest

from conftest import assert_close
from test_gpu_tree import SEED, check_attention, cu, host, kda_case, kda_inputs, rounded, run_attention, typ
from tree_form import Cache, Kda, path_of, random_tree

pytestmark = pytest.mark.gpu


def shifted(t):
    """The same values in memory that starts one element behind an aligned place."""
    import torch
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    buf[1:].copy_(t.flatten())
    return buf[1:].view(t.shape)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("B,N,H", [(70, 2, 3), (130, 1, 16)])
def test_attention_many_sequences(gpu, B, N, H, bf16):
    rng = np.random.default_rng(SEED + 101 + B)
    KL, R, ctx = 512, 64, 70
    lens = rng.integers(0, ctx + 1, B).astype(np.int32)
    counts = rng.integers(0, N + 1, B).astype(np.int32)
    counts[:3], counts[-1], lens[-1] = 0, N, ctx   # the first steps are not the first sequence's
    cache = Cache(rng, B, ctx + N, 16, KL + R)
    cache.pages = rounded(cache.pages, bf16)
    q = rounded(rng.standard_normal((B, N, H, KL + R)).astype(np.float32), bf16)
    parents = random_tree(rng, B, N)
    got, lse = run_attention(gpu, q, cache, lens, counts, parents, 0.05, KL, bf16, False)
    check_attention(got, lse, q, cache, lens, counts, parents, 0.05, KL, bf16, False)


@pytest.mark.parametrize("bf16,KL,R,H", [(True, 512, 64, 516), (False, 64, 8, 260)])
def test_attention_more_tiles_than_units(gpu, bf16, KL, R, H):
    """Over 256 tiles of query rows, of 128 (bf16) and 64 rows: a launch of more workgroups than the card has units."""
    rng = np.random.default_rng(SEED + 111)
    B, N, ctx = 1, 64, 45
    lens, counts = np.array([ctx], np.int32), np.array([N - 1], np.int32)
    cache = Cache(rng, B, ctx + N, 24, KL + R)
    cache.pages = rounded(cache.pages, bf16)
    q = rounded(rng.standard_normal((B, N, H, KL + R)).astype(np.float32), bf16)
    parents = random_tree(rng, B, N)
    got, lse = run_attention(gpu, q, cache, lens, counts, parents, 0.05, KL, bf16, bf16)
    check_attention(got, lse, q, cache, lens, counts, parents, 0.05, KL, bf16, bf16)


@pytest.mark.parametrize("page,ctx,bf16", [(8, 300, True), (40, 161, True), (12, 200, True), (8, 97, False), (1, 70, True), (1, 40, False)])
def test_attention_long_chains_and_small_pages(gpu, page, ctx, bf16):
    rng = np.random.default_rng(SEED + 121 + page)
    B, N, H, KL, R = 2, 64, 2, 512, 64
    lens, counts = np.array([ctx, ctx - 31], np.int32), np.array([N, N - 1], np.int32)
    cache = Cache(rng, B, ctx + N, page, KL + R)
    cache.pages = rounded(cache.pages, bf16)
    q = rounded(rng.standard_normal((B, N, H, KL + R)).astype(np.float32), bf16)
    got, lse = run_attention(gpu, q, cache, lens, counts, None, 0.05, KL, bf16, False)
    check_attention(got, lse, q, cache, lens, counts, None, 0.05, KL, bf16, False)


def test_attention_rows_of_all_sizes(gpu):
    """fp32 caches whose rows are of size 2^-60 or 2^60, with queries that make up for it, and of sizes 2^-15 .. 2^15 mixed,
    zeros among them: each keeps its accuracy. There the queries have no latent part, so that the scores stay small
    and every row counts."""
    rng = np.random.default_rng(SEED + 131)
    B, N, H, KL, R, ctx = 4, 3, 5, 512, 64, 90
    lens, counts = np.full(B, ctx, np.int32), np.full(B, N, np.int32)
    cache = Cache(rng, B, ctx + N, 16, KL + R)
    q = rng.standard_normal((B, N, H, KL + R)).astype(np.float32)
    q[2:, ..., :KL] = 0
    for b, k in ((0, -60), (1, 60)):
        q[b] *= np.float32(2.0 ** -k)
        for t in range(ctx + N):
            cache.pages[cache.at(b, t)] *= np.float32(2.0 ** k)
    for b in (2, 3):
        for t in range(ctx + N):
            cache.pages[cache.at(b, t)][:KL] *= np.float32(2.0 ** int(rng.integers(-15, 16)))
    for t in range(0, ctx, 3):
        cache.pages[cache.at(3, t)] = 0
    parents = random_tree(rng, B, N)
    got, lse = run_attention(gpu, q, cache, lens, counts, parents, 0.05, KL, False, False)
    check_attention(got, lse, q, cache, lens, counts, parents, 0.05, KL, False, False)


@pytest.mark.parametrize("k", [-28, -20, -10])
def test_attention_small_values_beside_large(gpu, k):
    """fp32 caches whose latents are 2^k of their rope slots, and queries whose latent part makes up for half of it."""
    rng = np.random.default_rng(SEED + 136)
    B, N, H, KL, R, ctx = 2, 3, 5, 512, 64, 80
    lens, counts = np.full(B, ctx, np.int32), np.full(B, N, np.int32)
    cache = Cache(rng, B, ctx + N, 16, KL + R)
    cache.pages[..., :KL] *= np.float32(2.0 ** k)
    q = rng.standard_normal((B, N, H, KL + R)).astype(np.float32)
    q[..., :KL] *= np.float32(2.0 ** (-k // 2))
    parents = random_tree(rng, B, N)
    got, lse = run_attention(gpu, q, cache, lens, counts, parents, 0.1, KL, False, False)
    check_attention(got, lse, q, cache, lens, counts, parents, 0.1, KL, False, False)


@pytest.mark.parametrize("bf16", [True, False])
def test_pool_past_4_gib(gpu, bf16):
    """Append, attention and commit on pages that lie more than 4 GiB into their pool."""
    import torch
    rng = np.random.default_rng(SEED + 141)
    B, N, H, KL, R, page, ctx = 2, 5, 4, 512, 64, 64, 130
    W = KL + R
    small = Cache(rng, B, ctx + N, page, W)
    small.pages = rounded(small.pages, bf16)
    n = small.pages.shape[0]
    row = page * W * (2 if bf16 else 4)
    first = (1 << 32) // row + 5
    pool = torch.empty((first + n, page, W), dtype=typ(bf16), device="cuda")
    pool[first:].copy_(cu(small.pages, typ(bf16)))
    near, far = cu(small.pages, typ(bf16)), pool
    lens, counts, parents = np.array([ctx, 77], np.int32), np.array([N, 3], np.int32), random_tree(rng, B, N)
    accept = np.array([N - 1, 2], np.int32)
    rows = cu(rng.standard_normal((B, N, W)).astype(np.float32))
    q = cu(rng.standard_normal((B, N, H, W)).astype(np.float32), typ(bf16))
    freq = cu((10000.0 ** (-np.arange(R // 2) / (R // 2))).astype(np.float32))
    out = []
    for pages, base in ((near, 0), (far, first)):
        table, ln = cu(small.table + np.int32(base)), cu(lens)
        kw = {"counts": cu(counts), "parents": cu(parents)}
        o = torch.zeros((B, N, H, KL), device="cuda")
        gpu.latent_append(rows, pages, table, ln, KL, inv_freq=freq, **kw)
        gpu.mla_tree_attention(q, pages, table, ln, o, KL, 0.05, **kw)
        gpu.latent_commit(pages, table, ln, cu(accept), N, lens_out=ln, **kw)
        torch.cuda.synchronize()
        out.append((o, pages[base:base + n].clone(), ln))
    for a, b in zip(*out):
        assert torch.equal(a, b)


# -------------------------------------------------------------- unaligned ----
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("D,N", [(128, 11), (128, 40), (32, 64), (64, 33), (16, 5)])
def test_kda_unaligned(gpu, D, N, bf16):
    """Inputs and outputs one element off their alignment: the same bits as aligned ones, which match the plain form."""
    import torch
    rng = np.random.default_rng(SEED + 151 + D + N)
    B, H, K, lb, eps, qs = 2, 2, 4, -5.0, 1e-5, float(np.float32(D ** -0.5))
    w, x, S0, h0 = kda_case(rng, B, N, H, D, K, lb, bf16, bf16)
    parents, accept = random_tree(rng, B, N), np.array([N - 1, N // 2], np.int32)
    ins, ws, o_norm = kda_inputs(w, x, bf16)
    gate = cu(x["gate"], typ(bf16))
    res = []
    for move in (lambda t: t, shifted):
        S, hist = cu(S0), move(cu(h0))
        y = move(torch.zeros((B, N, H * D), dtype=typ(bf16), device="cuda"))
        kw = {"parents": cu(parents)}
        gpu.kda_tree_step(*map(move, ins), move(gate), *map(move, ws), move(o_norm), hist, S, y, H, D, K, lb, eps, qs, **kw)
        gpu.kda_tree_commit(*map(move, ins), *map(move, ws), hist, S, cu(accept), H, D, K, lb, **kw)
        torch.cuda.synchronize()
        res.append((y, S, hist))
    for a, b in zip(*res):
        assert torch.equal(a, b)
    ref = Kda(w, H, D, K, lb, eps, qs)
    for b in range(B):
        xb = {n: a[b] for n, a in x.items()}
        want, states = ref.step(xb, N, parents[b], S0[b], h0[b])
        assert_close(host(res[0][0])[b], want, 1e-4 * np.sqrt(np.mean(want ** 2)), 1e-4 + 2.0 ** -8 * bf16, f"y of sequence {b}")
        st = states[int(accept[b])]
        assert_close(host(res[0][1])[b], st, 1e-4 * np.sqrt(np.mean(st ** 2)), 1e-4, f"S of sequence {b}")
        assert np.array_equal(host(res[0][2])[b], ref.hist_after(xb, path_of(parents[b], int(accept[b])), h0[b]))


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("src,dst", [(False, False), (False, True), (True, True)])
def test_append_unaligned(gpu, src, dst, halves):
    """Rows, queries and pages one element off: the same bits as aligned ones."""
    import torch
    rng = np.random.default_rng(SEED + 161)
    B, N, H, KL, R, page, ctx = 2, 6, 3, 512, 64, 16, 50
    cache = Cache(rng, B, ctx + N, page, KL + R)
    rows = cu(rng.standard_normal((B, N, KL + R)).astype(np.float32), typ(src))
    q = cu(rng.standard_normal((B, N, H, R)).astype(np.float32), typ(src))
    nw = cu((1 + 0.1 * rng.standard_normal(KL)).astype(np.float32))
    freq = cu((10000.0 ** (-np.arange(R // 2) / (R // 2))).astype(np.float32))
    lens, parents, res = cu(np.array([ctx, 9], np.int32)), cu(random_tree(rng, B, N)), []
    for move in (lambda t: t, shifted):
        pages = move(cu(cache.pages, typ(dst)))
        qo = move(torch.zeros((B, N, H, R), dtype=typ(dst), device="cuda"))
        gpu.latent_append(move(rows), pages, cu(cache.table), lens, KL, norm_w=move(nw), inv_freq=move(freq), q=move(q), q_out=qo,
                          rope_style=gpu.ROPE_HALVES if halves else gpu.ROPE_PAIRS, parents=parents)
        torch.cuda.synchronize()
        res.append((pages, qo))
    for a, b in zip(*res):
        assert torch.equal(a, b)


# ------------------------------------------------------------------ graphs ----
@pytest.mark.parametrize("bf16", [True, False])
def test_graphs_side_by_side(gpu, bf16):
    """Two graphs of one call each with a workspace of its own, and two that share one, replayed in turn with eager calls and
    new inputs between: every replay gives the eager call's bits."""
    import torch
    rng = np.random.default_rng(SEED + 171)
    B, N, H, KL, R, ctx = 3, 4, 16, 512, 64, 700
    cache = Cache(rng, B, ctx + N, 32, KL + R)
    pages, table, lens = cu(cache.pages, typ(bf16)), cu(cache.table), cu(np.array([ctx, 33, 400], np.int32))
    parents = cu(random_tree(rng, B, N))
    size = gpu.mla_tree_workspace(B, N, H, KL)
    space = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(3)]
    q = [torch.zeros((B, N, H, KL + R), dtype=typ(bf16), device="cuda") for _ in range(4)]
    o = [torch.zeros((B, N, H, KL), device="cuda") for _ in range(4)]
    call = lambda i, dst, ws: gpu.mla_tree_attention(q[i], pages, table, lens, dst, KL, 0.05, parents=parents, workspace=ws)  # noqa: E731
    stream, graphs = torch.cuda.Stream(), []
    with torch.cuda.stream(stream):
        call(0, o[0], space[0])
        torch.cuda.synchronize()
        for i in range(4):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                call(i, o[i], space[min(i, 2)])
            graphs.append(g)
    torch.cuda.synchronize()
    for step in range(4):
        for t in q:
            t.copy_(cu(rng.standard_normal(t.shape).astype(np.float32)))
        lens.copy_(cu(np.array([ctx - 90 * step, 33 + step, 400], np.int32)))
        for i in (step % 4, (step + 1) % 4, (step + 2) % 4, (step + 3) % 4):
            graphs[i].replay()
        want = [torch.zeros_like(t) for t in o]
        for i in range(4):
            call(i, want[i], None)
        torch.cuda.synchronize()
        for i in range(4):
            assert torch.equal(o[i], want[i]), f"graph {i} in round {step}"


# -------------------------------------------------------- not finite nodes ----
@pytest.mark.parametrize("what", [np.nan, np.inf])
@pytest.mark.parametrize("name", ["k", "v", "z", "b"])
@pytest.mark.parametrize("D,N", [(128, 12), (64, 40), (16, 20)])
def test_kda_nodes_that_are_not_finite(gpu, D, N, name, what):
    """A node whose inputs hold an infinity or a NaN: nodes that do not follow it are as without it, and so is a commit
    along another branch."""
    import torch
    rng = np.random.default_rng(SEED + 181 + D)
    B, H, K, lb, eps, qs = 1, 2, 4, -5.0, 1e-5, float(np.float32(D ** -0.5))
    w, x, S0, h0 = kda_case(rng, B, N, H, D, K, lb, False, False)
    parents = np.arange(N, dtype=np.int32)[None] - 2   # two branches, a node of each in turn
    parents[0][:6] = [-1, 0, 1, 1, 3, 2]
    hit = np.array([2 in path_of(parents[0], n) for n in range(N)])
    assert hit.sum() >= 2 and (~hit[3:]).sum() >= 3
    clean = {n: a.copy() for n, a in x.items()}
    x[name][0, 2, ::3] = what
    accept = int(np.flatnonzero(~hit)[-1])
    ins, ws, o_norm = kda_inputs(w, x, False)
    S, hist, y = cu(S0), cu(h0), torch.zeros((B, N, H * D), device="cuda")
    kw = {"parents": cu(parents)}
    gpu.kda_tree_step(*ins, cu(x["gate"]), *ws, o_norm, hist, S, y, H, D, K, lb, eps, qs, **kw)
    gpu.kda_tree_commit(*ins, *ws, hist, S, cu(np.array([accept], np.int32)), H, D, K, lb, **kw)
    torch.cuda.synchronize()
    ref = Kda(w, H, D, K, lb, eps, qs)
    want, states = ref.step({n: a[0] for n, a in clean.items()}, N, parents[0], S0[0], h0[0])
    got = host(y)[0]
    assert_close(got[~hit], want[~hit], 1e-4 * np.sqrt(np.mean(want ** 2)), 1e-4, "y")
    if what is np.nan:
        assert np.isnan(got[2]).any(), "the node itself"
    st = states[accept]
    assert_close(host(S)[0], st, 1e-4 * np.sqrt(np.mean(st ** 2)), 1e-4, "S")
