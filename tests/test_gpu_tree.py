# SPDX-License-Identifier: Apache-2.0
"""The operators on trees of drafted tokens (latent_append, mla_tree_attention, latent_commit,
kda_tree_step, kda_tree_commit) against their plain 64-bit forms (tree_form.py).

Tolerances, fixed before the first run. u = 2^-24, a rounding of fp32; h = 2^-8 one of bf16; values of
the plain form on the same (already rounded) inputs.
  append     latent: the mean of KL squares is off by (KL + 2) u, half of that after the root, and root,
             reciprocal and two products by 8 u: rtol (KL / 2 + 9) u. Rope: the angle in turns is rounded
             once (pi u of angle), sine and cosine 4 u, products and sum 3 u: 16 u (|a| + |b|). bf16: + h.
  attention  a score is a sum of CW products: off by CW u times the sum of their sizes (d below), the base
             2 form adds 4 u of its size, a weight is off by twice that and 8 u relative, the sums over T
             positions by (T + 4) u: e = 2 (CW + 4) u d + (T + 16) u of sum p|c|. bf16 weights: + h of the
             same; bf16 results: + h |o|. lse: e + 8 u |lse|; with bf16 weights it is the log of the sum of the
             weights as they are used, each off by at most h of itself, so the sum by at most h of itself
             and its log by at most -log(1 - h) < 1.003 h: + 1.003 h.
  moves      bit for bit (rows, conv history).
  KDA        the decode bar of the other decode tests: rtol 1e-4 and atol 1e-4 rms; bf16 results + h."""
from __future__ import annotations

import numpy as np
import pytest

from conftest import assert_close
from tree_form import Cache, Kda, attention, path_of, random_tree, rotate

pytestmark = pytest.mark.gpu
U, HALF = 2.0 ** -24, 2.0 ** -8
SEED = 0x54524545


def cu(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def rounded(a, bf16: bool):
    """The values that a tensor of the given type holds."""
    import torch
    return torch.from_numpy(a).to(torch.bfloat16).float().numpy() if bf16 else a


def typ(bf16: bool):
    import torch
    return torch.bfloat16 if bf16 else torch.float32


def host(t):
    return t.float().cpu().numpy()


def within(got, want, tol, what):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} outside, worst {np.max(np.abs(got - want)[bad] / np.broadcast_to(tol, got.shape)[bad]):.3g}x"


def sequences(rng, B, N, ctx):
    lens = rng.integers(0, ctx + 1, B).astype(np.int32)
    lens[0] = ctx
    counts = rng.integers(0, N + 1, B).astype(np.int32)
    counts[0] = N
    return lens, counts


# ---------------------------------------------------------------- attention ----
def run_attention(gpu, q, cache, lens, counts, parents, scale, KL, bf16, o_bf16, workspace=None, fill=7.0):
    import torch
    B, N, H, _ = q.shape
    o = torch.full((B, N, H, KL), fill, device="cuda", dtype=typ(o_bf16))
    lse = torch.full((B, N, H), fill, device="cuda")
    gpu.mla_tree_attention(cu(q, typ(bf16)), cu(cache.pages, typ(bf16)), cu(cache.table), cu(lens), o, KL, scale,
                           counts=None if counts is None else cu(counts), parents=None if parents is None else cu(parents),
                           lse=lse, workspace=workspace)
    torch.cuda.synchronize()
    return host(o), lse.cpu().numpy()


def check_attention(got, got_lse, q, cache, lens, counts, parents, scale, KL, bf16, o_bf16, fill=7.0):
    B, N, H, W = q.shape
    counts = np.full(B, N) if counts is None else counts
    o, lse, mag, dot = attention(q, cache, lens, counts, parents, scale, KL)
    T = int(max(lens)) + N
    e = (2 * (W + 4) * U * dot + (T + 16) * U)[..., None] * mag
    tol = e + HALF * mag * bf16 + HALF * (np.abs(o) + e) * o_bf16 + 1e-30
    live = np.arange(N)[None, :] < counts[:, None]
    within(got[live], o[live], tol[live], "o")
    seen = live[:, :, None] & np.isfinite(lse)
    el = 2 * (W + 4) * U * dot + (T + 16) * U + 8 * U * np.abs(np.where(seen, lse, 0)) + 1.003 * HALF * bf16
    within(got_lse[seen], lse[seen], el[seen], "lse")
    assert np.all(np.isneginf(got_lse[live[:, :, None] & ~np.isfinite(lse)]))
    assert np.all(got[~live] == fill) and np.all(got_lse[~live] == fill), "rows past the nodes were written"


ATTENTION = [
    # B, N, H, KL, R, ctx, page, bf16, o_bf16, tree
    (1, 1, 64, 512, 64, 500, 64, True, True, False),      # a decode step
    (3, 1, 16, 512, 64, 130, 16, True, False, False),     # 16 rows: four position groups
    (2, 5, 6, 512, 64, 63, 48, True, True, True),         # 30 rows, pages that end inside a tile
    (2, 13, 5, 512, 64, 64, 7, True, True, True),         # 65 rows: two row tiles, odd pages
    (2, 64, 3, 512, 64, 1000, 128, True, True, True),     # the largest tree, several ranges
    (3, 33, 64, 512, 64, 257, 64, True, True, True),      # 2112 rows
    (5, 3, 8, 512, 64, 0, 16, True, True, True),          # no context at all
    (2, 4, 8, 64, 8, 90, 32, True, True, True),           # a small layer: channels past its width
    (2, 4, 9, 264, 0, 90, 32, True, False, True),         # no rope slot, a latent that ends inside a tile
    (1, 1, 64, 512, 64, 321, 64, False, False, False),
    (3, 1, 8, 512, 64, 100, 16, False, False, False),     # 8 rows, fp32
    (2, 7, 4, 512, 64, 95, 48, False, True, True),        # 28 rows
    (2, 13, 16, 512, 64, 700, 64, False, False, True),    # several row tiles and ranges
    (2, 3, 5, 40, 8, 77, 5, False, False, True),
]


@pytest.mark.parametrize("B,N,H,KL,R,ctx,page,bf16,o_bf16,tree", ATTENTION)
def test_attention(gpu, B, N, H, KL, R, ctx, page, bf16, o_bf16, tree):
    rng = np.random.default_rng(SEED + B * 1000 + N * 100 + H + ctx)
    W = KL + R
    lens, counts = sequences(rng, B, N, ctx)
    cache = Cache(rng, B, ctx + N, page, W)
    cache.pages = rounded(cache.pages, bf16)
    q = rounded(rng.standard_normal((B, N, H, W)).astype(np.float32), bf16)
    parents = random_tree(rng, B, N) if tree else None
    scale = float(np.float32(1.7 / np.sqrt(W)))
    got, lse = run_attention(gpu, q, cache, lens, counts, parents, scale, KL, bf16, o_bf16)
    check_attention(got, lse, q, cache, lens, counts, parents, scale, KL, bf16, o_bf16)


@pytest.mark.parametrize("case", range(10))
def test_attention_random(gpu, case):
    rng = np.random.default_rng(SEED + 77 + case)
    B, N, H = int(rng.integers(1, 6)), int(rng.integers(1, 65)), int(rng.integers(1, 40))
    KL, R = 8 * int(rng.integers(1, 65)), 8 * int(rng.integers(0, 9))
    ctx, page, bf16 = int(rng.integers(0, 400)), int(rng.integers(1, 100)), bool(rng.integers(0, 2))
    if N * H > 600:
        H = max(1, 600 // N)
    print(B, N, H, KL, R, ctx, page, bf16, flush=True)
    test_attention(gpu, B, N, H, KL, R, ctx, page, bf16, bool(rng.integers(0, 2)), True)


@pytest.mark.parametrize("bf16", [True, False])
def test_attention_values_out_of_range(gpu, bf16):
    """Pages that are none, lengths past the table or negative, counts past N, parents that are no earlier
    node: read as said, and nothing outside the buffers is touched (a stray read would bring in NaN)."""
    rng = np.random.default_rng(SEED + 5)
    B, N, H, KL, R, page = 5, 6, 9, 512, 64, 16
    cache = Cache(rng, B, 90 + N, page, KL + R)
    cache.pages = rounded(cache.pages, bf16)
    table = cache.table.copy()
    table[0, 1], table[1, :], table[2, -1], table[3, 0] = -1, 1 << 30, cache.pages.shape[0], -7
    lens = np.array([90, 64, 1 << 30, 40, -3], np.int32)
    counts = np.array([N, N, 4, 99, N], np.int32)
    parents = random_tree(rng, B, N)
    parents[3] = [5, 0, 2, 1 << 30, -9, 4]
    q = rounded(rng.standard_normal((B, N, H, KL + R)).astype(np.float32), bf16)
    cache.table = table
    got, lse = run_attention(gpu, q, cache, lens, counts, parents, 0.05, KL, bf16, False)
    cap = table.shape[1] * page
    check_attention(got, lse, q, cache, np.clip(lens, 0, cap), np.clip(counts, 0, N), parents, 0.05, KL, bf16, False)
    assert np.all(got[1] == 0) and np.all(np.isneginf(lse[1])), "a sequence without pages sees nothing"


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_attention_masked_places(gpu, bf16, what):
    """Not finite: one node of a tree, everything behind the last node and every page that is not in a
    table. Rows that see the node go NaN, all others are as without it."""
    rng = np.random.default_rng(SEED + 6)
    B, N, H, KL, R, page, ctx = 2, 9, 16, 512, 64, 16, 75
    cache = Cache(rng, B, ctx + N + page, page, KL + R)
    cache.pages = rounded(cache.pages, bf16)
    lens, counts = np.array([ctx, 70], np.int32), np.array([N, N - 2], np.int32)
    parents = random_tree(rng, B, N, 3)
    parents[0][:5] = [-1, 0, 0, 1, 2]
    q = rounded(rng.standard_normal((B, N, H, KL + R)).astype(np.float32), bf16)
    clean = Cache.__new__(Cache)
    clean.page, clean.table, clean.pages = page, cache.table, cache.pages.copy()
    used = np.zeros(cache.pages.shape[:2], bool)
    for b in range(B):
        for t in range(int(lens[b] + counts[b])):
            used[cache.at(b, t)] = True
    cache.pages[~used] = what
    cache.pages[cache.at(0, ctx + 2)][::3] = what
    got, lse = run_attention(gpu, q, cache, lens, counts, parents, 0.05, KL, bf16, False)
    hit = np.zeros((B, N), bool)
    for n in range(N):
        hit[0, n] = 2 in path_of(parents[0], n)
    assert hit.sum() >= 2 and not np.isfinite(got[hit]).all(axis=(1, 2)).any()
    clean.pages[cache.at(0, ctx + 2)] = 0
    o, l = got.copy(), lse.copy()
    ref, rl, _, _ = attention(q, clean, lens, counts, parents, 0.05, KL)
    o[hit], l[hit] = ref[hit], rl[hit]
    check_attention(o, l, q, clean, lens, counts, parents, 0.05, KL, bf16, False)


def test_attention_workspace_and_repeats(gpu):
    """The caller's workspace and the library's give the same bits, twice; one too small is refused."""
    import torch
    rng = np.random.default_rng(SEED + 8)
    B, N, H, KL, R, ctx = 2, 3, 16, 512, 64, 900
    lens, counts = sequences(rng, B, N, ctx)
    cache = Cache(rng, B, ctx + N, 64, KL + R)
    q, parents = rng.standard_normal((B, N, H, KL + R)).astype(np.float32), random_tree(rng, B, N)
    size = gpu.mla_tree_workspace(B, N, H, KL)
    ws = torch.full((size,), 0xff, dtype=torch.uint8, device="cuda")   # NaN wherever it is read unwritten
    runs = [run_attention(gpu, q, cache, lens, counts, parents, 0.04, KL, True, True, w) for w in (ws, None, ws)]
    for r in runs[1:]:
        assert np.array_equal(r[0], runs[0][0]) and np.array_equal(r[1], runs[0][1])
    with pytest.raises(gpu.K3HipError) as e:
        run_attention(gpu, q, cache, lens, counts, parents, 0.04, KL, True, True, ws[:4096])
    assert e.value.code == gpu.EINVAL


# ------------------------------------------------------- append and commit ----
@pytest.mark.parametrize("B,N,H,KL,R,ctx,page,dst,src,halves,norm,turn,tree", [
    (3, 8, 64, 512, 64, 900, 64, True, False, False, True, True, True),
    (2, 64, 5, 512, 64, 130000, 48, True, True, True, True, True, True),
    (2, 150, 3, 512, 64, 77, 16, False, False, False, True, True, False),   # a prompt's chunk
    (4, 5, 0, 512, 64, 0, 16, False, True, True, True, False, True),        # NoPE, no queries
    (2, 7, 3, 40, 6, 300, 5, True, False, False, False, True, True),        # element by element, no norm
    (2, 7, 3, 33, 10, 2000000, 5, False, False, True, True, True, True),    # far positions
    (1, 1, 2, 512, 0, 10, 16, True, True, False, True, False, False),       # no rope slot
])
def test_append(gpu, B, N, H, KL, R, ctx, page, dst, src, halves, norm, turn, tree):
    import torch
    rng = np.random.default_rng(SEED + B + N * 10 + KL)
    W = KL + R
    lens, counts = sequences(rng, B, N, ctx)
    lens = np.maximum(lens, ctx - 500).clip(0)      # close together: their pages are held
    first = int(lens.min()) // page
    cache = Cache(rng, B, ctx + N - first * page, page, W)
    cache.table = np.concatenate((np.full((B, first), -1, np.int32), cache.table), 1)
    cache.pages = rounded(cache.pages, dst)
    cache.table[-1, -1] = -1                        # the last sequence's last page does not exist
    parents = random_tree(rng, B, N) if tree else None
    wide = rounded(rng.standard_normal((B, N, W + 24)).astype(np.float32), src)
    w = (1 + 0.1 * rng.standard_normal(KL)).astype(np.float32) if norm else None
    freq = (10000.0 ** (-np.arange(R // 2) / max(1, R // 2))).astype(np.float32) if turn else None
    rows = cu(wide, typ(src))[..., 8:8 + W]         # rows of a wider projection
    pages = cu(cache.pages, typ(dst))
    q = qo = None
    if H and R:
        qh = rounded(rng.standard_normal((B, N, H, R + 16)).astype(np.float32), src)
        q, out = cu(qh, typ(src))[..., 16:], torch.full((B, N, H, W), 3.0, device="cuda", dtype=typ(dst))
        qo = out[..., KL:]
    gpu.latent_append(rows, pages, cu(cache.table), cu(lens), KL, norm_w=None if w is None else cu(w), eps=1e-5,
                      inv_freq=None if freq is None else cu(freq), rope_style=gpu.ROPE_HALVES if halves else gpu.ROPE_PAIRS,
                      q=q, q_out=qo, counts=cu(counts), parents=None if parents is None else cu(parents))
    torch.cuda.synchronize()
    want, tol = cache.pages.astype(np.float64), np.zeros_like(cache.pages, np.float64)
    if q is not None:
        wq, tq = np.full((B, N, H, R), 3.0), np.zeros((B, N, H, R))
    size = lambda x: np.abs(rotate(np.abs(x), 0, np.zeros(R // 2), halves)) + np.abs(  # noqa: E731
        np.concatenate((np.abs(x)[..., R // 2:], np.abs(x)[..., :R // 2]), -1) if halves else
        np.stack((np.abs(x)[..., 1::2], np.abs(x)[..., 0::2]), -1).reshape(x.shape))
    for b in range(B):
        for n in range(int(counts[b])):
            pos = int(lens[b]) + len(path_of(None if parents is None else parents[b], n)) - 1
            x = wide[b, n, 8:8 + W].astype(np.float64)
            lat, rope = x[:KL], x[KL:]
            if norm:
                lat = w * lat / np.sqrt((lat ** 2).mean() + 1e-5)
            t = size(rope) * 16 * U * turn
            if turn:
                rope = rotate(rope, pos, freq, halves)
            at = cache.at(b, int(lens[b]) + n)
            if at:
                want[at] = np.concatenate((lat, rope))
                tol[at] = np.concatenate(((KL / 2 + 9) * U * norm * np.abs(lat), t)) + HALF * dst * np.abs(want[at])
            if q is not None:
                x = qh[b, n, :, 16:]
                wq[b, n] = rotate(x, pos, freq, halves) if turn else x
                tq[b, n] = size(x) * 16 * U * turn + HALF * dst * np.abs(wq[b, n])
    within(host(pages), want, tol * 1.01, "cache")
    if q is not None:
        within(host(qo), wq, tq * 1.01, "queries")
        assert np.all(host(out[..., :KL]) == 3.0)


def test_append_of_single_tokens_from_a_projection(gpu):
    """[B, 1, ...] views whose token dimension has a stride of its own: the rows are B's."""
    import torch
    rng = np.random.default_rng(SEED + 22)
    B, H, KL, R = 3, 2, 64, 16
    wide = rng.standard_normal((B, 200)).astype(np.float32)
    pages, table, lens = torch.zeros((B, 16, KL + R), device="cuda"), cu(np.arange(B, dtype=np.int32)[:, None]), cu(np.array([3, 0, 15], np.int32))
    x = cu(wide)
    q, out = x[:, None, 88:88 + 2 * R].unflatten(-1, (H, R)), torch.zeros((B, 1, H, R), device="cuda")
    gpu.latent_append(x[:, None, 8:8 + KL + R], pages, table, lens, KL, q=q, q_out=out)
    torch.cuda.synchronize()
    for b, l in enumerate((3, 0, 15)):
        assert np.array_equal(host(pages)[b, l], wide[b, 8:8 + KL + R])
    assert np.array_equal(host(out)[:, 0].reshape(B, -1), wide[:, 88:88 + 2 * R])


def test_append_rotates_in_place(gpu):
    import torch
    rng = np.random.default_rng(SEED + 21)
    B, N, H, KL, R = 2, 5, 3, 64, 16
    cache = Cache(rng, B, 64, 16, KL + R)
    q0 = rng.standard_normal((B, N, H, R)).astype(np.float32)
    freq = (10000.0 ** (-np.arange(R // 2) / (R // 2))).astype(np.float32)
    args = (cu(rng.standard_normal((B, N, KL + R)).astype(np.float32)), cu(cache.pages), cu(cache.table),
            cu(np.array([9, 30], np.int32)), KL)
    q, out = cu(q0), torch.empty((B, N, H, R), device="cuda")
    gpu.latent_append(*args, inv_freq=cu(freq), q=q, q_out=out)
    gpu.latent_append(*args, inv_freq=cu(freq), q=q, q_out=q)
    assert torch.equal(q, out) and not torch.equal(q.cpu(), torch.from_numpy(q0))


@pytest.mark.parametrize("B,N,W,ctx,page,bf16,tree", [
    (8, 16, 576, 300, 64, True, True), (3, 64, 576, 77, 16, False, True), (4, 9, 45, 30, 7, True, True),
    (3, 64, 2400, 50, 16, False, True), (4, 6, 576, 40, 16, True, False), (2, 1, 576, 0, 16, True, True),
    (5, 12, 33, 21, 1, False, True),
])
def test_latent_commit(gpu, B, N, W, ctx, page, bf16, tree):
    import torch
    rng = np.random.default_rng(SEED + B * N + W)
    lens, counts = sequences(rng, B, N, ctx)
    counts = np.maximum(counts, 1).astype(np.int32)
    cache = Cache(rng, B, ctx + N, page, W)
    cache.pages = rounded(cache.pages, bf16)
    parents = random_tree(rng, B, N, 9) if tree else None
    accept = np.array([rng.integers(0, c) for c in counts], np.int32)
    accept[-1] = [-1, int(counts[-1]), 1 << 30][B % 3]     # none accepted
    pages, lens_d = cu(cache.pages, typ(bf16)), cu(lens)
    out = torch.full((B,), -5, dtype=torch.int32, device="cuda")
    args = (pages, cu(cache.table), lens_d, cu(accept), N)
    kw = {"counts": cu(counts), "parents": None if parents is None else cu(parents)}
    want, new = cache.pages.copy(), lens.copy()
    for b in range(B):
        path = path_of(None if parents is None else parents[b], int(accept[b])) if 0 <= accept[b] < counts[b] else []
        moved = [cache.pages[cache.at(b, int(lens[b]) + n)] for n in path]
        for i, r in enumerate(moved):
            want[cache.at(b, int(lens[b]) + i)] = r
        new[b] += len(path)
    gpu.latent_commit(*args, lens_out=out, **kw)
    torch.cuda.synchronize()
    assert np.array_equal(host(pages), want) and np.array_equal(out.cpu().numpy(), new)
    pages.copy_(cu(cache.pages, typ(bf16)))
    gpu.latent_commit(*args, lens_out=lens_d, **kw)       # the lengths moved in place
    torch.cuda.synchronize()
    assert np.array_equal(host(pages), want) and np.array_equal(lens_d.cpu().numpy(), new)


# ------------------------------------------------------------------- KDA ----
def kda_case(rng, B, N, H, D, K, lb, bf16, g_bf16):
    P = H * D
    f = lambda *s, scale=1.0: (rng.standard_normal(s) * scale).astype(np.float32)  # noqa: E731
    w = {"q_conv": f(P, K, scale=0.5), "k_conv": f(P, K, scale=0.5), "v_conv": f(P, K, scale=0.5),
         "A_log": rng.uniform(0, 1.5, H).astype(np.float32), "dt_bias": f(P), "o_norm": 1 + f(D, scale=0.1)}
    x = {n: rounded(f(B, N, P), bf16) for n in ("q", "k", "v")}
    x |= {"z": f(B, N, P, scale=0.5), "b": f(B, N, H), "gate": rounded(f(B, N, P), g_bf16)}
    return w, x, f(B, H, D, D, scale=0.1), f(B, 3, P, K - 1)


def kda_inputs(w, x, bf16):
    d = {n: cu(a) for n, a in w.items()}
    q, k, v = (cu(x[n], typ(bf16)) for n in ("q", "k", "v"))
    return (q, k, v, cu(x["z"]), cu(x["b"])), (d["q_conv"], d["k_conv"], d["v_conv"], d["A_log"], d["dt_bias"]), d["o_norm"]


def slots(S, hist):
    """State and history of each sequence in one slot, as k3hip_kda_layer_decode keeps them."""
    import torch
    B = S.shape[0]
    n, m = S[0].size, hist[0].size
    pad = (-(n + m)) % 4 + 8
    buf = torch.full((B, n + m + pad), 5.0, device="cuda")
    s, h = buf[:, :n].view(S.shape), buf[:, n:n + m].view(hist.shape)
    s.copy_(cu(S))
    if m:
        h.copy_(cu(hist))
    return buf, s, h if m else None


KDA = [
    # B, N, H, D, K, lb, bf16 in / gate / y, tree, slots
    (3, 8, 4, 128, 4, -5.0, True, True, False, True, False),
    (2, 16, 2, 128, 4, -5.0, False, False, False, True, True),
    (2, 64, 2, 128, 4, -5.0, True, False, True, True, False),
    (2, 64, 1, 128, 3, -0.1, False, False, False, False, True),    # a chain of 64 that hardly decays
    (2, 33, 3, 64, 2, 0.0, False, True, False, True, False),       # softplus gate
    (3, 5, 2, 32, 1, -5.0, True, True, True, True, False),         # no history
    (2, 17, 3, 16, 4, -2.0, False, False, False, True, False),
    (4, 1, 3, 128, 4, -5.0, True, True, True, False, True),        # single tokens
    (2, 48, 1, 16, 2, -5.0, True, False, False, True, False),
]


@pytest.mark.parametrize("B,N,H,D,K,lb,bf16,g_bf16,y_bf16,tree,slot", KDA)
def test_kda_step_and_commit(gpu, B, N, H, D, K, lb, bf16, g_bf16, y_bf16, tree, slot):
    import torch
    rng = np.random.default_rng(SEED + 13 * B + N + D + K)
    P, eps, qs = H * D, 1e-5, float(np.float32(D ** -0.5))
    w, x, S0, h0 = kda_case(rng, B, N, H, D, K, lb, bf16, g_bf16)
    parents = random_tree(rng, B, N) if tree else None
    _, counts = sequences(rng, B, N, 0)
    ins, ws, o_norm = kda_inputs(w, x, bf16)
    if slot:
        buf, S, hist = slots(S0, h0)
    else:
        S, hist = cu(S0), cu(h0) if K > 1 else None
    y = torch.full((B, N, P), 9.0, device="cuda", dtype=typ(y_bf16))
    kw = {"counts": cu(counts), "parents": None if parents is None else cu(parents)}
    gpu.kda_tree_step(*ins, cu(x["gate"], typ(g_bf16)), *ws, o_norm, hist, S, y, H, D, K, lb, eps, qs, **kw)
    torch.cuda.synchronize()
    assert np.array_equal(host(S), S0) and (K == 1 or np.array_equal(host(hist), h0)), "the step changed the state"
    ref = Kda(w, H, D, K, lb, eps, qs)
    states = []
    got = host(y)
    for b in range(B):
        c = int(counts[b])
        xb = {n: a[b] for n, a in x.items()}
        want, st = ref.step(xb, c, None if parents is None else parents[b], S0[b], h0[b])
        states.append(st)
        if c:
            assert_close(got[b, :c], want[:c], 1e-4 * np.sqrt(np.mean(want[:c] ** 2)), 1e-4 + HALF * y_bf16, f"y of sequence {b}")
        assert np.all(got[b, c:] == 9.0)
    accept = np.array([rng.integers(c // 2, c) if c else 0 for c in counts], np.int32)
    if B > 2:
        accept[1] = -1
    gpu.kda_tree_commit(*ins, *ws, hist, S, cu(accept), H, D, K, lb, **kw)
    torch.cuda.synchronize()
    gS, gh = host(S), host(hist) if K > 1 else None
    for b in range(B):
        n = int(accept[b])
        if not 0 <= n < counts[b]:
            assert np.array_equal(gS[b], S0[b]) and (K == 1 or np.array_equal(gh[b], h0[b]))
            continue
        want = states[b][n]
        assert_close(gS[b], want, 1e-4 * np.sqrt(np.mean(want ** 2)), 1e-4, f"S of sequence {b}")
        if K > 1:
            path = path_of(None if parents is None else parents[b], n)
            assert np.array_equal(gh[b], ref.hist_after({m: a[b] for m, a in x.items()}, path, h0[b]))
    if slot:
        used = S0[0].size + h0[0].size
        assert torch.all(buf[:, used:] == 5.0)


def test_kda_decay_to_nothing(gpu):
    """Decays that underflow to zero (a softplus gate of hundreds) leave zeros, not NaN."""
    import torch
    rng = np.random.default_rng(SEED + 31)
    B, N, H, D, K = 1, 20, 2, 64, 4
    w, x, S0, h0 = kda_case(rng, B, N, H, D, K, 0.0, False, False)
    x["z"][:, ::3] = 400.0
    parents = random_tree(rng, B, N)
    ins, ws, o_norm = kda_inputs(w, x, False)
    y = torch.zeros((B, N, H * D), device="cuda")
    gpu.kda_tree_step(*ins, cu(x["gate"]), *ws, o_norm, cu(h0), cu(S0), y, H, D, K, 0.0, 1e-5, 0.125, parents=cu(parents))
    want, _ = Kda(w, H, D, K, 0.0, 1e-5, 0.125).step({n: a[0] for n, a in x.items()}, N, parents[0], S0[0], h0[0])
    assert_close(host(y)[0], want, 1e-4 * np.sqrt(np.mean(want ** 2)), 1e-4, "y")


def test_kda_step_matches_decode_steps(gpu):
    """A tree step's accepted path and commit against kda_decode_step token by token, over three rounds with
    the state carried: the loop the operators replace."""
    import torch
    rng = np.random.default_rng(SEED + 41)
    B, N, H, D, K = 3, 10, 3, 128, 4
    P, qs = H * D, float(np.float32(D ** -0.5))
    S = hist = None
    for step in range(3):
        w, x, S0, h0 = kda_case(np.random.default_rng(SEED + 43), B, N, H, D, K, -5.0, True, True)
        x = kda_case(rng, B, N, H, D, K, -5.0, True, True)[1]
        if S is None:
            S, hist = cu(S0), cu(h0)
        S1, h1 = S.clone(), hist.clone()
        parents = random_tree(rng, B, N)
        counts = np.array([N, 7, N], np.int32)
        accept = np.array([N - 1, 3, -1], np.int32)
        ins, ws, o_norm = kda_inputs(w, x, True)
        gate = cu(x["gate"], torch.bfloat16)
        y = torch.zeros((B, N, P), device="cuda")
        kw = {"counts": cu(counts), "parents": cu(parents)}
        gpu.kda_tree_step(*ins, gate, *ws, o_norm, hist, S, y, H, D, K, -5.0, 1e-5, qs, **kw)
        gpu.kda_tree_commit(*ins, *ws, hist, S, cu(accept), H, D, K, -5.0, **kw)
        for b in range(B):
            for n in path_of(parents[b], int(accept[b])):
                y1 = torch.zeros((1, P), device="cuda")
                r = [t[b, n][None].contiguous() for t in ins]
                gpu.kda_decode_step(*r, gate[b, n][None].contiguous(), *ws, o_norm, h1[b:b + 1], S1[b:b + 1], y1, H, D, K,
                                    -5.0, 1e-5, qs)
                torch.cuda.synchronize()
                want = y1[0].cpu().numpy()
                assert_close(host(y)[b, n], want, 2e-4 * np.sqrt(np.mean(want ** 2)), 2e-4, f"round {step} sequence {b} node {n}")
        assert torch.equal(hist, h1)
        assert_close(host(S), host(S1), 2e-4 * np.sqrt(np.mean(host(S1) ** 2)), 2e-4, f"round {step} S")


# --------------------------------------------------------------- together ----
def test_speculative_round(gpu):
    """Rounds of a hybrid layer pair as a serving loop runs them: append, attention, KDA step, then both
    commits, captured into one graph and replayed against the plain forms, with eager calls between."""
    import torch
    rng = np.random.default_rng(SEED + 51)
    B, N, HA, KL, R, page, H, D, K = 3, 6, 8, 512, 64, 16, 2, 64, 4
    W, P, qs, scale = KL + R, H * D, 0.125, 0.05
    cache = Cache(rng, B, 200, page, W)
    cache.pages = rounded(cache.pages, True)
    lens = np.array([40, 7, 95], np.int32)
    w, x, S0, h0 = kda_case(rng, B, N, H, D, K, -5.0, False, False)
    freq = (10000.0 ** (-np.arange(R // 2) / (R // 2))).astype(np.float32)
    nw = (1 + 0.1 * rng.standard_normal(KL)).astype(np.float32)
    d = {"pages": cu(cache.pages, torch.bfloat16), "table": cu(cache.table), "lens": cu(lens), "S": cu(S0), "hist": cu(h0),
         "rows": torch.zeros((B, N, W), device="cuda"), "qin": torch.zeros((B, N, HA, W), device="cuda", dtype=torch.bfloat16),
         "q": torch.zeros((B, N, HA, W), device="cuda", dtype=torch.bfloat16), "parents": torch.zeros((B, N), dtype=torch.int32, device="cuda"),
         "counts": torch.full((B,), N, dtype=torch.int32, device="cuda"), "accept": torch.zeros(B, dtype=torch.int32, device="cuda"),
         "o": torch.zeros((B, N, HA, KL), device="cuda"), "y": torch.zeros((B, N, P), device="cuda"),
         "ws": torch.empty(gpu.mla_tree_workspace(B, N, HA, KL), dtype=torch.uint8, device="cuda")}
    ins, ws, o_norm = kda_inputs(w, x, False)
    gate, nwd, fr = cu(x["gate"]), cu(nw), cu(freq)

    def verify():
        kw = {"counts": d["counts"], "parents": d["parents"]}
        d["q"].copy_(d["qin"])
        gpu.latent_append(d["rows"], d["pages"], d["table"], d["lens"], KL, norm_w=nwd, inv_freq=fr, q=d["qin"][..., KL:],
                          q_out=d["q"][..., KL:], **kw)
        gpu.mla_tree_attention(d["q"], d["pages"], d["table"], d["lens"], d["o"], KL, scale, workspace=d["ws"], **kw)
        gpu.kda_tree_step(*ins, gate, *ws, o_norm, d["hist"], d["S"], d["y"], H, D, K, -5.0, 1e-5, qs, **kw)
        gpu.kda_tree_commit(*ins, *ws, d["hist"], d["S"], d["accept"], H, D, K, -5.0, **kw)
        gpu.latent_commit(d["pages"], d["table"], d["lens"], d["accept"], N, lens_out=d["lens"], **kw)

    keep = {n: d[n].clone() for n in ("pages", "lens", "S", "hist")}
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        verify()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            verify()
    torch.cuda.synchronize()
    for n, t in keep.items():
        d[n].copy_(t)
    ref, S, hist = Kda(w, H, D, K, -5.0, 1e-5, qs), S0.astype(np.float64), h0.copy()
    for step in range(4):
        parents = random_tree(rng, B, N)
        counts = np.array([N, 1 + step, 3], np.int32)
        accept = np.array([N - 1 - step, 0, -1], np.int32)
        rows = rng.standard_normal((B, N, W)).astype(np.float32)
        qn = rounded(rng.standard_normal((B, N, HA, W)).astype(np.float32), True)
        for n, a in (("rows", rows), ("parents", parents), ("counts", counts), ("accept", accept), ("qin", qn)):
            d[n].copy_(cu(a))
        if step % 2:
            verify()   # eager, between the replays
        else:
            g.replay()
        torch.cuda.synchronize()
        # what the plain forms make of it
        q = qn.astype(np.float64)
        before = Cache.__new__(Cache)
        before.page, before.table, before.pages = page, cache.table, cache.pages.copy()
        for b in range(B):
            for n in range(int(counts[b])):
                pos = int(lens[b]) + len(path_of(parents[b], n)) - 1
                lat = rows[b, n, :KL].astype(np.float64)
                lat = nw * lat / np.sqrt((lat ** 2).mean() + 1e-5)
                row = np.concatenate((lat, rotate(rows[b, n, KL:], pos, freq, False))).astype(np.float32)
                before.pages[before.at(b, int(lens[b]) + n)] = rounded(row, True)
                q[b, n, :, KL:] = rotate(qn[b, n, :, KL:], pos, freq, False)
        q = rounded(q.astype(np.float32), True)
        o, _, mag, _ = attention(q, before, lens, counts, parents, scale, KL)
        live = np.arange(N)[None, :] < counts[:, None]
        # rows and queries rounded on either side of a tie: a step of 2^-7 in a few of them; the weights' rounding
        within(host(d["o"])[live], o[live], (6 * HALF * mag + 1e-3)[live], f"o of round {step}")
        after, new = before.pages.copy(), lens.copy()
        for b in range(B):
            path = path_of(parents[b], int(accept[b])) if 0 <= accept[b] < counts[b] else []
            for i, n in enumerate(path):
                after[before.at(b, int(lens[b]) + i)] = before.pages[before.at(b, int(lens[b]) + n)]
            new[b] += len(path)
            xb = {n: a[b] for n, a in x.items()}
            want, states = ref.step(xb, int(counts[b]), parents[b], S[b], hist[b])
            assert_close(host(d["y"])[b, :counts[b]], want[:counts[b]], 4e-4 * np.sqrt(np.mean(want ** 2)), 4e-4, f"y of round {step}")
            if path:
                S[b], hist[b] = states[path[-1]], ref.hist_after(xb, path, hist[b])
        assert np.array_equal(d["lens"].cpu().numpy(), new) and np.array_equal(host(d["hist"]), hist)
        assert_close(host(d["S"]), S, 4e-4 * np.sqrt(np.mean(S ** 2)), 4e-4, f"S of round {step}")
        got = host(d["pages"])
        within(got, after, 2.02 * HALF * np.abs(after) + 1e-30, f"cache of round {step}")
        cache.pages, lens = got, new


def test_on_another_stream(gpu):
    """Calls on a stream of their own, two in flight on two streams with workspaces of their own."""
    import torch
    rng = np.random.default_rng(SEED + 61)
    B, N, H, KL, R, ctx = 2, 4, 16, 512, 64, 600
    lens, counts = sequences(rng, B, N, ctx)
    cache = Cache(rng, B, ctx + N, 64, KL + R)
    cache.pages = rounded(cache.pages, True)
    q = [rounded(rng.standard_normal((B, N, H, KL + R)).astype(np.float32), True) for _ in range(2)]
    parents = random_tree(rng, B, N)
    pages, table, ln, ct, pr = cu(cache.pages, torch.bfloat16), cu(cache.table), cu(lens), cu(counts), cu(parents)
    qd = [cu(a, torch.bfloat16) for a in q]
    o = [torch.full((B, N, H, KL), 7.0, device="cuda") for _ in range(2)]
    lse = [torch.full((B, N, H), 7.0, device="cuda") for _ in range(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        for i, s in enumerate(streams):
            gpu.mla_tree_attention(qd[i], pages, table, ln, o[i], KL, 0.05, counts=ct, parents=pr, lse=lse[i], stream=s)
    torch.cuda.synchronize()
    for i in range(2):
        check_attention(host(o[i]), lse[i].cpu().numpy(), q[i], cache, lens, counts, parents, 0.05, KL, True, False)


def test_empty_calls(gpu):
    """No sequences, or no nodes: nothing is launched, nothing written."""
    import torch
    z = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    pages = z(2, 16, 72)
    gpu.mla_tree_attention(z(0, 3, 2, 72), pages, i(0, 1), i(0), z(0, 3, 2, 64), 64, 0.1)
    gpu.mla_tree_attention(z(2, 0, 2, 72), pages, i(2, 1), i(2), z(2, 0, 2, 64), 64, 0.1)
    gpu.latent_append(z(0, 3, 72), pages, i(0, 1), i(0), 64)
    gpu.latent_append(z(2, 0, 72), pages, i(2, 1), i(2), 64)
    gpu.latent_commit(pages, i(0, 1), i(0), i(0), 3)
    torch.cuda.synchronize()
    assert not pages.any()
