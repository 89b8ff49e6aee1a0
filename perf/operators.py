# SPDX-License-Identifier: Apache-2.0
"""Performance cases of the operators that verify a tree of drafted tokens on a hybrid KDA / MLA
stack: what a serving engine calls per layer and step of speculative decoding, through the public
binding (``k3kda``).

Kinds of case (``"kind"``):
  append       latent_append: MLA latents normalised, rotated and written to a paged cache
  attention    mla_tree_attention: drafted tokens over the paged cache and their ancestors
  move         latent_commit: the accepted path's rows moved together
  kda_step     kda_tree_step: a KDA layer's core over the tree, the state only read
  kda_commit   kda_tree_commit: state and conv history moved along the accepted path

Sizes are those of the repository's benchmark and tests (64 MLA heads, kv_lora 512, rope 64, 8192
cached positions, 16 sequences; 32 KDA heads of 128, up to 64 sequences) and odd ones between
them. Lengths, trees and accepted nodes are made from the case, values from the seed. Trees grow
as drafters grow them: each node hangs on one of the few before it, or on the context.
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

LB, EPS, CONV = -5.0, 1e-5, 4
KL, QR = 512, 64          # the benchmark's MLA layer: latent and rope widths
QH = 128 + 64             # its score scale, (nope + rope)^-0.5
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed() -> list[dict]:
    return [
        # one interactive sequence, one token over a short context: latency counts
        {"name": "attn_b1_token", "kind": "attention", "B": 1, "N": 1, "H": 64, "ctx": 500, "page": 64, "type": "bf16"},
        # a serving batch's ordinary decode step over 8k contexts: the cache is read once
        {"name": "attn_b64_token", "kind": "attention", "B": 64, "N": 1, "H": 64, "ctx": 8192, "page": 64, "type": "bf16"},
        # full-accuracy cache, ragged batch and trees, pages that end inside a tile
        {"name": "attn_fp32_ragged", "kind": "attention", "B": 7, "N": 13, "H": 64, "ctx": 3001, "page": 48, "type": "fp32"},
        # large trees over long documents: bound by the matrix cores
        {"name": "attn_tree64_32k", "kind": "attention", "B": 4, "N": 64, "H": 64, "ctx": 32768, "page": 64, "type": "bf16"},
        # the latents and queries of one drafted tree per sequence
        {"name": "append_tree_b16", "kind": "append", "B": 16, "N": 8, "H": 64, "ctx": 8192, "page": 64, "type": "bf16", "rows": "fp32"},
        # prompt chunks of a prefill entering the cache, far positions
        {"name": "append_prompt", "kind": "append", "B": 5, "N": 1733, "H": 64, "ctx": 130001, "page": 64, "type": "bf16", "rows": "bf16"},
        # the accepted paths of a serving batch
        {"name": "move_b64", "kind": "move", "B": 64, "N": 16, "ctx": 5000, "page": 64, "type": "bf16"},
        # one sequence, a large tree, full-accuracy rows
        {"name": "move_b1", "kind": "move", "B": 1, "N": 64, "ctx": 777, "page": 16, "type": "fp32"},
        # one interactive sequence's tree through a KDA layer: latency counts
        {"name": "kda_step_b1", "kind": "kda_step", "B": 1, "N": 8, "H": 32, "D": 128, "act": "bf16", "y": "fp32"},
        # a serving batch's trees: 128 MiB of state read
        {"name": "kda_step_b64", "kind": "kda_step", "B": 64, "N": 16, "H": 32, "D": 128, "act": "bf16", "y": "bf16"},
        # the state of one sequence moved on
        {"name": "kda_commit_b1", "kind": "kda_commit", "B": 1, "N": 8, "H": 32, "D": 128, "act": "bf16"},
        # the states of a serving batch moved on
        {"name": "kda_commit_b64", "kind": "kda_commit", "B": 64, "N": 16, "H": 32, "D": 128, "act": "bf16"},
    ]


def _logint(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["attention", "attention", "attention", "append", "move", "kda_step", "kda_step", "kda_commit"])
    page = rng.choice([16, 32, 48, 64, 64, 128])
    if kind == "attention":
        typ = rng.choice(["bf16", "bf16", "fp32"])
        B, N, H = _logint(rng, 1, 64), _logint(rng, 1, 64), rng.choice([8, 16, 32, 64, 64, 96])
        most = 4 * 64 * 64 * 32768 // (4 if typ == "fp32" else 1)   # rows x positions, as the largest listed
        ctx = _logint(rng, 60, max(61, min(32768, most // (B * N * H), 64 * 8192 // B)))
        return {"kind": kind, "B": B, "N": N, "H": H, "ctx": ctx, "page": page, "type": typ}
    if kind == "append":
        B = _logint(rng, 1, 64)
        N = _logint(rng, 1, 64) if rng.random() < 0.6 else _logint(rng, 65, max(66, 8000 // B))
        return {"kind": kind, "B": B, "N": N, "H": rng.choice([8, 16, 32, 64]), "ctx": _logint(rng, 10, 130000), "page": page,
                "type": rng.choice(["bf16", "fp32"]), "rows": rng.choice(["bf16", "fp32"])}
    if kind == "move":
        return {"kind": kind, "B": _logint(rng, 1, 64), "N": _logint(rng, 1, 64), "ctx": _logint(rng, 10, 30000), "page": page,
                "type": rng.choice(["bf16", "fp32"])}
    D, H, N = rng.choice([64, 128, 128]), rng.choice([4, 8, 16, 32, 32]), _logint(rng, 1, 64)
    B = _logint(rng, 1, max(1, min(64, 64 * 16 // N)))
    if kind == "kda_step":
        return {"kind": kind, "B": B, "N": N, "H": H, "D": D, "act": rng.choice(["bf16", "fp32"]), "y": rng.choice(["bf16", "fp32"])}
    return {"kind": kind, "B": B, "N": N, "H": H, "D": D, "act": rng.choice(["bf16", "fp32"])}


# ------------------------------------------------- lengths and trees, from the case alone ----
def _layout(case) -> dict:
    """lens, counts, parents (lists), accept, and per node the path of its ancestors."""
    r = random.Random("%s %s %s %s" % (case["kind"], case["B"], case["N"], case.get("ctx")))
    B, N, ctx = case["B"], case["N"], case.get("ctx", 0)
    lens = [ctx if b == 0 else r.randint(ctx // 2, ctx) for b in range(B)]
    counts = [N if b % 4 != 3 else r.randint(1, N) for b in range(B)]
    parents = [[-1 if n == 0 else r.randint(max(-1, n - 6), n - 1) for n in range(N)] for _ in range(B)]
    if N > 64:   # a prompt: a chain
        parents = [[n - 1 for n in range(N)] for _ in range(B)]
    accept = [r.randint(counts[b] // 2, counts[b] - 1) if b % 8 != 5 else -1 for b in range(B)]
    return {"lens": lens, "counts": counts, "parents": parents, "accept": accept}


def _path(parents, n) -> list[int]:
    p = []
    while n >= 0:
        p.append(n)
        n = parents[n]
    return p[::-1]


def work(case) -> dict:
    L, B = _layout(case), case["B"]
    nodes = sum(L["counts"])
    e = 2 if case.get("type") == "bf16" else 4
    if case["kind"] == "attention":
        seen = sum(c * l for c, l in zip(L["counts"], L["lens"])) * case["H"]
        seen += sum(len(_path(L["parents"][b], n)) for b in range(B) for n in range(L["counts"][b])) * case["H"]
        return {"bytes": (sum(L["lens"]) + nodes) * (KL + QR) * e + nodes * case["H"] * (KL + QR + KL) * e,
                "flops": 2.0 * seen * (KL + QR + KL)}
    if case["kind"] == "append":
        er = 2 if case["rows"] == "bf16" else 4
        return {"bytes": nodes * ((KL + QR) * (e + er) + case["H"] * QR * (e + er)),
                "flops": nodes * (5.0 * KL + 6.0 * QR * (1 + case["H"]))}
    paths = [_path(L["parents"][b], L["accept"][b]) for b in range(B)]
    if case["kind"] == "move":
        moved = sum(1 for p in paths for i, n in enumerate(p) if i != n)
        return {"bytes": 2.0 * moved * (KL + QR) * e + 12.0 * B + 4.0 * B * case["N"], "flops": 0.0}
    H, D = case["H"], case["D"]
    P, ea = H * D, 2 if case["act"] == "bf16" else 4
    if case["kind"] == "kda_step":
        ey = 2 if case["y"] == "bf16" else 4
        pairs = sum(len(_path(L["parents"][b], n)) for b in range(B) for n in range(L["counts"][b])) * H
        return {"bytes": B * P * D * 4.0 + B * 3 * P * (CONV - 1) * 4.0 + nodes * (P * (4 * ea + 4 + ey) + 4 * H),
                "flops": nodes * P * (4.0 * D + 60) + pairs * 9.0 * D}
    on = [p for p in paths if p]
    return {"bytes": len(on) * (2.0 * P * D * 4 + 2.0 * 3 * P * (CONV - 1) * 4) + sum(map(len, on)) * (P * (3 * ea + 4) + 4 * H),
            "flops": sum(map(len, on)) * P * (7.0 * D + 60)}


# ---------------------------------------------------------------------- inputs ----
def _inputs(case, seed) -> dict:
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 2654435761 % (1 << 62) + 1)
    L, B, N = _layout(case), case["B"], case["N"]
    dev = lambda v, t=torch.int32: torch.tensor(v, dtype=t, device="cuda")  # noqa: E731

    def randn(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)

    s = {"case": case, "lens": dev(L["lens"]), "counts": dev(L["counts"]), "parents": dev(L["parents"]), "accept": dev(L["accept"])}
    if case["kind"] in ("attention", "append", "move"):
        typ, page, W = DT[case["type"]], case["page"], KL + QR
        cols = -(-(max(L["lens"]) + N) // page)
        if case["kind"] == "attention":   # every page its own
            pool = B * cols + 3
            s["table"] = torch.randperm(pool, device="cuda", generator=g)[: B * cols].reshape(B, cols).to(torch.int32)
        else:   # the pages that are written are each sequence's own, those before them of a shared prompt
            tail = -(-N // page) + 1
            pool = B * tail + 3
            perm = torch.randperm(pool, device="cuda", generator=g).to(torch.int32)
            col = torch.arange(cols, device="cuda")[None, :] - s["lens"][:, None] // page
            mine = perm[torch.arange(B, device="cuda")[:, None] * tail + col.clamp(0, tail - 1)]
            s["table"] = torch.where(col >= 0, mine, perm[-1]).to(torch.int32).contiguous()
        s["pages"] = randn(pool, page, W, dtype=typ)
        if case["kind"] == "attention":
            s["q"] = randn(B, N, case["H"], W, dtype=typ)
            s["o"] = torch.zeros((B, N, case["H"], KL), dtype=typ, device="cuda")
        elif case["kind"] == "append":
            tr = DT[case["rows"]]
            s["rows"] = randn(B, N, W, scale=0.6, dtype=tr)
            s["q"] = randn(B, N, case["H"], QR, dtype=tr)
            s["q_out"] = torch.zeros((B, N, case["H"], QR), dtype=typ, device="cuda")
            s["norm_w"] = 1 + randn(KL, scale=0.1)
            s["inv_freq"] = (10000.0 ** (-torch.arange(0, QR, 2, device="cuda", dtype=torch.float64) / QR)).float()
        else:
            s["lens_out"] = torch.zeros(B, dtype=torch.int32, device="cuda")
        return s
    H, D = case["H"], case["D"]
    P, act = H * D, DT[case["act"]]
    for n in ("q_in", "k_in", "v_in", "gate"):
        s[n] = randn(B, N, P, dtype=act)
    s["z"], s["b_logit"] = randn(B, N, P, scale=0.5), randn(B, N, H)
    for n in ("q_conv", "k_conv", "v_conv"):
        s[n] = randn(P, CONV, scale=0.5)
    s["A_log"] = torch.rand(H, device="cuda", generator=g) * 1.5
    s["dt_bias"], s["o_norm"] = randn(P), 1 + randn(D, scale=0.1)
    s["conv_state"], s["S"] = randn(B, 3, P, CONV - 1), randn(B, H, D, D, scale=0.1)
    s["y"] = torch.zeros((B, N, P), dtype=DT[case.get("y", "fp32")], device="cuda")
    return s


def prepare(case, seed) -> dict:
    return _inputs(case, seed)


# ---------------------------------------------------------------------- plain forms ----
def _ancestors(parents):
    """[B, N, N] truth values: column m is n itself or an ancestor of n (up to 64 nodes)."""
    N = parents.shape[1]
    one = torch.arange(N, device=parents.device)
    a = ((one[None, :, None] == one[None, None, :]) | (parents[:, :, None] == one[None, None, :])).float()
    a = (a @ a > 0).float()
    a = (a @ a > 0).float()
    a = (a @ a > 0).float()
    a = (a @ a > 0).float()
    a = (a @ a > 0).float()
    return a @ a > 0


def _depth(parents):
    N = parents.shape[1]
    if N > 64:   # a chain
        return torch.arange(N, device=parents.device).expand_as(parents)
    return _ancestors(parents).sum(-1) - 1


def _attention(s):
    case, W = s["case"], KL + QR
    B, N, H = case["B"], case["N"], case["H"]
    T = s["table"].shape[1] * case["page"]
    cache = s["pages"][s["table"].long()].reshape(B, T, W).float()
    t = torch.arange(T, device="cuda")[None, None, :] - s["lens"][:, None, None]       # slot of a drafted token
    drafted = torch.gather(_ancestors(s["parents"]), 2, t.clamp(0, N - 1).expand(B, N, T)) & (t >= 0) & (t < N)
    seen = ((t < 0) | drafted)[:, :, None, :]
    x = (s["q"].float().reshape(B, N * H, W) @ cache.transpose(1, 2)).reshape(B, N, H, T) * QH ** -0.5
    x = torch.where(seen, x, float("-inf"))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).reshape(B, N * H, T)
    o = (p @ torch.where((t < N).reshape(B, T, 1), cache[:, :, :KL], 0.0)).reshape(B, N, H, KL)
    live = (torch.arange(N, device="cuda")[None, :] < s["counts"][:, None])[:, :, None, None]
    s["o"] = torch.where(live, o.to(s["o"].dtype), s["o"])
    return s["o"]


def _turn(x, cos, sin):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def _append(s):
    B, N, page = s["case"]["B"], s["case"]["N"], s["case"]["page"]
    n = torch.arange(N, device="cuda")[None, :]
    angle = (s["lens"][:, None] + _depth(s["parents"])).double()[:, :, None] * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    x = s["rows"].float()
    c = x[..., :KL]
    c = s["norm_w"] * c * torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS)
    row = torch.cat((c, _turn(x[..., KL:], cos, sin)), -1).to(s["pages"].dtype)
    live = n < s["counts"][:, None]
    slot = s["lens"][:, None] + n
    at = torch.gather(s["table"].long(), 1, slot // page) * page + slot % page
    s["pages"].view(-1, KL + QR)[at[live]] = row[live]
    q = _turn(s["q"].float(), cos[:, :, None], sin[:, :, None]).to(s["q_out"].dtype)
    s["q_out"] = torch.where(live[:, :, None, None], q, s["q_out"])
    return s["pages"], s["q_out"]


def _accepted(s):
    """[B, N] truth values of the accepted path, and each of its nodes' place on it."""
    N = s["parents"].shape[1]
    anc = _ancestors(s["parents"])
    on = torch.gather(anc, 1, s["accept"].clamp(0, N - 1).long()[:, None, None].expand(-1, 1, N))[:, 0]
    on = on & (s["accept"] >= 0)[:, None]
    return on, on.long().cumsum(1) - 1


def _move(s):
    page = s["case"]["page"]
    on, place = _accepted(s)
    flat = s["pages"].view(-1, KL + QR)
    src = s["lens"][:, None] + torch.arange(on.shape[1], device="cuda")[None, :]
    dst = s["lens"][:, None] + place.clamp(min=0)
    at = lambda slot: torch.gather(s["table"].long(), 1, slot // page) * page + slot % page  # noqa: E731
    flat[at(dst)[on]] = flat[at(src)[on]]
    s["lens_out"] = (s["lens"] + on.sum(1)).to(torch.int32)
    return s["pages"], s["lens_out"]


def _silu_conv(hist, x, up1, up2, up3, w):
    """The short convolution of every node: its own input, then its ancestors', then the history."""
    xs = torch.cat((hist.transpose(1, 2), x.float()), 1)
    pick = lambda i: torch.gather(xs, 1, i[:, :, None].expand(-1, -1, xs.shape[2]))  # noqa: E731
    a = w[:, 3] * x.float() + w[:, 0] * pick(up3) + w[:, 1] * pick(up2) + w[:, 2] * pick(up1)
    return a * torch.sigmoid(a)


def _kda_prepared(s):
    """q, k, v [B, H, N, D], the decay logs and beta of every node."""
    case = s["case"]
    B, N, H, D = case["B"], case["N"], case["H"], case["D"]
    par = s["parents"].long()
    node = torch.arange(N, device="cuda")[None, :].expand(B, N) + CONV - 1
    before = torch.tensor([0, 0, 1], device="cuda").expand(B, 3)
    up = torch.cat((before, torch.where(par >= 0, par + CONV - 1, CONV - 2)), 1)     # over history, then nodes
    up1 = torch.gather(up, 1, node)
    up2 = torch.gather(up, 1, up1)
    up3 = torch.gather(up, 1, up2)
    hd = lambda t: t.reshape(B, N, H, D).transpose(1, 2)  # noqa: E731
    q = hd(_silu_conv(s["conv_state"][:, 0], s["q_in"], up1, up2, up3, s["q_conv"]))
    k = hd(_silu_conv(s["conv_state"][:, 1], s["k_in"], up1, up2, up3, s["k_conv"]))
    v = hd(_silu_conv(s["conv_state"][:, 2], s["v_in"], up1, up2, up3, s["v_conv"]))
    q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) + 1e-6) * D ** -0.5
    k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    g = LB * torch.sigmoid(torch.exp(s["A_log"])[:, None, None] * hd(s["z"] + s["dt_bias"]))
    return q, k, v, g, torch.sigmoid(s["b_logit"]).transpose(1, 2)


def _kda_tree(s):
    """Everything of the tree by products: decays E between nodes, the delta values w, the ancestors."""
    q, k, v, g, beta = _kda_prepared(s)
    anc = _ancestors(s["parents"])
    G = anc.double()[:, None] @ g.double()                                            # decay logs from the context
    E = torch.exp((G[:, :, :, None] - G[:, :, None, :]).masked_fill_(~anc[:, None, :, :, None], float("-inf"))).float()
    from0 = torch.exp(G).float()
    kk = (E * k[:, :, :, None] * k[:, :, None, :]).sum(-1)
    qk = (E * q[:, :, :, None] * k[:, :, None, :]).sum(-1)
    eye = torch.eye(anc.shape[1], device="cuda", dtype=torch.float64)
    M = beta[..., None].double() * kk.double() * (1 - eye)
    M2 = M @ M
    M4 = M2 @ M2
    M8 = M4 @ M4
    M16 = M8 @ M8
    M32 = M16 @ M16
    inv = ((eye - M) @ (eye + M2) @ (eye + M4) @ (eye + M8) @ (eye + M16) @ (eye + M32)).float()   # (I + M)^-1, M^64 = 0
    w = inv @ (beta[..., None] * (v - (k * from0) @ s["S"]))
    return q, k, w, qk, from0, E


def _kda_step(s):
    case = s["case"]
    B, N, H, D = case["B"], case["N"], case["H"], case["D"]
    q, k, w, qk, from0, E = _kda_tree(s)
    o = ((q * from0) @ s["S"] + qk @ w).transpose(1, 2)                               # [B, N, H, D]
    o = s["o_norm"] * o * torch.rsqrt((o * o).mean(-1, keepdim=True) + EPS)
    y = (o.reshape(B, N, H * D) * torch.sigmoid(s["gate"].float())).to(s["y"].dtype)
    live = torch.arange(N, device="cuda")[None, :] < s["counts"][:, None]
    s["y"] = torch.where(live[:, :, None], y, s["y"])
    return s["y"]


def _kda_commit(s):
    case = s["case"]
    B, H, D = case["B"], case["H"], case["D"]
    q, k, w, qk, from0, E = _kda_tree(s)
    on, place = _accepted(s)
    took = (s["accept"] >= 0)
    at = s["accept"].clamp(min=0).long()
    row = lambda t: t[torch.arange(B, device="cuda"), :, at]  # noqa: E731
    S = row(from0)[..., None] * s["S"] + (row(E) * k).transpose(-1, -2) @ w
    n = on.sum(1)
    last = n[:, None] + torch.arange(CONV - 1, device="cuda")[None, :]                # of the history, then the path
    order = torch.argsort((~on).long(), dim=1, stable=True)                           # the path's nodes first
    src = torch.where(last < CONV - 1, last, torch.gather(order, 1, (last - (CONV - 1)).clamp(0, on.shape[1] - 1)) + CONV - 1)
    x = torch.stack((s["q_in"], s["k_in"], s["v_in"]), 1).float().transpose(2, 3)     # [B, 3, P, N]
    hist = torch.gather(torch.cat((s["conv_state"], x), 3), 3, src[:, None, None, :].expand(-1, 3, H * D, -1))
    s["S"] = torch.where(took[:, None, None, None], S, s["S"])
    s["conv_state"] = torch.where(took[:, None, None, None], hist, s["conv_state"])
    return s["S"], s["conv_state"]


def run(s):
    case = s["case"]
    if not own:
        return {"attention": _attention, "append": _append, "move": _move, "kda_step": _kda_step, "kda_commit": _kda_commit}[case["kind"]](s)
    k3 = _binding()
    tree = {"counts": s["counts"], "parents": None if case["N"] > 64 else s["parents"]}
    if case["kind"] == "attention":
        if "workspace" not in s:   # kept between the calls, as a serving loop keeps it
            size = k3.mla_tree_workspace(case["B"], case["N"], case["H"], KL)
            s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        k3.mla_tree_attention(s["q"], s["pages"], s["table"], s["lens"], s["o"], KL, QH ** -0.5, workspace=s["workspace"], **tree)
        return s["o"]
    if case["kind"] == "append":
        k3.latent_append(s["rows"], s["pages"], s["table"], s["lens"], KL, norm_w=s["norm_w"], eps=EPS, inv_freq=s["inv_freq"],
                         q=s["q"], q_out=s["q_out"], **tree)
        return s["pages"], s["q_out"]
    if case["kind"] == "move":
        k3.latent_commit(s["pages"], s["table"], s["lens"], s["accept"], case["N"], lens_out=s["lens_out"], **tree)
        return s["pages"], s["lens_out"]
    H, D = case["H"], case["D"]
    if case["kind"] == "kda_step":
        k3.kda_tree_step(s["q_in"], s["k_in"], s["v_in"], s["z"], s["b_logit"], s["gate"], s["q_conv"], s["k_conv"], s["v_conv"],
                         s["A_log"], s["dt_bias"], s["o_norm"], s["conv_state"], s["S"], s["y"], H, D, CONV, LB, EPS, D ** -0.5, **tree)
        return s["y"]
    k3.kda_tree_commit(s["q_in"], s["k_in"], s["v_in"], s["z"], s["b_logit"], s["q_conv"], s["k_conv"], s["v_conv"],
                       s["A_log"], s["dt_bias"], s["conv_state"], s["S"], s["accept"], H, D, CONV, LB, **tree)
    return s["S"], s["conv_state"]


def _binding():
    if "k3kda" not in sys.modules:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "kimi-k3-in-c_amd"))
    import k3kda
    return k3kda


# ---------------------------------------------------------------------- 64 bits ----
# From the definitions, sequence by sequence and node by node.
def exact(case, seed):
    s, L = _inputs(case, seed), _layout(case)
    return {"attention": _exact_attention, "append": _exact_append, "move": _exact_move, "kda_step": _exact_kda_step,
            "kda_commit": _exact_kda_commit}[case["kind"]](case, s, L)


def _slots(case, s, b, n):
    """Rows of the pool that hold slots 0 .. n - 1 of sequence b."""
    t = torch.arange(n, device="cuda")
    return s["table"][b].long()[t // case["page"]] * case["page"] + t % case["page"]


def _exact_attention(case, s, L):
    out = s["o"].double()
    for b in range(case["B"]):
        rows = s["pages"].view(-1, KL + QR)[_slots(case, s, b, L["lens"][b] + case["N"])].double()
        ctx = rows[: L["lens"][b]]
        for n in range(L["counts"][b]):
            path = [L["lens"][b] + m for m in _path(L["parents"][b], n)]
            q = s["q"][b, n].double()
            x = torch.cat((q @ ctx.T, q @ rows[path].T), 1) / math.sqrt(QH)
            p = torch.softmax(x, 1)
            out[b, n] = p[:, : ctx.shape[0]] @ ctx[:, :KL] + p[:, ctx.shape[0]:] @ rows[path][:, :KL]
    return out


def _exact_append(case, s, L):
    pages, q_out = s["pages"].double(), s["q_out"].double()
    flat = pages.view(-1, KL + QR)
    freq = s["inv_freq"].double()
    for b in range(case["B"]):
        c = L["counts"][b]
        deep = range(c) if case["N"] > 64 else [len(_path(L["parents"][b], n)) - 1 for n in range(c)]
        turn = torch.polar(torch.ones((), device="cuda", dtype=torch.float64),
                           torch.tensor([L["lens"][b] + d for d in deep], device="cuda", dtype=torch.float64)[:, None] * freq)
        x = s["rows"][b, :c].double()
        lat = x[:, :KL] / (x[:, :KL].square().mean(1, keepdim=True) + EPS).sqrt() * s["norm_w"].double()
        rot = torch.view_as_real(torch.view_as_complex(x[:, KL:].reshape(c, QR // 2, 2)) * turn).reshape(c, QR)
        flat[_slots(case, s, b, L["lens"][b] + c)[L["lens"][b]:]] = torch.cat((lat, rot), 1)
        q = torch.view_as_complex(s["q"][b, :c].double().reshape(c, case["H"], QR // 2, 2)) * turn[:, None]
        q_out[b, :c] = torch.view_as_real(q).reshape(c, case["H"], QR)
    return pages, q_out


def _exact_move(case, s, L):
    pages, lens = s["pages"].double(), list(L["lens"])
    flat = pages.view(-1, KL + QR)
    for b in range(case["B"]):
        path = _path(L["parents"][b], L["accept"][b])
        at = _slots(case, s, b, L["lens"][b] + case["N"])[L["lens"][b]:]
        flat[at[: len(path)]] = flat[at[path]]
        lens[b] += len(path)
    return pages, torch.tensor(lens, dtype=torch.int32)


def _exact_node(case, s, b, path, S):
    """Node path[-1] from its parent's state S [H, D, D]: (its state, its o)."""
    H, D, n = case["H"], case["D"], path[-1]
    out = []
    for i, name in enumerate(("q", "k", "v")):
        x = torch.cat((s["conv_state"][b, i].double(), s[name + "_in"][b, path].double().T), 1)[:, -CONV:]
        a = (x * s[name + "_conv"].double()).sum(1)
        out.append((a / (1 + torch.exp(-a))).reshape(H, D))
    q, k, v = out
    q = q / (q.square().sum(1, keepdim=True) + 1e-6).sqrt() / math.sqrt(D)
    k = k / (k.square().sum(1, keepdim=True) + 1e-6).sqrt()
    z = (s["z"][b, n].double() + s["dt_bias"].double()).reshape(H, D)
    a = torch.exp(LB / (1 + torch.exp(-torch.exp(s["A_log"].double())[:, None] * z)))
    beta = 1 / (1 + torch.exp(-s["b_logit"][b, n].double()))
    S = S * a[:, :, None]
    u = (S * k[:, :, None]).sum(1)
    S = S + k[:, :, None] * (beta[:, None] * (v - u))[:, None, :]
    return S, (S * q[:, :, None]).sum(1)


def _exact_kda_step(case, s, L):
    out = s["y"].double()
    for b in range(case["B"]):
        states = {-1: s["S"][b].double()}
        for n in range(L["counts"][b]):
            path = _path(L["parents"][b], n)
            states[n], o = _exact_node(case, s, b, path, states[L["parents"][b][n]])
            o = s["o_norm"].double() * o / (o.square().mean(1, keepdim=True) + EPS).sqrt()
            out[b, n] = o.reshape(-1) / (1 + torch.exp(-s["gate"][b, n].double()))
    return out


def _exact_kda_commit(case, s, L):
    S, hist = s["S"].double(), s["conv_state"].double()
    for b in range(case["B"]):
        path = _path(L["parents"][b], L["accept"][b])
        for i in range(len(path)):
            S[b], _ = _exact_node(case, s, b, path[: i + 1], S[b])
        for i, name in enumerate(("q_in", "k_in", "v_in")):
            hist[b, i] = torch.cat((s["conv_state"][b, i].double(), s[name][b, path].double().T), 1)[:, -(CONV - 1):]
    return S, hist
