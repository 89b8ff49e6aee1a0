# SPDX-License-Identifier: Apache-2.0
"""Plain 64-bit forms (numpy) of the operators on trees of drafted tokens, node by node from their
definitions, and random lengths, trees and paged caches for their tests."""
from __future__ import annotations

import numpy as np


def path_of(parents, n: int) -> list[int]:
    """Node n's ancestors from the context down, n last; parents None: a chain."""
    p = []
    while n >= 0:
        p.append(n)
        up = n - 1 if parents is None else int(parents[n])
        n = up if 0 <= up < n else -1   # a number that is no earlier node: the committed context
    return p[::-1]


def random_tree(rng, B: int, N: int, reach: int = 5) -> np.ndarray:
    return np.array([[-1 if n == 0 else int(rng.integers(max(-1, n - reach), n)) for n in range(N)] for _ in range(B)],
                    np.int32).reshape(B, N)


class Cache:
    """A paged cache of B sequences on the host: pages [n_pages, page, W], a random table with spare pages."""

    def __init__(self, rng, B: int, slots: int, page: int, W: int, spare: int = 3):
        cols = max(1, -(-slots // page))
        n = B * cols + spare
        self.page, self.table = page, rng.permutation(n)[:B * cols].reshape(B, cols).astype(np.int32)
        self.pages = rng.standard_normal((n, page, W)).astype(np.float32)

    def at(self, b: int, t: int):
        """(page, row) of slot t of sequence b, None where it has no page."""
        i = t // self.page
        if i >= self.table.shape[1] or not 0 <= self.table[b, i] < self.pages.shape[0]:
            return None
        return int(self.table[b, i]), t % self.page


def attention(q, cache: Cache, lens, counts, parents, scale: float, KL: int):
    """o, lse, and the bounds' ingredients: sum_t p_t |c_t| and max_t scale |q| . |c_t| of each row."""
    B, N, H, W = q.shape
    o = np.zeros((B, N, H, KL))
    lse, mag, dot = np.full((B, N, H), -np.inf), np.zeros((B, N, H, KL)), np.zeros((B, N, H))
    cap = cache.table.shape[1] * cache.page
    for b in range(B):
        L = min(max(int(lens[b]), 0), cap)
        for n in range(int(counts[b])):
            at = [cache.at(b, t) for t in list(range(L)) + [L + m for m in path_of(None if parents is None else parents[b], n)]]
            at = [a for a in at if a]
            if not at:
                continue
            c = np.stack([cache.pages[a] for a in at]).astype(np.float64)
            x = q[b, n].astype(np.float64) @ c.T * scale
            m = x.max(1, keepdims=True)
            p = np.exp(x - m)
            l = p.sum(1, keepdims=True)
            p /= l
            o[b, n], mag[b, n] = p @ c[:, :KL], p @ np.abs(c[:, :KL])
            lse[b, n] = (m + np.log(l))[:, 0]
            dot[b, n] = (np.abs(q[b, n].astype(np.float64)) @ np.abs(c).T).max(1) * scale
    return o, lse, mag, dot


def rotate(x, pos: int, inv_freq, halves: bool):
    """x [..., R] rotated as position pos."""
    R = x.shape[-1]
    ang = pos * np.asarray(inv_freq, np.float64)
    c, s = np.cos(ang), np.sin(ang)
    x = x.astype(np.float64)
    a, b = (x[..., :R // 2], x[..., R // 2:]) if halves else (x[..., 0::2], x[..., 1::2])
    u, v = a * c - b * s, a * s + b * c
    return np.concatenate((u, v), -1) if halves else np.stack((u, v), -1).reshape(x.shape)


class Kda:
    """A KDA layer's core (conv, norms, gate, recurrence, output norm and gate) on one sequence."""

    def __init__(self, w: dict, H: int, D: int, K: int, lb: float, eps: float, q_scale: float):
        self.w = {n: np.asarray(a, np.float64) for n, a in w.items()}
        self.H, self.D, self.K, self.lb, self.eps, self.qs = H, D, K, lb, eps, q_scale

    def node(self, x: dict, n: int, path: list[int], S, hist):
        """(state, y row) of node n = path[-1] from its parent's state S [H, D, D]; x: the sequence's inputs."""
        H, D, K, w = self.H, self.D, self.K, self.w
        qkv = []
        for i, name in enumerate(("q", "k", "v")):
            win = np.concatenate((hist[i].T, x[name][path].astype(np.float64)))[-K:]       # [K, P]
            a = (win * w[name + "_conv"].T).sum(0)
            qkv.append((a / (1 + np.exp(-a))).reshape(H, D))
        q, k, v = qkv
        q = q / np.sqrt((q ** 2).sum(1, keepdims=True) + 1e-6) * self.qs
        k = k / np.sqrt((k ** 2).sum(1, keepdims=True) + 1e-6)
        z = (x["z"][n].astype(np.float64) + w["dt_bias"]).reshape(H, D)
        a = np.exp(w["A_log"])[:, None]
        g = self.lb / (1 + np.exp(-a * z)) if self.lb else -a * np.logaddexp(0, z)
        beta = 1 / (1 + np.exp(-x["b"][n].astype(np.float64)))
        S = S * np.exp(g)[:, :, None]
        u = np.einsum("hij,hi->hj", S, k)
        S = S + k[:, :, None] * (beta[:, None] * (v - u))[:, None, :]
        o = np.einsum("hij,hi->hj", S, q)
        y = w["o_norm"] * o / np.sqrt((o ** 2).mean(1, keepdims=True) + self.eps)
        return S, y.reshape(-1) / (1 + np.exp(-x["gate"][n].astype(np.float64)))

    def step(self, x: dict, count: int, parents, S, hist):
        """y [N, P] of the first `count` nodes, and every node's state."""
        y, states = np.zeros_like(x["gate"], np.float64), {}
        for n in range(count):
            path = path_of(parents, n)
            states[n], y[n] = self.node(x, n, path, states[path[-2]] if len(path) > 1 else S.astype(np.float64),
                                        hist.astype(np.float64))
        return y, states

    def hist_after(self, x: dict, path: list[int], hist):
        """The conv history [3, P, K-1] after the path: inputs themselves, nothing rounded."""
        return np.stack([np.concatenate((hist[i].T, x[n][path]))[len(path):].T for i, n in enumerate(("q", "k", "v"))])
