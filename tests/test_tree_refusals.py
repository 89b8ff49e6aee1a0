# SPDX-License-Identifier: Apache-2.0
"""What the entry points of the tree operators refuse, with the message's subject. The checks run on the
host before any device call, so no GPU is needed and the pointers are never read."""
from __future__ import annotations

import ctypes as C

import pytest

import k3kda

A = C.c_void_p(1 << 20)    # an address that satisfies every alignment
ODD = C.c_void_p((1 << 20) + 4)


def call(name, defaults, **changed):
    args = dict(defaults)
    assert set(changed) <= set(args), changed
    args.update(changed)
    L = k3kda.lib()
    return getattr(L, name)(*args.values()), L.k3hip_last_error().decode()


APPEND = dict(B=1, N=4, kv_lora=512, rope=64, pages=A, dtype=1, n_pages=8, page=16, table=A, max_pages=4, lens=A, counts=None,
              parents=None, rows=A, rows_dtype=0, rows_ld=576, norm_w=None, eps=1e-5, inv_freq=None, style=0, H=2, q=A, q_dtype=0,
              q_ld=128, q_head=64, q_out=A, q_out_dtype=1, q_out_ld=1152, q_out_head=576, stream=None)
ATTENTION = dict(B=1, N=4, H=8, kv_lora=512, rope=64, scale=0.1, q=A, pages=A, dtype=1, n_pages=8, page=16, table=A, max_pages=4,
                 lens=A, counts=None, parents=None, o=A, o_dtype=1, lse=None, ws=None, ws_bytes=0, stream=None)
COMMIT = dict(B=1, N=4, width=576, pages=A, dtype=1, n_pages=8, page=16, table=A, max_pages=4, lens=A, counts=None, parents=None,
              accept=A, lens_out=None, stream=None)
STEP = dict(B=1, N=4, H=2, D=128, K=4, lb=-5.0, eps=1e-5, in_dtype=1, q=A, k=A, v=A, z=A, b=A, gate=A, gate_dtype=1, qc=A, kc=A, vc=A,
            A_log=A, dt_bias=A, o_norm=A, conv=A, conv_stride=3 * 256 * 3, q_scale=0.1, S=A, s_stride=2 * 128 * 128, counts=None,
            parents=None, y=A, y_dtype=0, stream=None)
KCOMMIT = dict(B=1, N=4, H=2, D=128, K=4, lb=-5.0, in_dtype=1, q=A, k=A, v=A, z=A, b=A, qc=A, kc=A, vc=A, A_log=A, dt_bias=A, conv=A,
               conv_stride=3 * 256 * 3, S=A, s_stride=2 * 128 * 128, counts=None, parents=None, accept=A, stream=None)
PAGED = [("B", -1, "EINVAL"), ("N", -1, "EINVAL"), ("n_pages", 0, "EINVAL"), ("page", 0, "EINVAL"), ("max_pages", 0, "EINVAL"),
         ("max_pages", 1 << 29, "EINVAL"), ("pages", None, "EINVAL"), ("table", None, "EINVAL"), ("lens", None, "EINVAL"),
         ("dtype", 3, "EINVAL")]
LAYER = [("B", -1, "EINVAL"), ("N", -1, "EINVAL"), ("N", 65, "EUNSUPPORTED"), ("H", 0, "EINVAL"), ("D", 48, "EUNSUPPORTED"),
         ("K", 5, "EUNSUPPORTED"), ("K", 0, "EUNSUPPORTED"), ("lb", 0.5, "EINVAL"), ("lb", float("nan"), "EINVAL"),
         ("in_dtype", 3, "EINVAL"), ("s_stride", 2 * 128 * 128 - 4, "EINVAL"), ("s_stride", 2 * 128 * 128 + 2, "EINVAL"),
         ("conv_stride", 100, "EINVAL"), ("conv", None, "EINVAL"), ("S", None, "EINVAL"), ("S", ODD, "EINVAL"), ("z", None, "EINVAL"),
         ("v", None, "EINVAL"), ("B", 65536, "EINVAL")]


@pytest.mark.parametrize("name,defaults,arg,value,code", [
    *[("k3hip_latent_append", APPEND, *c) for c in PAGED],
    ("k3hip_latent_append", APPEND, "rope", 7, "EINVAL"),
    ("k3hip_latent_append", APPEND, "rope", 258, "EINVAL"),
    ("k3hip_latent_append", APPEND, "kv_lora", 0, "EINVAL"),
    ("k3hip_latent_append", APPEND, "rows", None, "EINVAL"),
    ("k3hip_latent_append", APPEND, "rows_ld", 575, "EINVAL"),
    ("k3hip_latent_append", APPEND, "rows_dtype", 2, "EINVAL"),
    ("k3hip_latent_append", APPEND, "style", 2, "EINVAL"),
    ("k3hip_latent_append", APPEND, "q_out", None, "EINVAL"),
    ("k3hip_latent_append", APPEND, "q_head", 63, "EINVAL"),
    ("k3hip_latent_append", APPEND, "q_dtype", 9, "EINVAL"),
    ("k3hip_latent_append", APPEND, "H", 0, "EINVAL"),
    *[("k3hip_mla_tree_attention", ATTENTION, *c) for c in PAGED],
    ("k3hip_mla_tree_attention", ATTENTION, "N", 65, "EUNSUPPORTED"),
    ("k3hip_mla_tree_attention", ATTENTION, "kv_lora", 520, "EUNSUPPORTED"),
    ("k3hip_mla_tree_attention", ATTENTION, "rope", 72, "EUNSUPPORTED"),
    ("k3hip_mla_tree_attention", ATTENTION, "rope", 4, "EUNSUPPORTED"),
    ("k3hip_mla_tree_attention", ATTENTION, "scale", 0.0, "EINVAL"),
    ("k3hip_mla_tree_attention", ATTENTION, "scale", float("nan"), "EINVAL"),
    ("k3hip_mla_tree_attention", ATTENTION, "H", 0, "EINVAL"),
    ("k3hip_mla_tree_attention", ATTENTION, "q", None, "EINVAL"),
    ("k3hip_mla_tree_attention", ATTENTION, "q", ODD, "EINVAL"),
    ("k3hip_mla_tree_attention", ATTENTION, "pages", ODD, "EINVAL"),
    ("k3hip_mla_tree_attention", ATTENTION, "o_dtype", 3, "EINVAL"),
    *[("k3hip_latent_commit", COMMIT, *c) for c in PAGED],
    ("k3hip_latent_commit", COMMIT, "N", 65, "EUNSUPPORTED"),
    ("k3hip_latent_commit", COMMIT, "width", 0, "EINVAL"),
    ("k3hip_latent_commit", COMMIT, "accept", None, "EINVAL"),
    *[("k3hip_kda_tree_step", STEP, *c) for c in LAYER],
    ("k3hip_kda_tree_step", STEP, "gate", None, "EINVAL"),
    ("k3hip_kda_tree_step", STEP, "y", None, "EINVAL"),
    ("k3hip_kda_tree_step", STEP, "y_dtype", 3, "EINVAL"),
    ("k3hip_kda_tree_step", STEP, "gate_dtype", 2, "EINVAL"),
    *[("k3hip_kda_tree_commit", KCOMMIT, *c) for c in LAYER],
    ("k3hip_kda_tree_commit", KCOMMIT, "accept", None, "EINVAL"),
])
def test_refused(name, defaults, arg, value, code):
    rc, msg = call(name, defaults, **{arg: value})
    assert rc == getattr(k3kda, code), (rc, msg)
    assert msg.startswith(name)


def test_tree_with_many_nodes_is_refused_a_chain_is_not():
    rc, _ = call("k3hip_latent_append", APPEND, N=65, parents=A)
    assert rc == k3kda.EUNSUPPORTED
    rc, _ = call("k3hip_latent_append", APPEND, N=65, B=0)
    assert rc == k3kda.OK


def test_workspace_of_calls_that_are_refused():
    L = k3kda.lib()
    for bad in ((0, 1, 1, 512), (1, 65, 1, 512), (1, 1, 0, 512), (1, 1, 1, 513)):
        assert L.k3hip_mla_tree_workspace(*bad) == 0


def test_binding_refuses_host_and_misshapen_tensors():
    import torch
    z = lambda *s: torch.zeros(s)  # noqa: E731
    with pytest.raises(ValueError):
        k3kda.latent_append(z(1, 2, 72), z(2, 16, 80), z(1, 1), z(1), 64)
    with pytest.raises(ValueError):
        k3kda.latent_append(z(1, 2, 72), z(2, 16, 72), z(1, 1), z(1), 64)
    with pytest.raises(ValueError):
        k3kda.mla_tree_attention(z(1, 2, 3, 72), z(2, 16, 72).bfloat16(), z(1, 1), z(1), z(1, 2, 3, 64), 64, 0.1)
    with pytest.raises(ValueError):
        k3kda.latent_commit(z(2, 16, 72), z(1, 1), z(1), z(1), 2)


def test_rotated_queries_that_overlap_are_refused():
    rc, msg = call("k3hip_latent_append", APPEND, q_out_ld=63)
    assert rc == k3kda.EINVAL and msg.startswith("k3hip_latent_append")
