"""Refusals of the entries for several continuations that need no device: they
come before any HIP call, with the outputs untouched (CPU)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from conftest import gncx


@pytest.fixture(scope="module")
def plib():
    return gncx.load()


def refused(lib, text):
    assert lib.gncx_hip_last_status() != 0
    assert text in lib.gncx_hip_last_error().decode()


def tree(lib, parents, n=None, pos0=0, H=4, KV=2, hd=64, weight=-1, factors=0, base=0.0):
    p = None if parents is None else np.asarray(parents, np.int32)
    out = np.full(8, 7.0, np.float32)
    lib.gncx_hip_last_status()
    lib.gncx_hip_attention_tree(None, None, None, None, None, pos0, len(parents) if n is None else n,
                                None if p is None else p.ctypes.data, H, KV, hd, 1.0, 0, None, 0, 0, weight, 1e-6, 0,
                                factors, base, out.ctypes.data)
    assert (out == 7.0).all()


@pytest.mark.parametrize("parents", [[0], [1, -1], [-1, 1], [-1, 0, 2], [-2], [-1, -3], [-1, 2, 1], [-1] * 513])
def test_tree_refuses_what_is_no_tree(plib, parents):
    tree(plib, parents)
    refused(plib, "every parent is -1 or an earlier node")


def test_tree_refuses_negative_and_missing(plib):
    tree(plib, [-1], n=-1)
    refused(plib, "1 to 512 nodes")
    tree(plib, None, n=1)
    refused(plib, "parents must be host memory")
    tree(plib, [-1], weight=1)
    refused(plib, "no norm weights")
    tree(plib, [-1], factors=1, base=1e4)
    refused(plib, "rope factors")


@pytest.mark.parametrize("geo", [dict(H=3), dict(H=0), dict(KV=0), dict(hd=96), dict(hd=0), dict(pos0=-1),
                                 dict(H=8193, KV=1),
                                 dict(pos0=2 ** 31 - 512)])
def test_tree_refuses_geometry(plib, geo):
    tree(plib, [-1], **geo)
    refused(plib, "invalid head geometry")


def test_no_nodes_and_no_rows_are_no_error(plib):
    plib.gncx_hip_last_status()
    tree(plib, [])
    plib.gncx_hip_kv_keep_rows(None, None, 1, 64, 0, None, 0)
    plib.gncx_hip_kv_reorder(None, None, 1, 2, 64, 64, 0, 0, None)
    assert plib.gncx_hip_last_status() == 0


@pytest.mark.parametrize("rows", [[1, 1], [2, 1], [-1], [0, 65536]])
def test_keep_refuses_rows_out_of_order(plib, rows):
    r, none = np.asarray(rows, np.int32), (C.c_void_p * 1)()
    plib.gncx_hip_kv_keep_rows(none, none, 1, 64, 0, r.ctypes.data, len(rows))
    refused(plib, "ascend strictly")


@pytest.mark.parametrize("kv_dim,row0,n", [(6, 0, 1), (0, 0, 1), (64, -1, 1), (64, 0, 513), (64, 0, -1),
                                           (2 ** 24 + 4, 0, 1)])
def test_keep_refuses_sizes(plib, kv_dim, row0, n):
    r, none = np.arange(max(n, 1), dtype=np.int32), (C.c_void_p * 1)()
    plib.gncx_hip_kv_keep_rows(none, none, 1, kv_dim, row0, r.ctypes.data, n)
    refused(plib, "multiple of 4")


@pytest.mark.parametrize("beams,vocab,n_out", [(0, 10, 1), (33, 10, 1), (1, 0, 1), (1, 2 ** 22 + 1, 1), (1, 10, 0),
                                               (1, 10, 65)])
def test_select_refuses_sizes(plib, beams, vocab, n_out):
    plib.gncx_hip_beam_select(None, beams, vocab, None, None, 0, n_out, None, None, None)
    refused(plib, "beams")


@pytest.mark.parametrize("token", [-1, 10])
def test_select_refuses_a_finished_token_outside_the_vocabulary(plib, token):
    done = np.zeros(2, np.int32)
    plib.gncx_hip_beam_select(None, 2, 10, None, done.ctypes.data, token, 1, None, None, None)
    refused(plib, "finished_token")


@pytest.mark.parametrize("beams,stride,kv_dim,row0,n", [(0, 64, 64, 0, 1), (33, 64, 64, 0, 1), (2, 63, 64, 0, 1),
                                                        (2, 66, 64, 0, 1), (2, 128, 6, 0, 1), (2, 128, 64, 1, 2),
                                                        (2, 128, 64, -1, 1), (2, 128, 64, 0, -1),
                                                        (2, 2 ** 62, 64, 0, 1), (2, 2 ** 25, 2 ** 24 + 4, 0, 1)])
def test_reorder_refuses_sizes(plib, beams, stride, kv_dim, row0, n):
    none = (C.c_void_p * 1)()
    plib.gncx_hip_kv_reorder(none, none, 1, beams, stride, kv_dim, row0, n, None)
    refused(plib, "1 to 32 beams")


@pytest.mark.parametrize("layers", [0, -1, 4097, 2 ** 31 - 1])
def test_caches_refuse_numbers_of_layers(plib, layers):
    r, none = np.zeros(1, np.int32), (C.c_void_p * 1)()
    plib.gncx_hip_kv_keep_rows(none, none, layers, 64, 0, r.ctypes.data, 1)
    refused(plib, "at least one layer")
    plib.gncx_hip_kv_reorder(none, none, layers, 2, 64, 64, 0, 1, None)
    refused(plib, "at least one layer")


@pytest.mark.parametrize("ids,tokens,parents", [
    ([], [], []), ([7], [], []), ([1, 2, 3], [], []),
    ([4, 9, 8, 4], [9, 8, 4], [-1, 0, 1]),  # no earlier pair: behind the last id
    ([1, 2, 3, 4, 1, 2, 5, 6, 1, 2], [5, 6, 1, 2, 3, 4, 1, 2, 5, 6, 1, 2],
     [-1, 0, 1, 2, -1, 4, 5, 6, 7, 8, 9, 10]),
    ([3, 3, 3, 3], [3, 3], [-1, 0]),  # branches that begin alike are one
])
def test_lookup_draft(ids, tokens, parents):
    import gncx_amd.decode as dec
    assert dec.lookup_draft(ids) == (tokens, parents)


def test_lookup_draft_has_a_depth_and_a_width():
    import gncx_amd.decode as dec
    ids = [x for i in range(10) for x in (1, 2, 10 + i, 20 + i, 30 + i)] + [1, 2]
    tokens, parents = dec.lookup_draft(ids, depth=2, width=3)
    assert (tokens, parents) == ([19, 29, 18, 28, 17, 27], [-1, 0, -1, 2, -1, 4])


def drafted(dec, next_of, prompt, n_new, draft, max_seq=64):
    """generate_drafted over a stand-in model whose greedy next id is next_of[id];
    the ids, and the paths it kept."""
    import types
    import torch
    logits = lambda t: torch.nn.functional.one_hot(torch.tensor(next_of[t]), len(next_of)).float()  # noqa: E731
    kept = []
    d = types.SimpleNamespace(torch=torch, max_seq=max_seq, prefill=lambda ids: logits(ids[-1]),
                              greedy=lambda x: int(x.argmax()),
                              verify_tree=lambda tokens, parents, pos: torch.stack([logits(t) for t in tokens]),
                              keep_path=lambda pos, path: kept.append((pos, list(path))))
    return dec.Decoder.generate_drafted(d, prompt, n_new, draft), kept


def test_drafted_generation_takes_the_longest_of_equal_branches():
    """Two drafted nodes of one token below the same node: the branch that is
    accepted further is kept, whichever comes first."""
    import gncx_amd.decode as dec
    next_of = [1, 2, 3, 4, 5, 6, 7, 0]
    # below the chosen token 1: the token 2 twice; below the second, 3 and 4
    draft = lambda ids: ([2, 7, 2, 3, 4, 5], [-1, 0, -1, 2, 3, 0])  # noqa: E731
    new, kept = drafted(dec, next_of, [0], 5, draft)
    assert new == [1, 2, 3, 4, 5] and kept[0] == (1, [0, 3, 4, 5])
    # equally long ones: the first
    draft = lambda ids: ([2, 2, 3, 3], [-1, -1, 1, 0])  # noqa: E731
    new, kept = drafted(dec, next_of, [0], 4, draft)
    assert new == [1, 2, 3, 4] and kept[0] == (1, [0, 2, 3])


@pytest.mark.parametrize("n_new", range(1, 9))
def test_drafted_generation_stops_at_the_number_of_ids(n_new):
    import gncx_amd.decode as dec
    next_of = [1, 2, 3, 4, 5, 6, 7, 0]
    draft = lambda ids: ([next_of[ids[-1]], 0, next_of[next_of[ids[-1]]]], [-1, 0, 0])  # noqa: E731
    new, kept = drafted(dec, next_of, [5, 6], n_new, draft)
    assert new == [7, 0, 1, 2, 3, 4, 5, 6][:n_new]
    assert sum(len(p) for _, p in kept) <= n_new
