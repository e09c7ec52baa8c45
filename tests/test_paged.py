"""Many sequences at once: the rotations' frequencies, and the refusals that need
no device: they come before any HIP call, with the outputs untouched (CPU)."""
from __future__ import annotations

import ctypes as C
import math
import pathlib
import subprocess

import numpy as np
import pytest

from conftest import gncx

ROOT = pathlib.Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def plib():
    return gncx.load()


def refused(lib, text):
    assert lib.gncx_hip_last_status() != 0
    assert text in lib.gncx_hip_last_error().decode()


# ---- frequencies ----------------------------------------------------------------------
def frequencies(lib, n_rot, base=1e6, scaling=0, factor=1.0, trained=32768, fast=32.0, slow=1.0, factors=None):
    out, mag = np.full(max(n_rot // 2, 1), -7.0), C.c_float(-7.0)
    lib.gncx_hip_last_status()
    rc = lib.gncx_hip_rope_frequencies(n_rot, base, scaling, factor, trained, fast, slow,
                                       None if factors is None else factors.ctypes.data, out.ctypes.data,
                                       C.addressof(mag))
    return rc, out, mag.value


@pytest.mark.parametrize("n_rot", [2, 24, 64, 128, 256])
@pytest.mark.parametrize("base", [1e4, 1e6])
def test_plain_and_linear_frequencies(plib, n_rot, base):
    want = base ** (-2.0 * np.arange(n_rot // 2) / n_rot)
    rc, got, mag = frequencies(plib, n_rot, base)
    assert rc == 0 and mag == 1.0
    np.testing.assert_allclose(got, want, rtol=1e-14)
    rc, got, mag = frequencies(plib, n_rot, base, gncx.ROPE_LINEAR, 4.0)
    assert rc == 0 and mag == 1.0
    np.testing.assert_allclose(got, want / 4.0, rtol=1e-14)


def test_base_scaling_stretches_the_slowest_pair_by_the_factor(plib):
    # the last pair's exponent is (n - 2) / n, so factor^(n / (n - 2)) of the base is the factor
    for n in (64, 128):
        plain = frequencies(plib, n, 1e4)[1]
        rc, got, mag = frequencies(plib, n, 1e4, gncx.ROPE_BASE, 8.0)
        assert rc == 0 and mag == 1.0 and got[0] == 1.0
        assert math.isclose(got[-1], plain[-1] / 8.0, rel_tol=1e-13)
        assert (np.diff(got / plain) < 0).all()


@pytest.mark.parametrize("n_rot,base,trained", [(128, 1e6, 32768), (64, 1e4, 4096), (128, 1e4, 2048)])
def test_yarn_keeps_fast_pairs_and_stretches_slow_ones(plib, n_rot, base, trained):
    plain = frequencies(plib, n_rot, base)[1]
    rc, got, mag = frequencies(plib, n_rot, base, gncx.ROPE_YARN, 4.0, trained)
    assert rc == 0 and math.isclose(mag, 0.1 * math.log(4.0) + 1.0, rel_tol=2e-7)
    turns = trained * plain / (2 * math.pi)  # within the trained context
    share = (got / plain - 0.25) / 0.75      # 1: as it is, 0: divided by the factor
    # pairs well on either side (the borders are rounded outwards to whole pairs)
    step = plain[0] / plain[1]
    assert np.allclose(share[turns > 32 * step], 1.0, atol=1e-12)
    assert np.allclose(share[turns < 1 / step], 0.0, atol=1e-12)
    mixed = (turns < 30) & (turns > 1.1)
    assert ((share[mixed] > 0) & (share[mixed] < 1)).all() and (np.diff(share) <= 1e-15).all()


def test_factors_divide_and_zero_leaves(plib):
    fac = np.linspace(1, 8, 32, dtype=np.float32)
    fac[5] = 0
    plain = frequencies(plib, 64)[1]
    rc, got, _ = frequencies(plib, 64, factors=fac)
    assert rc == 0
    np.testing.assert_allclose(got, plain / np.where(fac == 0, 1, fac), rtol=1e-14)


@pytest.mark.parametrize("bad", [dict(n_rot=0), dict(n_rot=3), dict(n_rot=1026), dict(n_rot=-2), dict(base=0.0),
                                 dict(base=-1.0), dict(base=math.nan), dict(base=math.inf), dict(scaling=4),
                                 dict(scaling=-1), dict(scaling=1, factor=0.0), dict(scaling=3, factor=math.nan),
                                 dict(scaling=3, factor=2.0, trained=0), dict(scaling=3, factor=2.0, base=1.0),
                                 dict(scaling=3, factor=2.0, fast=0.0), dict(scaling=3, factor=2.0, slow=-1.0),
                                 dict(scaling=2, factor=2.0, n_rot=2)])
def test_frequencies_refuse(plib, bad):
    rc, got, mag = frequencies(plib, **{"n_rot": 64, **bad})
    assert rc == -1 and (got == -7.0).all() and mag == -7.0
    refused(plib, "n_rot is even")


def test_frequencies_without_output(plib):
    assert plib.gncx_hip_rope_frequencies(64, 1e4, 0, 1.0, 0, 0.0, 0.0, None, None, None) == -1
    refused(plib, "no output")
    out = np.zeros(32)
    assert plib.gncx_hip_rope_frequencies(64, 1e4, 3, 2.0, 4096, 32.0, 1.0, None, out.ctypes.data, None) == -1
    refused(plib, "no output")
    assert plib.gncx_hip_rope_frequencies(64, 1e4, 0, 1.0, 0, 0.0, 0.0, None, out.ctypes.data, None) == 0
    assert out[0] == 1.0


# ---- refusals -------------------------------------------------------------------------------
def cache(**over):
    f = dict(k_pages=None, v_pages=None, scales=None, n_pages=4, page_tokens=32, n_kv_heads=2, head_dim=64)
    return gncx.PagedCache(**{**f, **over})


def batch(**over):
    f = dict(n_seqs=2, n_rows=3, max_pages=4, row_start=None, lengths=None, pages=None)
    return gncx.PagedBatch(**{**f, **over})


def attend(lib, c, b, heads=4):
    out = np.full(8, 7.0, np.float32)
    lib.gncx_hip_last_status()
    lib.gncx_hip_attention_paged(None if c is None else C.byref(c), None if b is None else C.byref(b), None, heads, 1.0,
                                 0, out.ctypes.data)
    assert (out == 7.0).all()


def append(lib, c, b, heads=4, weight=-1):
    out = np.full(8, 7.0, np.float32)
    lib.gncx_hip_last_status()
    lib.gncx_hip_kv_append_paged(None if c is None else C.byref(c), None if b is None else C.byref(b), None, None, None,
                                 heads, None, 0, 0, weight, 1e-6, None, out.ctypes.data)
    assert (out == 7.0).all()


@pytest.mark.parametrize("call", [attend, append])
def test_paged_refuses_geometry(plib, call):
    for c in (cache(head_dim=96), cache(head_dim=0), cache(n_kv_heads=0), cache(n_kv_heads=3), cache(n_pages=0),
              cache(page_tokens=8), cache(page_tokens=48), cache(page_tokens=512), cache(page_tokens=0),
              cache(n_kv_heads=65536)):
        call(plib, c, batch())
        refused(plib, "invalid cache geometry")
    for heads in (0, 3, -4, 65536):
        call(plib, cache(), batch(), heads)
        refused(plib, "invalid cache geometry")
    for b in (batch(n_seqs=0), batch(n_seqs=65537), batch(n_rows=-1), batch(max_pages=0), batch(max_pages=2 ** 25 + 1),
              batch(n_rows=2 ** 29)):
        call(plib, cache(), b)
        refused(plib, "invalid batch")
    call(plib, None, batch())
    refused(plib, "no cache or batch")
    call(plib, cache(), None)
    refused(plib, "no cache or batch")


def test_append_refuses_missing_norm_weights(plib):
    append(plib, cache(), batch(), weight=1)
    refused(plib, "no norm weights")


def test_rope_rows_refuses_geometry(plib):
    out = np.full(8, 7.0, np.float32)
    for rows, stride, heads, hd, ostride in ((-1, 64, 1, 64, 64), (1, 64, 0, 64, 64), (1, 64, 1, 63, 64),
                                             (1, 64, 1, 0, 64), (1, 2048, 1, 1026, 2048), (1, 127, 2, 64, 128),
                                             (1, 128, 2, 64, 127), (1, -128, 1, 64, 128), (1, 2 ** 30, 65536, 2, 2 ** 30)):
        plib.gncx_hip_last_status()
        plib.gncx_hip_rope_rows(None, rows, stride, heads, hd, None, None, ostride, out.ctypes.data)
        refused(plib, "head_dim is even")
    assert (out == 7.0).all()


def test_logprobs_refuse_sizes_and_lone_outputs(plib):
    out = np.full(8, 7.0, np.float32)
    o = out.ctypes.data
    for rows, vocab, top in ((-1, 10, 0), (1, 0, 0), (1, 2 ** 22 + 1, 0), (1, 10, -1), (1, 10, 65)):
        plib.gncx_hip_last_status()
        plib.gncx_hip_token_logprobs(None, rows, vocab, None, top, None, o, o, o)
        refused(plib, "0 to 64 alternatives")
    for tokens, logp, top, words, best in ((None, o, 0, None, None), (o, None, 0, None, None), (None, None, 1, None, o),
                                           (None, None, 1, o, None)):
        plib.gncx_hip_last_status()
        plib.gncx_hip_token_logprobs(None, 1, 10, tokens, top, logp, None, words, best)
        refused(plib, "come with")
    assert (out == 7.0).all()


def test_no_rows_are_no_error(plib):
    plib.gncx_hip_last_status()
    attend(plib, cache(), batch(n_rows=0))
    append(plib, cache(), batch(n_rows=0))
    plib.gncx_hip_rope_rows(None, 0, 0, 0, 0, None, None, 0, None)
    plib.gncx_hip_token_logprobs(None, 0, 0, None, 0, None, None, None, None)
    assert plib.gncx_hip_last_status() == 0


def test_structs_match_header(tmp_path):
    """The ctypes mirrors have the layout that the header declares."""
    py = {"GNCXPagedCache": gncx.PagedCache, "GNCXPagedBatch": gncx.PagedBatch, "GNCXRotation": gncx.Rotation}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "gncx_llm_core.h"', "int main(void) {"]
    for s, t in py.items():
        lines.append(f'printf("{s} sizeof %zu\\n", sizeof({s}));')
        lines += [f'printf("{s} {f} %zu\\n", offsetof({s}, {f}));' for f, _ in t._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    for ln in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        s, f, v = ln.split()
        assert (C.sizeof(py[s]) if f == "sizeof" else getattr(py[s], f).offset) == int(v), (s, f)


# ---- the decode driver -----------------------------------------------------------------
class Stand:
    """A stand-in model whose next id is 3 t + 1 (and 0 the second choice), over sequences
    that only count; the passes' rows."""

    def __init__(self, dec, monkeypatch, vocab=50):
        import types
        import torch
        self.torch, self.scale, self.hidden, self.lib, self.m = torch, 1.0, torch.zeros(vocab), None, None
        self.s = types.SimpleNamespace(vocab=vocab, embed=vocab)
        self.passes, stand = [], self

        class Counts:
            def __init__(self, lib, torch, model, room, *_):
                self.room, self.lengths = room, [0] * len(room)

            def begin(self, counts):
                stand.passes.append(counts)
                self.counts = counts

            def end(self):
                self.lengths = [a + n for a, n in zip(self.lengths, self.counts)]
                assert all(a <= r for a, r in zip(self.lengths, self.room))

        monkeypatch.setattr(dec, "PagedSequences", Counts)
        monkeypatch.setattr(dec, "check", lambda lib: None)

    def _device_only(self, what):
        pass

    def _rows_normed(self, tokens, attention, keep=None):
        assert len(tokens) == sum(self.passes[-1])
        return self.torch.nn.functional.one_hot(self.torch.tensor(tokens), self.s.vocab).float()[
            range(len(tokens)) if keep is None else keep]

    def _rows_head(self, rows):
        t = rows.argmax(1)
        return self.torch.nn.functional.one_hot((3 * t + 1) % self.s.vocab, self.s.vocab).float()

    def _logprobs(self, logits, tokens=None, n_top=0):
        top = self.torch.topk(logits.log_softmax(1), n_top)
        return None, None, top.indices.int(), top.values


@pytest.mark.parametrize("at_once", [1, 2, 3, 7, 100])
def test_generate_batch_fills_its_passes(plib, monkeypatch, at_once):
    import gncx_amd.decode as dec
    d = Stand(dec, monkeypatch)
    prompts, n_new = [[5], [1, 2, 3, 4], [9, 8], [7] * 9, [2]], 4
    got = dec.Decoder.generate_batch(d, prompts, n_new, n_top=1, rows_at_once=at_once)
    follow = lambda t, n: [t := (3 * t + 1) % 50 for _ in range(n)]  # noqa: E731
    assert [ids for ids, _, _ in got] == [follow(p[-1], n_new) for p in prompts]
    assert all(len(lps) == len(tops) == n_new and top[0] == (t, lp) and len(top) == 1
               for ids, lps, tops in got for t, lp, top in zip(ids, lps, tops))
    first = d.passes[:-(n_new - 1)]
    assert [sum(c) for c in zip(*first)] == [len(p) for p in prompts]
    assert [sum(c) for c in first] == [at_once] * (17 // at_once) + [17 % at_once] * (17 % at_once > 0)
    assert d.passes[-(n_new - 1):] == [[1] * 5] * (n_new - 1)
    # 16 = 3 * 5 + 1 ends the first sequence at once
    d.passes.clear()
    got = dec.Decoder.generate_batch(d, prompts, n_new, end=16)
    assert got[0][0] == [16] and got[0][2] == [[]] and d.passes[1][0] == 0
    assert all(ids == (full[:full.index(16) + 1] if 16 in full else full)
               for (ids, _, _), full in zip(got, (follow(p[-1], n_new) for p in prompts)))


def test_driver_refusals(plib, monkeypatch):
    import gncx_amd.decode as dec
    d = Stand(dec, monkeypatch)
    for args, kw in ((([], 3), {}), (([[1], []], 3), {}), (([[1]], 0), {}), (([[1]], 1), dict(page=48)),
                     (([[1]], 1), dict(n_top=65)), (([[1]], 1), dict(rows_at_once=0)), (([[50]], 1), {}), (([[-1]], 1), {})):
        with pytest.raises(ValueError):
            dec.Decoder.generate_batch(d, *args, **kw)
    d.max_seq = 3
    for ids, top in (([], 0), ([1], 0), ([1] * 5, 0), ([1, 2], 65), ([1, 2], -1)):
        with pytest.raises(ValueError):
            dec.Decoder.score(d, ids, top)
    assert not d.passes
    import types
    import torch
    host = types.SimpleNamespace(hidden=torch.zeros(1))
    host._device_only = lambda what: dec.Decoder._device_only(host, what)
    for call in (lambda: dec.Decoder.generate_batch(host, [[1]], 1), lambda: dec.Decoder.score(host, [1, 2])):
        with pytest.raises(ValueError, match="device memory"):
            call()


def test_sequences_refuse_factors_that_are_not_the_models(plib):
    """The library reads head_dim / 2 floats where the tensor's memory begins."""
    import types
    import torch
    import gncx_amd.decode as dec
    model = types.SimpleNamespace(shape=types.SimpleNamespace(n_layers=1, n_kv=1, head_dim=64, rope_base=1e4))
    make = lambda f: dec.PagedSequences(plib, torch, model, [5], 16, dict(factors=f), "cpu")  # noqa: E731
    plain = make(None).freqs
    assert torch.equal(make(torch.full((32,), 2.0)).freqs, plain / 2)
    for f in (torch.ones(31), torch.ones(64), torch.ones(32, dtype=torch.float64), torch.ones(64)[::2],
              torch.ones(32, dtype=torch.float16)):
        with pytest.raises(ValueError, match="factors"):
            make(f)


def test_driver_refuses_ids_and_sizes_before_a_pass(plib, monkeypatch):
    """Ids outside the vocabulary (a pass would leave the decoder's caches without them, and a
    last one gets -inf), and more rows than the embedding rows' call takes."""
    import gncx_amd.decode as dec
    d = Stand(dec, monkeypatch)
    d.max_seq = 10 ** 6
    for ids in ([50, 1], [1, 50], [1, -1, 2], [1] * 65537):
        with pytest.raises(ValueError):
            dec.Decoder.score(d, ids)
    for prompts, kw in (([[1]] * 65536, {}), ([[1]], dict(rows_at_once=65536))):
        with pytest.raises(ValueError):
            dec.Decoder.generate_batch(d, prompts, 1, **kw)
    assert not d.passes
