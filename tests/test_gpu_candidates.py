"""GPU: the operators for several continuations of one sequence, through the
C-ABI with device pointers, against 64-bit formulas: attention of a drafted
tree (its prologue bit for bit that of decode steps), the kept rows of an
accepted path, beam search's selection, and the reordering of the caches."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest

from conftest import gncx

pytestmark = pytest.mark.gpu
U = 2.0 ** -24  # half a step of fp32
EPS = 1e-6


def addresses(t):
    """ctypes array of the addresses of t's first axis."""
    step = t.stride(0) * t.element_size()
    return (C.c_void_p * t.shape[0])(*(t.data_ptr() + i * step for i in range(t.shape[0])))


def refused(lib, text):
    assert lib.gncx_hip_last_status() != 0
    assert text in lib.gncx_hip_last_error().decode()


# ---- trees --------------------------------------------------------------------------
def make_parents(shape, n, seed=0):
    if shape == "chain":
        return list(range(-1, n - 1))
    if shape == "roots":
        return [-1] * n
    if shape == "binary":
        return [(i - 1) // 2 if i else -1 for i in range(n)]
    rng = np.random.default_rng(seed + n)
    return [-1 if i == 0 or rng.random() < 0.1 else int(rng.integers(max(0, i - 9), i)) for i in range(n)]


def depths(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


class Tree:
    """Device buffers of one call; the caches have spare rows behind the nodes."""

    def __init__(self, torch, H, KV, hd, pos0, parents, sw=0, weight=-1, base=0.0, seed=0, spare=3):
        self.torch, self.H, self.KV, self.hd, self.pos0, self.sw = torch, H, KV, hd, pos0, sw
        self.parents, self.n, self.weight, self.base = list(parents), len(parents), weight, base
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.q, self.k, self.v = r(self.n, H * hd), r(self.n, KV * hd), r(self.n, KV * hd)
        self.kc, self.vc = r(pos0 + self.n + spare, KV * hd), r(pos0 + self.n + spare, KV * hd)
        self.gamma = 1 + 0.1 * r(2, hd)
        self.out = torch.full((self.n, H * hd), float("nan"), device="cuda")
        self.scale = 1 / math.sqrt(hd)

    def call(self, lib, check=True):
        p = np.asarray(self.parents, np.int32)
        lib.gncx_hip_attention_tree(self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), self.kc.data_ptr(),
                                    self.vc.data_ptr(), self.pos0, self.n, p.ctypes.data, self.H, self.KV, self.hd,
                                    self.scale, self.sw, self.gamma.data_ptr(), 0, 4 * self.hd, self.weight, EPS, 0, 0,
                                    self.base, self.out.data_ptr())
        p[:] = -7  # read before the call returned
        if check:
            gncx.check(lib)

    def visible(self):
        """[n][pos0 + n] by walking each node's ancestors."""
        d = depths(self.parents)
        see = np.zeros((self.n, self.pos0 + self.n), bool)
        for i in range(self.n):
            at = self.pos0 + d[i]
            low = max(0, at - self.sw + 1) if self.sw > 0 else 0
            see[i, low:self.pos0] = True
            a = i
            while a >= 0:
                see[i, self.pos0 + a] = self.pos0 + d[a] >= low
                a = self.parents[a]
        return see

    def reference(self):
        """64-bit outputs of the prologue's results (q and the cache rows as the
        call left them), and how far fp32 sums of pair products may be off:
        |ds| <= (2^-21 + 8 sqrt(hd) u) max_j scale sum_d |q_d k_jd| for a score
        (operands kept to 2^-22 each, rounding errors of hd additions taken as
        independent), and per output 2 ds + 2^-20 + 8 sqrt(N) u of
        sum_j w_j |v_j| / l (the weights, their split, the sum over N keys).
        An element far below its row's largest is kept as a pair of halves whose
        last bit is that of the row: to 2^-22 of a key row's largest element,
        which adds 2^-22 scale max_j |k_j|_max sum_d |q_d| to ds, and to 2^-25 of
        a value row's, which adds 2^-25 sum_j w_j |v_j|_max / l.
        A weight is an fp32 number relative to its row's largest, 1, and an
        output one by itself: below the smallest normal number, 2^-126, either
        may count as zero, so an output may be off by 2^-126 sum_j |v_j| / l
        and by 2^-126 besides."""
        torch, n, H, KV, hd = self.torch, self.n, self.H, self.KV, self.hd
        see = torch.from_numpy(self.visible()).cuda()
        keys = self.pos0 + n
        q = self.q.double().view(n, H, hd)
        kc, vc = (c[:keys].double().view(keys, KV, hd) for c in (self.kc, self.vc))
        want, tol = torch.empty_like(q), torch.empty_like(q)
        for h in range(H):
            k, v = kc[:, h // (H // KV)].contiguous(), vc[:, h // (H // KV)].contiguous()
            # rows that a node does not see may hold anything: one that nobody sees counts as zeros
            seen = see.any(0).unsqueeze(1)
            k, v = torch.where(seen, k, 0.0), torch.where(seen, v, 0.0)
            qh = q[:, h].contiguous()
            s = torch.where(see, qh @ k.t().contiguous() * self.scale, -math.inf)
            size = torch.where(see, qh.abs() @ k.abs().t().contiguous() * self.scale, 0.0).amax(1, keepdim=True)
            w = torch.exp(s - s.amax(1, keepdim=True))
            l = w.sum(1, keepdim=True) + 1e-12
            want[:, h] = w @ v / l
            ds = (2.0 ** -21 + 8 * math.sqrt(hd) * U) * size
            largest = torch.where(see, k.abs().amax(1) * qh.abs().sum(1, keepdim=True), 0.0)
            ds += 2.0 ** -22 * self.scale * largest.amax(1, keepdim=True)
            tol[:, h] = (2 * ds + 2.0 ** -20 + 8 * math.sqrt(keys) * U) * (w @ v.abs() / l)
            tol[:, h] += 2.0 ** -25 * (w @ v.abs().amax(1, keepdim=True) / l)
            tol[:, h] += 2.0 ** -126 * (see.double() @ v.abs() / l + 1)
        return want.view(n, H * hd), tol.view(n, H * hd)

    def verify(self, lib):
        k_behind, v_behind = self.kc[self.pos0 + self.n:].clone(), self.vc[self.pos0 + self.n:].clone()
        self.call(lib)
        want, tol = self.reference()
        off = (self.out.double() - want).abs()
        assert bool((off <= tol).all()), (float((off / tol).nan_to_num(nan=1e9).max()), float(off.max()))
        assert self.torch.equal(self.kc[self.pos0:self.pos0 + self.n], self.k)
        assert self.torch.equal(self.vc[self.pos0:self.pos0 + self.n], self.v)
        # rows behind the last node stay as they were
        assert self.torch.equal(self.kc[self.pos0 + self.n:], k_behind)
        assert self.torch.equal(self.vc[self.pos0 + self.n:], v_behind)


# heads: GQA, one group, odd group, MQA, groups of 16, many heads; widths 64, 128, 256
HEADS = [(32, 8, 128), (4, 4, 64), (12, 4, 128), (32, 1, 128), (8, 2, 256), (16, 1, 64), (64, 8, 128), (5, 1, 128)]


@pytest.mark.parametrize("H,KV,hd", HEADS)
@pytest.mark.parametrize("shape,n,pos0,sw", [("chain", 1, 0, 0), ("chain", 1, 1, 0), ("chain", 3, 31, 0),
                                             ("binary", 7, 32, 0), ("roots", 5, 33, 4), ("random", 17, 300, 0),
                                             ("random", 33, 127, 40), ("binary", 64, 700, 0), ("random", 2, 2049, 1)])
def test_tree_attention(lib, torch_mod, H, KV, hd, shape, n, pos0, sw):
    Tree(torch_mod, H, KV, hd, pos0, make_parents(shape, n), sw, seed=n + pos0).verify(lib)


@pytest.mark.parametrize("H,KV,hd,shape,n,pos0,sw", [
    (32, 8, 128, "random", 512, 100, 0), (32, 8, 128, "chain", 512, 1000, 77), (16, 16, 64, "random", 400, 1001, 600),
    (32, 4, 128, "binary", 130, 4001, 0), (32, 8, 128, "random", 25, 20011, 0), (32, 8, 128, "chain", 4, 16383, 1000),
    (32, 1, 128, "random", 65, 9000, 0), (8, 2, 256, "random", 129, 3001, 0), (8, 8, 64, "roots", 511, 2, 1),
    (2, 1, 64, "random", 100, 32000, 0), (12, 4, 128, "random", 300, 513, 0), (8, 1, 128, "chain", 4, 30000, 0),
    (4, 1, 64, "random", 40, 20000, 5000), (8, 2, 256, "random", 6, 12000, 0), (64, 1, 128, "binary", 3, 9001, 0)])
def test_tree_attention_large(lib, torch_mod, H, KV, hd, shape, n, pos0, sw):
    Tree(torch_mod, H, KV, hd, pos0, make_parents(shape, n), sw, seed=n).verify(lib)


@pytest.mark.parametrize("H,KV,hd", [(32, 8, 128), (4, 4, 64), (8, 2, 256)])
@pytest.mark.parametrize("weight", [1, 0])
def test_tree_prologue_is_that_of_decode_steps(lib, torch_mod, H, KV, hd, weight):
    """q, k and the cache rows of every node, bit for bit those of a fused decode
    step at the node's position."""
    torch = torch_mod
    t = Tree(torch, H, KV, hd, 1003, make_parents("random", 19), weight=weight, base=1e6, seed=5)
    q, k = t.q.clone(), t.k.clone()
    t.call(lib)
    out = torch.empty(H * hd, device="cuda")
    for i, d in enumerate(depths(t.parents)):
        kc, vc = torch.zeros(t.pos0 + d + 1, KV * hd, device="cuda"), torch.zeros(t.pos0 + d + 1, KV * hd, device="cuda")
        qi, ki = q[i].clone(), k[i].clone()
        lib.gncx_hip_attention_step_fused(qi.data_ptr(), ki.data_ptr(), t.v[i].data_ptr(), kc.data_ptr(),
                                          vc.data_ptr(), t.pos0 + d, H, KV, hd, t.scale, 0, 1, t.gamma.data_ptr(), 0,
                                          4 * hd, weight, EPS, 0, 0, t.base, out.data_ptr())
        gncx.check(lib)
        assert torch.equal(t.q[i], qi) and torch.equal(t.k[i], ki), i
    want, tol = t.reference()
    assert bool(((t.out.double() - want).abs() <= tol).all())


def test_tree_without_norms_rotates_as_the_rope_call(lib, torch_mod):
    torch = torch_mod
    H, KV, hd = 8, 2, 128
    t = Tree(torch, H, KV, hd, 77, make_parents("binary", 9), weight=-1, base=1e4, seed=2)
    q, k = t.q.clone(), t.k.clone()
    t.call(lib)
    for i, d in enumerate(depths(t.parents)):
        lib.gncx_apply_rope_xor11_ext(q[i].data_ptr(), k[i].data_ptr(), None, None, 0, 0, H, KV, hd, 77 + d, 1e4)
    gncx.check(lib)
    assert torch.equal(t.q, q) and torch.equal(t.k, k)


def test_tree_rope_frequency_factors(lib, torch_mod):
    torch = torch_mod
    H, KV, hd = 8, 2, 64
    t = Tree(torch, H, KV, hd, 40, make_parents("chain", 5), base=1e4, seed=3)
    fac = torch.linspace(1, 8, hd // 2, device="cuda")
    q = t.q.clone()
    p = np.asarray(t.parents, np.int32)
    lib.gncx_hip_attention_tree(t.q.data_ptr(), t.k.data_ptr(), t.v.data_ptr(), t.kc.data_ptr(), t.vc.data_ptr(), 40,
                                5, p.ctypes.data, H, KV, hd, t.scale, 0, fac.data_ptr(), 0, 0, -1, EPS, 0, 1, 1e4,
                                t.out.data_ptr())
    gncx.check(lib)
    k = t.k.clone()
    for i in range(5):
        lib.gncx_apply_rope_xor11_ext(q[i].data_ptr(), k[i].data_ptr(), None, fac.data_ptr(), 0, 1, H, KV, hd, 40 + i,
                                      1e4)
    assert torch.equal(t.q, q)


@pytest.mark.parametrize("H,KV,hd", [(32, 8, 128), (4, 4, 64), (8, 2, 256)])
@pytest.mark.parametrize("n", [6, 70])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_tree_hidden_rows_may_hold_anything(lib, torch_mod, H, KV, hd, n, bad):
    """Rows outside a node's window, its siblings' branches and the rows behind
    the last node have no part in its output."""
    torch = torch_mod
    # two chains from two roots; the second chain's rows are bad from its second node on
    parents = [-1, -1] + list(range(n - 2))
    t = Tree(torch, H, KV, hd, 90, parents, sw=60, seed=n)
    t.kc[:20], t.vc[:20] = bad, bad          # before every window (the first is 31..)
    t.kc[90 + n:], t.vc[90 + n:] = bad, bad
    for i in range(3, n, 2):
        t.k[i], t.v[i] = bad, bad
    t.call(lib)
    good = [i for i in range(n) if i % 2 == 0 or i == 1]
    out = t.out[good].clone()
    for i in range(3, n, 2):  # the reference's own products need finite rows
        t.kc[90 + i], t.vc[90 + i] = 0.0, 0.0
    want, tol = t.reference()
    off = (out.double() - want[good]).abs()
    assert bool((off <= tol[good]).all()), float(off.max())


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_tree_visible_infinities_and_nan_reach_their_own_nodes_only(lib, torch_mod, hd):
    torch = torch_mod
    H, KV, n, pos0 = 8, 2, 40, 50
    t = Tree(torch, H, KV, hd, pos0, make_parents("roots", n), seed=hd)
    t.v[3, 5] = float("inf")
    t.v[4, 6] = float("nan")
    t.k[7, :hd] = float("nan")    # KV head 0's key
    t.v[9] = 3.0e38
    t.call(lib)
    g, out = H // KV, t.out.view(n, H, hd)
    assert bool((out[3, :g, 5] == float("inf")).all()) and bool(out[4, :g, 6].isnan().all())
    assert bool(out[7, :g].isnan().all())
    assert bool((out[9].abs() > 1e30).all()) and bool(out[9].isfinite().all())
    clear = torch.ones(n, H, hd, dtype=torch.bool, device="cuda")
    clear[3, :g, 5], clear[4, :g, 6], clear[7, :g] = False, False, False
    for c in (t.kc, t.vc):
        c.copy_(c.nan_to_num(nan=0.0, posinf=0.0))
    want, tol = t.reference()
    off = (t.out.double() - want).abs().view(n, H, hd)
    # (outputs beside an infinite or NaN element of the same row are sums of finite values)
    assert bool((off[clear] <= tol.view(n, H, hd)[clear]).all())


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_tree_key_of_weight_zero(lib, torch_mod, hd):
    """A visible key whose score is -inf has weight 0."""
    torch = torch_mod
    t = Tree(torch, 4, 2, hd, 20, make_parents("binary", 5), seed=1)
    t.q.abs_()
    t.kc[4] = -float("inf")
    t.call(lib)
    t.kc[4] = -1e30
    want, tol = t.reference()
    # the key takes no part: bounds without its enormous products
    t.kc[4] = 0.0
    _, tol = t.reference()
    assert bool(((t.out.double() - want).abs() <= 2 * tol).all())


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("ks,vs", [(1e-6, 1e-6), (1.0, 1e6), (1e-3, 1e-30), (3.0, 1e30), (1e5, 1.0), (1e-20, 1e20)])
def test_tree_values_of_any_size(lib, torch_mod, hd, ks, vs):
    """Keys and values far from 1, and rows of very different sizes in one tile."""
    torch = torch_mod
    t = Tree(torch, 8, 2, hd, 200, make_parents("random", 21), seed=4)
    for c in (t.k, t.kc):
        c *= ks
    for c in (t.v, t.vc):
        c *= vs
    t.q *= min(1.0 / ks, 1e4)
    t.vc[60:70] *= 1e3
    t.verify(lib)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n", [5, 12, 40, 200])
@pytest.mark.parametrize("pos0", [0, 37])
def test_tree_neighbours_of_other_sizes(lib, torch_mod, hd, n, pos0):
    """First tokens that see themselves (and, with pos0, a few cached rows no
    larger than they are), of sizes from 0 to 1e30 side by side in a tile: each
    keeps the precision of its own size."""
    torch = torch_mod
    t = Tree(torch, 8, 2, hd, pos0, [-1] * n, seed=n)
    rng = np.random.default_rng(n)
    for rows, lo, hi in ((t.k, -25, 3), (t.v, -30, 30)):
        size = torch.from_numpy(10.0 ** rng.uniform(lo, hi, n)).float().cuda()
        size[rng.integers(n)] = 0.0
        rows *= size[:, None]
    t.kc[:pos0] *= 1e-25
    t.vc[:pos0] *= 1e-30
    if pos0:  # a row whose weight is 1 among cached ones
        t.k[:, ::7] = 0.0
    t.verify(lib)


@pytest.mark.parametrize("H,KV,hd,n,pos0", [(16, 16, 64, 400, 20000), (8, 8, 128, 20, 5000), (4, 1, 256, 3, 3000)])
def test_tree_many_rows_of_other_sizes(lib, torch_mod, H, KV, hd, n, pos0):
    """One row in eight far below its neighbours, over ranges of many tiles, and a
    few of them infinite where a window hides them."""
    torch = torch_mod
    t = Tree(torch, H, KV, hd, pos0, make_parents("random", n), sw=pos0 - 100, seed=n)
    t.vc[3:pos0:8] *= 1e-9
    t.kc[2:pos0:41] *= 1e-9
    t.vc[0] = float("inf")
    t.kc[1] = float("nan")
    t.verify(lib)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n", [6, 12, 40])
def test_tree_small_keys_beside_larger_ones(lib, torch_mod, hd, n):
    """Keys of 1e-5 to 1 side by side under large queries, where a key that is
    kept to the precision of a larger neighbour would change its score."""
    torch = torch_mod
    t = Tree(torch, 8, 2, hd, 2, [-1] * n, seed=n)
    rng = np.random.default_rng(n)
    t.k *= torch.from_numpy(10.0 ** rng.uniform(-5, 0, n)).float().cuda()[:, None]
    t.kc[:2] *= torch.from_numpy(10.0 ** rng.uniform(-5, -4, 2)).float().cuda()[:, None]
    t.q *= 1e4
    t.verify(lib)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("below,value", [(100, 1e33), (115, 3e36), (120, 3e36), (124, 1e38)])
def test_tree_large_value_of_a_small_weight(lib, torch_mod, hd, below, value):
    """A value row far above the others, under a weight of 2^-below: together
    they are most of the output."""
    torch = torch_mod
    t = Tree(torch, 8, 2, hd, 120, [-1, 0, 0], seed=hd)
    for c in (t.q, t.k, t.kc):
        c.zero_()
    t.q[:, ::hd] = 16.0
    t.kc[50, ::hd] = -below * math.log(2.0) / (16.0 * t.scale)
    t.vc[50] *= value
    t.verify(lib)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("size", [1e-8, 1.0, 1e9])
@pytest.mark.parametrize("exponent", [12, 14, 20])
def test_tree_scores_of_any_size(lib, torch_mod, hd, size, exponent):
    """Scores so far apart that one key has all the weight, and so large that
    32 bits hold no fraction of them: the output is that key's value row.  (Its
    elements are kept to 2^-22 of themselves or 2^-25 of the row's largest, and
    the sum of weights is 1.)"""
    torch = torch_mod
    H, KV, n, pos0 = 8, 2, 5, 140
    t = Tree(torch, H, KV, hd, pos0, [-1] * n, seed=hd)
    for c in (t.q, t.k, t.kc):
        c.zero_()
    # scores j 2^(2 exponent - 7) scale, in a random order of j, the nodes' own 0
    t.q[:, ::hd] = 2.0 ** exponent
    order = torch.from_numpy(np.random.default_rng(exponent).permutation(pos0)).cuda()
    for h in range(KV):
        t.kc[:pos0, h * hd] = (order + 1 + h) % (pos0 + 1) * 2.0 ** (exponent - 7)
    t.v *= size
    t.vc *= size
    t.call(lib)
    for h in range(H):
        kv = h // (H // KV)
        want = t.vc[int(t.kc[:pos0, kv * hd].argmax()), kv * hd:(kv + 1) * hd].double()
        off = (t.out[:, h * hd:(h + 1) * hd].double() - want).abs()
        assert bool((off <= 2.0 ** -21 * want.abs() + 2.0 ** -24 * want.abs().max()).all()), h


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("pos0,rows", [(200, [3, 9]), (300, [3, 150, 290]), (5000, range(0, 5000, 100)),
                                       (20000, [1, 19999])])
def test_tree_means_of_the_largest_values(lib, torch_mod, hd, pos0, rows):
    """Value rows near the largest float, whose sum is past it and whose mean is
    not, in one part of the keys and over many."""
    torch = torch_mod
    t = Tree(torch, 8, 2, hd, pos0, [-1, -1, 0], seed=hd)
    t.q.zero_()
    t.vc[list(rows)] = 3e38
    t.vc[rows[-1], ::3] = -3e38
    t.v[0] = 3e38
    t.verify(lib)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("big", [1e6, 1e20, 3e38])
@pytest.mark.parametrize("flat", [False, True])
def test_tree_value_rows_of_zeros_beside_hidden_ones(lib, torch_mod, hd, big, flat):
    """A value row of zeros takes nothing from the precision of the others,
    whatever rows that its node does not see stand beside it: an earlier branch's
    among the nodes, or one before the window at the start of a long range.  With
    equal scores (flat) every weight is 1 of all."""
    torch = torch_mod
    for pos0, sw in ((100, 0), (9000, 8900)):
        t = Tree(torch, 8, 2, hd, pos0, [-1] + list(range(-1, 6)) + [-1, 7, 7], sw=sw, seed=hd)
        t.v[0] = big                        # node 0 stands alone; the others do not see it
        t.v[1], t.v[3] = 0.0, 0.0
        first = max(0, pos0 - sw + 1) if sw else 0
        if sw:
            t.vc[first] = big               # only nodes without a parent see it
            t.vc[first + 5:first + 7] = 0.0
        t.vc[first + 40] = 0.0
        t.vc[first + 64:first + 72] = 0.0   # a whole group
        if flat:
            t.q.zero_()
        t.verify(lib)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_tree_nodes_that_see_zeros_alone(lib, torch_mod, hd):
    torch = torch_mod
    t = Tree(torch, 8, 2, hd, 37, [-1] * 9, seed=hd)
    t.vc.zero_()
    t.v[:4] = 0.0
    t.v[5] = 1e30
    t.verify(lib)
    assert not t.out[:4].any() and bool(t.out[5].all())


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("pos0", [60, 4000])
@pytest.mark.parametrize("size,below", [(1.0, 110), (1e-20, 55), (1e-33, 10)])
def test_tree_small_terms_under_rows_of_zeros(lib, torch_mod, hd, pos0, size, below):
    """Value rows of zeros have almost all of the weight; what is left for the
    others, 2^-below of small values, is the output."""
    torch = torch_mod
    t = Tree(torch, 8, 2, hd, pos0, [-1, 0, 0], seed=hd)
    for c in (t.q, t.k, t.kc):
        c.zero_()
    t.q[:, ::hd] = 16.0
    zeros = torch.arange(pos0, device="cuda")
    zeros = zeros[(zeros % 3 == 0) | (zeros // 8 % 3 == 0)]
    t.kc[zeros[:, None], torch.arange(0, 2 * hd, hd, device="cuda")] = below * math.log(2.0) / (16.0 * t.scale)
    t.v *= size
    t.vc *= size
    t.vc[zeros] = 0.0
    t.verify(lib)


def test_tree_is_a_prefill_for_a_chain(lib, torch_mod):
    torch = torch_mod
    H, KV, hd, pos0, n = 32, 8, 128, 300, 40
    t = Tree(torch, H, KV, hd, pos0, make_parents("chain", n), weight=1, base=1e6, seed=8)
    q, k, kc, vc = t.q.clone(), t.k.clone(), t.kc.clone(), t.vc.clone()
    out = torch.empty_like(q)
    t.call(lib)
    lib.gncx_hip_attention_prefill(q.data_ptr(), k.data_ptr(), t.v.data_ptr(), kc.data_ptr(), vc.data_ptr(), pos0, n,
                                   H, KV, hd, t.scale, 0, t.gamma.data_ptr(), 0, 4 * hd, 1, EPS, 0, 0, 1e6,
                                   out.data_ptr())
    gncx.check(lib)
    assert torch.equal(t.q, q) and torch.equal(t.kc, kc) and torch.equal(t.vc, vc)
    _, tol = t.reference()
    assert bool(((t.out - out).abs() <= 2 * tol).all())


def test_tree_past_4_gib(lib, torch_mod):
    """Cache rows past 2^32 bytes, read and written."""
    torch = torch_mod
    Tree(torch, 8, 8, 128, 1060000, [-1, 0, 0, 1], seed=1).verify(lib)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("H,KV,hd", [(32, 8, 128), (4, 4, 64), (8, 2, 256)])
@pytest.mark.parametrize("shape,sw", [("chain", 5), ("random", 40), ("random", 90), ("roots", 1)])
def test_tree_with_a_window_is_its_branches_decoded(lib, torch_mod, H, KV, hd, shape, sw):
    """Every node's output against a fused decode step with the same window, over
    a cache that holds the node's branch alone."""
    torch = torch_mod
    pos0, n = 83, 23
    t = Tree(torch, H, KV, hd, pos0, make_parents(shape, n), sw=sw, weight=1, base=1e6, seed=sw)
    q, k = t.q.clone(), t.k.clone()
    t.call(lib)
    _, tol = t.reference()
    d, out = depths(t.parents), torch.empty(H * hd, device="cuda")
    for i in range(n):
        branch, a = [], i
        while a >= 0:
            branch.insert(0, pos0 + a)
            a = t.parents[a]
        rows = list(range(pos0)) + branch
        kc, vc = t.kc[rows].clone(), t.vc[rows].clone()
        qi, ki = q[i].clone(), k[i].clone()
        lib.gncx_hip_attention_step_fused(qi.data_ptr(), ki.data_ptr(), t.v[i].data_ptr(), kc.data_ptr(),
                                          vc.data_ptr(), pos0 + d[i], H, KV, hd, t.scale, sw, 1, t.gamma.data_ptr(),
                                          0, 4 * hd, 1, EPS, 0, 0, t.base, out.data_ptr())
        gncx.check(lib)
        # (both are within the bound of the 64-bit formula)
        assert bool(((t.out[i].double() - out.double()).abs() <= 2 * tol[i]).all()), i


def test_tree_rows_in_the_cache_itself(lib, torch_mod):
    """k_nodes and v_nodes may be the cache rows that they are stored to."""
    torch = torch_mod
    a = Tree(torch, 8, 2, 128, 33, make_parents("binary", 11), weight=1, base=1e6, seed=9)
    b = Tree(torch, 8, 2, 128, 33, a.parents, weight=1, base=1e6, seed=9)
    b.kc[33:44], b.vc[33:44] = b.k, b.v
    b.k, b.v = b.kc[33:44], b.vc[33:44]
    a.call(lib)
    b.call(lib)
    assert torch.equal(a.out, b.out) and torch.equal(a.kc, b.kc) and torch.equal(a.vc, b.vc)


def test_tree_same_bits_every_time(lib, torch_mod):
    torch = torch_mod
    outs = []
    for _ in range(3):
        t = Tree(torch, 32, 8, 128, 3001, make_parents("random", 60), seed=10)
        t.call(lib)
        outs.append(t.out.clone())
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_tree_on_other_streams(lib, torch_mod):
    """Calls on two streams in turn, the library's stream changed between them."""
    torch = torch_mod
    trees = [Tree(torch, 32, 8, 128, 2000 + 300 * i, make_parents("random", 20 + i), seed=i) for i in range(6)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    try:
        for i, t in enumerate(trees):
            lib.gncx_hip_set_stream(streams[i % 2].cuda_stream)
            t.call(lib)
    finally:
        lib.gncx_hip_set_stream(None)
    torch.cuda.synchronize()
    for t in trees:
        want, tol = t.reference()
        assert bool(((t.out.double() - want).abs() <= tol).all())


def test_tree_rotations_on_two_streams(lib, torch_mod):
    """Calls at other positions, in turn on two streams with nothing between
    them: none rewrites the rotations that another still reads."""
    torch = torch_mod
    calls = []
    for i in range(6):
        calls.append(Tree(torch, 8, 2, 128, 40 + 500 * i, make_parents("random", 60 + i), base=1e4, weight=1, seed=i))
    want = []
    for t in calls:
        q, k, kc, vc = (x.clone() for x in (t.q, t.k, t.kc, t.vc))
        t.call(lib)
        want.append(t.out.clone())
        for x, old in ((t.q, q), (t.k, k), (t.kc, kc), (t.vc, vc)):
            x.copy_(old)
        t.out.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    try:
        for i, t in enumerate(calls):
            lib.gncx_hip_set_stream(streams[i % 2].cuda_stream)
            t.call(lib)
    finally:
        lib.gncx_hip_set_stream(None)
    torch.cuda.synchronize()
    for t, w in zip(calls, want):
        assert torch.equal(t.out, w)


def test_tree_refuses_host_overlap_alignment_and_capture(lib, torch_mod):
    torch = torch_mod
    lib.gncx_hip_last_status()

    def unchanged(t, text, **swap):
        before = {n: getattr(t, n).clone() for n in ("q", "k", "kc", "vc")}
        old = {n: getattr(t, n) for n in swap}
        for n, v in swap.items():
            setattr(t, n, v)
        t.call(lib, check=False)
        refused(lib, text)
        for n, v in old.items():
            setattr(t, n, v)
        for n, v in before.items():
            assert torch.equal(getattr(t, n), v)

    t = Tree(torch, 8, 2, 128, 16, make_parents("chain", 4))
    unchanged(t, "q_nodes must be memory", q=t.q.cpu())
    unchanged(t, "v_cache_layer must be memory", vc=t.vc.cpu())
    unchanged(t, "out_nodes must be memory", out=t.out.cpu())
    unchanged(t, "overlap", out=t.q)
    unchanged(t, "overlap", k=t.kc[17:21])
    unchanged(t, "overlap", v=t.k)
    unchanged(t, "aligned", q=torch.randn(4 * 1024 + 1, device="cuda")[1:].view(4, 1024))
    dev = torch.tensor(t.parents, dtype=torch.int32, device="cuda")
    lib.gncx_hip_attention_tree(t.q.data_ptr(), t.k.data_ptr(), t.v.data_ptr(), t.kc.data_ptr(), t.vc.data_ptr(), 16,
                                4, dev.data_ptr(), 8, 2, 128, t.scale, 0, None, 0, 0, -1, EPS, 0, 0, 0.0,
                                t.out.data_ptr())
    refused(lib, "parents must be host memory")
    t.call(lib)
    before = t.q.clone()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        lib.gncx_hip_set_stream(s.cuda_stream)
        try:
            with torch.cuda.graph(g, stream=s):
                t.call(lib, check=False)
        finally:
            lib.gncx_hip_set_stream(None)
    refused(lib, "capture")
    assert torch.equal(t.q, before)
    t.call(lib)


# ---- kept rows ----------------------------------------------------------------------
@pytest.mark.parametrize("layers,kv_dim,row0,rows", [
    (1, 4, 0, [0]), (1, 4, 3, [1]), (2, 8, 0, [0, 2, 3]), (3, 128, 5, [0, 1, 2]), (36, 1024, 100, [0, 3, 4, 9, 15]),
    (65, 64, 7, [2, 3, 11]), (130, 12, 1, [4]), (2, 2052, 0, [1, 2, 3, 4, 5, 6, 7, 8, 9, 10]), (2, 512, 50, "even"),
    (2, 256, 9, "shift"), (3, 1024, 0, "random"), (1, 1024, 2, "far")])
def test_keep_rows(lib, torch_mod, layers, kv_dim, row0, rows):
    torch = torch_mod
    rows = {"even": list(range(0, 1022, 2)), "shift": list(range(1, 513)), "far": [0, 1, 70, 65535],
            "random": sorted(np.random.default_rng(1).choice(700, 300, replace=False).tolist())}.get(rows, rows) \
        if isinstance(rows, str) else rows
    total = row0 + max(rows[-1] + 1, len(rows)) + 2
    k, v = torch.randn(layers, total, kv_dim, device="cuda"), torch.randn(layers, total, kv_dim, device="cuda")
    k[0, -1], v[-1, -1] = float("nan"), float("inf")
    want = []
    for c in (k, v):
        w = c.clone()
        w[:, row0:row0 + len(rows)] = c[:, [row0 + r for r in rows]]
        want.append(w)
    r = np.asarray(rows, np.int32)
    lib.gncx_hip_kv_keep_rows(addresses(k), addresses(v), layers, kv_dim, row0, r.ctypes.data, len(rows))
    gncx.check(lib)
    for got, w in zip((k, v), want):
        assert torch.equal(got.view(torch.int32), w.view(torch.int32))


def test_rows_past_4_gib(lib, torch_mod):
    """Row offsets and beam strides past 2^32 bytes."""
    torch = torch_mod
    kv_dim, row0 = 4096, 270000
    k, v = (torch.zeros(row0 + 8, kv_dim, device="cuda") for _ in range(2))
    for c in (k, v):
        c[row0:] = torch.randn(8, kv_dim, device="cuda")
    want = [c[row0:].clone() for c in (k, v)]
    for w in want:
        w[0], w[1] = w[2].clone(), w[5].clone()
    r = np.asarray([2, 5], np.int32)
    lib.gncx_hip_kv_keep_rows((C.c_void_p * 1)(k.data_ptr()), (C.c_void_p * 1)(v.data_ptr()), 1, kv_dim, row0,
                              r.ctypes.data, 2)
    gncx.check(lib)
    for c, w in zip((k, v), want):
        assert torch.equal(c[row0:], w) and not c[:row0].any()
    # two beams, the second 4.4 GB behind the first
    first, second = k[:4], k[row0 + 4:]
    first.copy_(v[row0:row0 + 4])
    want = first.clone()
    p = torch.tensor([0, 0], dtype=torch.int32, device="cuda")
    lib.gncx_hip_kv_reorder((C.c_void_p * 1)(k.data_ptr()), (C.c_void_p * 1)(v.data_ptr()), 1, 2,
                            (row0 + 4) * kv_dim, kv_dim, 0, 4, p.data_ptr())
    gncx.check(lib)
    assert torch.equal(first, want) and torch.equal(second, want)


def test_caches_that_share_memory_or_end_early_are_refused(lib, torch_mod):
    torch = torch_mod
    lib.gncx_hip_last_status()
    c = torch.randn(4, 8, 64, device="cuda")
    before, r = c.clone(), np.asarray([1], np.int32)
    p = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    one, two = (C.c_void_p * 1)(c.data_ptr()), (C.c_void_p * 1)(c.data_ptr() + 256)
    for other in (one, two):
        lib.gncx_hip_kv_keep_rows(one, other, 1, 64, 0, r.ctypes.data, 1)
        refused(lib, "share memory")
        lib.gncx_hip_kv_reorder(one, other, 1, 2, 512, 64, 0, 8, p.data_ptr())
        refused(lib, "share memory")
    # beams of two layers in turn share nothing: [beam][layer][row]
    a, b = (C.c_void_p * 1)(c[0].data_ptr()), (C.c_void_p * 1)(c[1].data_ptr())
    lib.gncx_hip_kv_reorder(a, b, 1, 2, 2 * 512, 64, 0, 8, p.data_ptr())
    gncx.check(lib)
    assert torch.equal(c, before[[2, 3, 0, 1]])
    # the second layer starts where a beam of the first ends early
    b = (C.c_void_p * 1)(c[2].data_ptr() - 256)
    lib.gncx_hip_kv_reorder(a, b, 1, 2, 2 * 512, 64, 0, 8, p.data_ptr())
    refused(lib, "share memory")
    far = np.asarray([60000], np.int32)
    lib.gncx_hip_kv_keep_rows(a, (C.c_void_p * 1)(c[2].data_ptr()), 1, 1 << 20, 0, far.ctypes.data, 1)
    refused(lib, "end")


# ---- beam selection --------------------------------------------------------------------
def select(lib, torch, logits, scores, n_out, finished=None, token=0):
    B, V = logits.shape
    par, tok = (torch.full((n_out,), -9, dtype=torch.int32, device="cuda") for _ in range(2))
    out = torch.full((n_out,), float("nan"), device="cuda")
    lib.gncx_hip_beam_select(logits.data_ptr(), B, V, scores.data_ptr(), None if finished is None else
                             finished.data_ptr(), token, n_out, par.data_ptr(), tok.data_ptr(), out.data_ptr())
    gncx.check(lib)
    return par.cpu().numpy(), tok.cpu().numpy(), out.cpu().numpy()


def select_reference(logits, scores, n_out, finished=None, token=0):
    """The definition in 64 bits: (parents, words, scores)."""
    x = logits.cpu().numpy().astype(np.float64)
    s = scores.cpu().numpy().astype(np.float64)
    x, s = np.where(np.isnan(x), -np.inf, x), np.where(np.isnan(s), -np.inf, s)
    B, V = x.shape
    total = np.full((B, V), -np.inf)
    for b in range(B):
        if finished is not None and finished[b]:
            total[b, token] = s[b]
            continue
        m = x[b].max()
        if m == -np.inf:
            continue
        with np.errstate(invalid="ignore"):
            d = np.where(x[b] == m, 0.0, x[b] - m)
            total[b] = s[b] + (d - np.log(np.exp(d).sum()))
    flat = total.reshape(-1)
    best = np.argsort(-flat, kind="stable")[:n_out]
    best = best[flat[best] > -np.inf]
    pad = n_out - len(best)
    return (np.concatenate([best // V, np.full(pad, -1)]), np.concatenate([best % V, np.full(pad, -1)]),
            np.concatenate([flat[best], np.full(pad, -np.inf)]))


def check_select(lib, torch, logits, scores, n_out, finished=None, token=0):
    got = select(lib, torch, logits, scores, n_out, finished, token)
    want = select_reference(logits, scores, n_out, None if finished is None else finished.cpu().numpy(), token)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    some = want[2] > -np.inf
    assert np.array_equal(got[2][~some], want[2][~some])
    # a score is rounded once (half a step); the sum of exponentials, each within
    # 1 ulp, takes at most 64 additions of fp32 on its way to 64 bits, so its
    # logarithm is within 66 u < 2^-17
    assert (np.abs(got[2][some] - want[2][some]) <= U * np.abs(want[2][some]) + 2.0 ** -17).all()


@pytest.mark.parametrize("B,V,n_out", [(1, 1, 1), (1, 1, 3), (1, 5, 5), (2, 3, 64), (3, 63, 6), (1, 64, 64),
                                       (4, 255, 8), (4, 257, 64), (2, 4095, 4), (2, 4097, 4), (5, 50257, 10),
                                       (4, 32000, 8), (32, 1000, 64), (16, 151936, 32), (32, 32001, 64), (1, 262144, 64),
                                       (7, 12289, 14), (1, 1 << 21, 2)])
def test_select(lib, torch_mod, B, V, n_out):
    torch = torch_mod
    g = torch.Generator(device="cuda").manual_seed(B * 7 + V)
    logits = 3 * torch.randn(B, V, generator=g, device="cuda")
    scores = -10 + torch.randn(B, generator=g, device="cuda")
    check_select(lib, torch, logits, scores, n_out)


@pytest.mark.parametrize("V", [100, 5000, 40000])
@pytest.mark.parametrize("kind", ["equal", "few", "rising", "falling", "zeros", "steps"])
def test_select_ties_and_orders(lib, torch_mod, V, kind):
    """Equal logits go to the lowest word, equal scores to the lowest beam; the
    best words may all lie in one place."""
    torch = torch_mod
    B, n_out = 4, 24
    at = torch.arange(B * V, device="cuda").view(B, V)
    logits = {"equal": torch.ones(B, V, device="cuda"), "few": (at * 7919 % 5).float(),
              "rising": (at % V).float() / V * 8, "falling": -(at % V).float() / V * 8,
              "zeros": torch.where(at % 3 == 0, -0.0, 0.0), "steps": (at % V // 1000).float() * 0.5}[kind]
    check_select(lib, torch, logits.contiguous(), torch.full((B,), -3.0, device="cuda"), n_out)


def test_select_first_step_masks_and_missing_candidates(lib, torch_mod):
    torch = torch_mod
    inf, nan = float("inf"), float("nan")
    g = torch.Generator(device="cuda").manual_seed(3)
    logits = torch.randn(6, 9000, generator=g, device="cuda")
    scores = torch.tensor([0.0, -inf, -inf, -inf, -inf, nan], device="cuda")
    check_select(lib, torch, logits, scores, 12)  # one live beam
    logits[:] = -inf
    check_select(lib, torch, logits, scores, 12)  # nothing at all
    logits[0, [5, 4097, 8999]] = torch.tensor([1.0, 2.0, 1.0], device="cuda")
    logits[2, 7] = 3.0
    check_select(lib, torch, logits, scores, 12)  # three candidates
    scores[2] = -0.25
    check_select(lib, torch, logits, scores, 12)
    logits[0, 100:200] = nan
    check_select(lib, torch, logits, scores, 5)
    logits[0, [3, 8000]] = inf                     # an infinite logit takes all, two share it
    check_select(lib, torch, logits, scores, 5)
    logits[:] = nan
    check_select(lib, torch, logits, scores, 5)
    check_select(lib, torch, torch.full((2, 300), -3e38, device="cuda"), scores[[0, 2]].contiguous(), 5)
    check_select(lib, torch, torch.full((2, 300), 3e38, device="cuda"), scores[[0, 2]].contiguous(), 5)


def test_select_finished_beams(lib, torch_mod):
    torch = torch_mod
    g = torch.Generator(device="cuda").manual_seed(4)
    logits = torch.randn(5, 7001, generator=g, device="cuda")
    logits[1] = float("nan")  # never read
    scores = torch.tensor([-9.0, -2.0, -9.0, -8.5, -30.0], device="cuda")
    done = torch.tensor([0, 1, 0, 7, 1], dtype=torch.int32, device="cuda")
    for n_out in (1, 2, 10, 64):
        check_select(lib, torch, logits, scores, n_out, done, 2)
    check_select(lib, torch, logits, scores, 64, torch.ones_like(done), 7000)


def test_select_unaligned_rows_and_outputs_over_inputs(lib, torch_mod):
    torch = torch_mod
    B, V = 3, 4099
    flat = torch.randn(B * V + 1, device="cuda")
    logits = flat[1:].view(B, V)
    scores = torch.tensor([-1.0, -1.5, -2.0], device="cuda")
    done = torch.tensor([0, 0, 1], dtype=torch.int32, device="cuda")
    want = select_reference(logits, scores, 3, done.cpu().numpy(), 4)
    tok = torch.zeros(3, dtype=torch.int32, device="cuda")
    lib.gncx_hip_beam_select(logits.data_ptr(), B, V, scores.data_ptr(), done.data_ptr(), 4, 3, done.data_ptr(),
                             tok.data_ptr(), scores.data_ptr())
    gncx.check(lib)
    assert np.array_equal(done.cpu().numpy(), want[0]) and np.array_equal(tok.cpu().numpy(), want[1])
    assert np.allclose(scores.cpu().numpy(), want[2], rtol=1e-6)


@pytest.mark.parametrize("V", [16384, 151936])
@pytest.mark.parametrize("gap", [12.0, 14.0, 15.5])
def test_select_sums_of_many_small_exponentials(lib, torch_mod, V, gap):
    """One large logit among equal small ones, whose exponentials are lost one by
    one in a 32-bit sum that holds the large one's.  The exponentials are formed
    in 32 bits (1 ulp of expf and the difference's half step, gap u, each of
    itself), so the sum is off by at most (2 + gap) u of the small ones' part of
    it, and the score by that and its own rounding."""
    torch = torch_mod
    logits = torch.full((1, V), -gap, device="cuda")
    logits[0, V // 3] = 0.0
    _, tok, got = select(lib, torch, logits, torch.zeros(1, device="cuda"), 1)
    small = (V - 1) * math.exp(-gap)
    want = -math.log1p(small)
    assert tok[0] == V // 3
    assert abs(float(got[0]) - want) <= (2 + gap) * U * small / (1 + small) + U * abs(want) + 2.0 ** -50


@pytest.mark.parametrize("V", [7, 200, 5000, 151936])
@pytest.mark.parametrize("score", [1e20, -1e20, float("inf"), 0.0])
def test_select_scores_that_64_bits_do_not_part(lib, torch_mod, V, score):
    """Words of a beam whose scores are equal in 64 bits although their logits are
    not (a beam's score that swallows them, logits next to 0): the larger logit
    first, equal ones by the lower word; beams with equal scores by the lower beam."""
    torch = torch_mod
    n_out = 20
    g = torch.Generator(device="cuda").manual_seed(V)
    logits = torch.randint(-40, 40, (3, V), generator=g, device="cuda").float() / 4
    if score == 0.0:
        logits *= 1e-30
    scores = torch.tensor([-1e30, score, score], device="cuda")  # (the first beam comes last)
    order = np.argsort(-logits.cpu().numpy(), axis=1, kind="stable")
    par, tok, _ = select(lib, torch, logits, scores, n_out)
    assert par.tolist() == np.repeat([1, 2, 0], V)[:n_out].tolist()
    assert np.array_equal(tok, order[[1, 2, 0]].reshape(-1)[:n_out])


def test_select_scores_below_the_least_float(lib, torch_mod):
    """A score that 32 bits hold as -inf is no candidate."""
    torch = torch_mod
    logits = torch.tensor([[0.0, -3e38, -1e38, 0.0], [-3e38, 5.0, 1.0, -3e38]], device="cuda")
    scores = torch.tensor([-3e38, -1.0], device="cuda")
    par, tok, out = select(lib, torch, logits, scores, 10)
    # (beam 1's words 0 and 3 are at -3e38 - 6, equal in 64 bits to beam 0's -3e38 -
    # log 2, and come behind them; beam 0's word 2 is at -4e38)
    assert par.tolist() == [1, 1, 0, 0, 1, 1] + [-1] * 4
    assert tok.tolist() == [1, 2, 0, 3, 0, 3] + [-1] * 4
    assert np.isfinite(out[:6]).all() and (out[6:] == -np.inf).all()
    par, tok, out = select(lib, torch, logits[:1].contiguous(), scores, 3)
    assert par.tolist() == [0, 0, -1] and tok.tolist() == [0, 3, -1] and out[2] == -np.inf


# ---- reordering ------------------------------------------------------------------------
@pytest.mark.parametrize("layers,beams,kv_dim,row0,rows,parents", [
    (1, 1, 4, 0, 1, [0]), (1, 1, 4, 0, 1, [-1]), (2, 2, 8, 1, 3, [1, 0]), (3, 4, 128, 5, 17, [0, 0, 0, 0]),
    (2, 4, 64, 0, 9, [1, 2, 3, 0]), (2, 4, 64, 2, 9, [0, 1, 2, 3]), (65, 3, 12, 1, 5, [2, 2, 1]),
    (2, 5, 1024, 7, 33, [4, -1, 9, 0, 4]), (1, 32, 256, 3, 50, "swap"), (2, 17, 132, 0, 11, "random"),
    (1, 31, 64, 9, 1000, "random"), (36, 8, 1024, 40, 25, "random"), (2, 6, 8, 3, 2, [2 ** 31 - 1, -2 ** 31, 0, 5, 6, 1])])
def test_reorder(lib, torch_mod, layers, beams, kv_dim, row0, rows, parents):
    torch = torch_mod
    rng = np.random.default_rng(beams)
    parents = {"swap": list(range(beams))[::-1], "random": rng.integers(0, beams, beams).tolist()}.get(parents) \
        if isinstance(parents, str) else parents
    total = row0 + rows + 2
    k, v = (torch.randn(layers, beams, total, kv_dim, device="cuda") for _ in range(2))
    k[0, 0, row0] = float("nan")
    source = [p if 0 <= p < beams else b for b, p in enumerate(parents)]
    want = []
    for c in (k, v):
        w = c.clone()
        w[:, :, row0:row0 + rows] = c[:, source, row0:row0 + rows]
        want.append(w)
    dev = torch.tensor(parents, dtype=torch.int32, device="cuda")
    lib.gncx_hip_kv_reorder(addresses(k), addresses(v), layers, beams, total * kv_dim, kv_dim, row0, rows,
                            dev.data_ptr())
    gncx.check(lib)
    for got, w in zip((k, v), want):
        assert torch.equal(got.view(torch.int32), w.view(torch.int32))


def test_reorder_refuses_parents_within_the_caches(lib, torch_mod):
    """The parents are read while the beams' rows are written."""
    torch = torch_mod
    c = torch.zeros(2, 3, 8, 64, device="cuda")  # (zeros: parents 0, wherever they are read)
    ks, vs = addresses(c[:1]), addresses(c[1:])
    lib.gncx_hip_last_status()
    for at in (c[0, 0, 2], c[0, 2, 7, 60:], c[1, 1, 5]):
        lib.gncx_hip_kv_reorder(ks, vs, 1, 3, 512, 64, 2, 6, at.data_ptr())
        refused(lib, "parents lie")
    before = c[:, 1].normal_().clone()
    lib.gncx_hip_kv_reorder(ks, vs, 1, 3, 512, 64, 2, 6, c[0, 2, 1].data_ptr())  # (a row before row0)
    gncx.check(lib)
    assert not c[:, 1, 2:].any() and torch.equal(c[:, 1, :2], before[:, :2])


def test_refusals_on_the_device(lib, torch_mod):
    torch = torch_mod
    lib.gncx_hip_last_status()
    c = torch.zeros(2, 64, device="cuda")
    good, host = addresses(c.view(1, 2, 64)), (C.c_void_p * 1)(torch.zeros(2, 64).data_ptr())
    odd = (C.c_void_p * 1)(c.data_ptr() + 4)
    r, p = np.zeros(1, np.int32), torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad, text in ((host, "must be memory of"), (odd, "16-byte aligned"), ((C.c_void_p * 1)(), "must be memory of")):
        lib.gncx_hip_kv_keep_rows(good, bad, 1, 64, 0, r.ctypes.data, 1)
        refused(lib, text)
        lib.gncx_hip_kv_reorder(bad, good, 1, 2, 64, 64, 0, 1, p.data_ptr())
        refused(lib, text)
    lib.gncx_hip_kv_keep_rows(good, good, 1, 64, 0, p.data_ptr(), 1)
    refused(lib, "rows must be host memory")
    lib.gncx_hip_kv_reorder(good, good, 1, 2, 64, 64, 0, 1, r.ctypes.data)
    refused(lib, "parents must be memory of")
    lib.gncx_hip_kv_reorder(None, good, 1, 2, 64, 64, 0, 1, p.data_ptr())
    refused(lib, "at least one layer")
    x = torch.zeros(2, 10)
    lib.gncx_hip_beam_select(x.data_ptr(), 2, 10, c.data_ptr(), None, 0, 1, p.data_ptr(), p.data_ptr(), c.data_ptr())
    refused(lib, "logits must be memory of")
    assert not c.any() and not p.any()


def past_the_end(torch, t):
    """Bytes from t's first to the end of the allocation that it lies in."""
    at = t.data_ptr()
    for s in torch.cuda.memory_snapshot():
        if s["address"] <= at < s["address"] + s["total_size"]:
            return s["address"] + s["total_size"] - at
    raise AssertionError("not the allocator's memory")


@pytest.mark.parametrize("short", ["q", "k", "v", "kc", "vc", "out"])
def test_tree_vectors_and_caches_that_end_early_are_refused(lib, torch_mod, short):
    """Nothing is launched where a vector, cache or output would be read or
    written past the end of its memory."""
    torch = torch_mod
    t = Tree(torch, 8, 2, 128, 16, make_parents("chain", 4))
    before = {n: getattr(t, n).clone() for n in ("q", "k", "kc", "vc")}
    lib.gncx_hip_last_status()
    old, old_pos = getattr(t, short), t.pos0
    if short in ("kc", "vc"):
        t.pos0 = past_the_end(torch, old) // (4 * 256) - 3  # 3 of 4 rows fit
    else:
        # the last 16 bytes of its memory
        end = past_the_end(torch, old)

        class Last:
            data_ptr = staticmethod(lambda: old.data_ptr() + end - 16)
        setattr(t, short, Last)
    t.call(lib, check=False)
    refused(lib, "end")
    setattr(t, short, old)
    t.pos0 = old_pos
    for n, v in before.items():
        assert torch.equal(getattr(t, n), v)
    t.call(lib)


def test_select_and_reorder_refuse_what_ends_early(lib, torch_mod):
    torch = torch_mod
    B, V, n = 3, 100, 4
    flat = torch.zeros(4096, device="cuda")
    lib.gncx_hip_last_status()
    last = flat.data_ptr() + past_the_end(torch, flat) - 4  # a float, where more are needed
    x, sc, fin = torch.randn(B, V, device="cuda"), torch.zeros(B, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    out = torch.zeros(3, n, dtype=torch.int32, device="cuda")
    good = [x.data_ptr(), sc.data_ptr(), fin.data_ptr(), out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr()]
    for i in range(6):
        a = list(good)
        a[i] = last
        lib.gncx_hip_beam_select(a[0], B, V, a[1], a[2], 0, n, *a[3:])
        refused(lib, "end")
    assert not out.any()
    lib.gncx_hip_beam_select(good[0], B, V, good[1], good[2], 0, n, *good[3:])
    gncx.check(lib)
    c = torch.randn(2, B, 8, 64, device="cuda")
    before = c.clone()
    lib.gncx_hip_kv_reorder(addresses(c[:1]), addresses(c[1:]), 1, B, 512, 64, 0, 8, last)
    refused(lib, "end")
    assert torch.equal(c, before)


# ---- graphs ------------------------------------------------------------------------------
def test_selection_and_reordering_captured(lib, torch_mod):
    """A beam step's selection and reordering in a graph, replayed between eager
    work, next to a second graph and an eager call that needs more workspace."""
    torch = torch_mod
    B, V, n, layers, kv_dim, rows = 4, 20000, 4, 2, 64, 12
    logits, scores = torch.empty(B, V, device="cuda"), torch.empty(B, device="cuda")
    par, tok = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))
    best = torch.zeros(n, device="cuda")
    k, v = (torch.randn(layers, B, rows, kv_dim, device="cuda") for _ in range(2))
    ka, va = addresses(k), addresses(v)

    def step():
        lib.gncx_hip_beam_select(logits.data_ptr(), B, V, scores.data_ptr(), None, 0, n, par.data_ptr(),
                                 tok.data_ptr(), best.data_ptr())
        lib.gncx_hip_kv_reorder(ka, va, layers, B, rows * kv_dim, kv_dim, 2, rows - 2, par.data_ptr())

    logits.normal_()
    scores.fill_(-1.0)
    step()
    gncx.check(lib)
    graphs = []
    s = torch.cuda.Stream()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        lib.gncx_hip_set_stream(s.cuda_stream)
        try:
            with torch.cuda.graph(g, stream=s):
                step()
        finally:
            lib.gncx_hip_set_stream(None)
        gncx.check(lib)
        graphs.append(g)
    for i in range(6):
        logits.normal_()
        scores.normal_()
        before = [c.clone() for c in (k, v)]
        torch.cuda.synchronize()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        want = select_reference(logits, scores, n)
        assert np.array_equal(par.cpu().numpy(), want[0]) and np.array_equal(tok.cpu().numpy(), want[1])
        for c, old in zip((k, v), before):
            old[:, :, 2:] = old[:, par.long(), 2:]
            assert torch.equal(c, old)
        # a call that needs a larger workspace leaves the graphs theirs
        check_select(lib, torch, torch.randn(4 * (i + 1), 151936, device="cuda"),
                     torch.randn(4 * (i + 1), device="cuda"), 64)


def test_kept_rows_captured(lib, torch_mod):
    torch = torch_mod
    layers, kv_dim, row0, rows = 66, 72, 3, [0, 2, 3, 9]
    k, v = (torch.empty(layers, 16, kv_dim, device="cuda") for _ in range(2))
    ka, va, r = addresses(k), addresses(v), np.asarray(rows, np.int32)
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    lib.gncx_hip_set_stream(s.cuda_stream)
    try:
        with torch.cuda.graph(g, stream=s):
            lib.gncx_hip_kv_keep_rows(ka, va, layers, kv_dim, row0, r.ctypes.data, len(rows))
    finally:
        lib.gncx_hip_set_stream(None)
    gncx.check(lib)
    r[:] = 0  # read before the call returned
    for _ in range(4):
        k.normal_()
        v.normal_()
        want = [c.clone() for c in (k, v)]
        for w, c in zip(want, (k, v)):
            w[:, row0:row0 + len(rows)] = c[:, [row0 + i for i in rows]]
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_select_outputs_that_overlap_are_refused(lib, torch_mod):
    torch = torch_mod
    x, sc = torch.randn(2, 50, device="cuda"), torch.zeros(2, device="cuda")
    out = torch.zeros(12, dtype=torch.int32, device="cuda")
    at = [out.data_ptr() + 16 * i for i in range(3)]
    lib.gncx_hip_last_status()
    for a, b, c in ((0, 0, 1), (0, 1, 0), (0, 1, 1)):
        lib.gncx_hip_beam_select(x.data_ptr(), 2, 50, sc.data_ptr(), None, 0, 4, at[a], at[b], at[c])
        refused(lib, "outputs overlap")
    lib.gncx_hip_beam_select(x.data_ptr(), 2, 50, sc.data_ptr(), None, 0, 5, *at)
    refused(lib, "outputs overlap")
    assert not out.any()
    lib.gncx_hip_beam_select(x.data_ptr(), 2, 50, sc.data_ptr(), None, 0, 4, *at)
    gncx.check(lib)


def test_select_graphs_run_beside_one_another(lib, torch_mod):
    """Two graphs captured with no call before them, replayed on two streams at
    once and beside eager calls on a third: each has a workspace of its own."""
    torch = torch_mod
    B, V, n = 6, 151936, 64
    streams = [torch.cuda.Stream() for _ in range(2)]
    sets = []
    for s in streams:
        t = dict(x=torch.randn(B, V, device="cuda"), sc=torch.randn(B, device="cuda"),
                 par=torch.zeros(n, dtype=torch.int32, device="cuda"),
                 tok=torch.zeros(n, dtype=torch.int32, device="cuda"), best=torch.zeros(n, device="cuda"))
        g = torch.cuda.CUDAGraph()
        lib.gncx_hip_set_stream(s.cuda_stream)
        try:
            with torch.cuda.graph(g, stream=s):
                for _ in range(3):
                    lib.gncx_hip_beam_select(t["x"].data_ptr(), B, V, t["sc"].data_ptr(), None, 0, n,
                                             t["par"].data_ptr(), t["tok"].data_ptr(), t["best"].data_ptr())
        finally:
            lib.gncx_hip_set_stream(None)
        gncx.check(lib)
        sets.append((g, s, t))
    x, sc = torch.randn(B, V, device="cuda"), torch.randn(B, device="cuda")
    alone = select_reference(x, sc, n)
    for _ in range(4):
        for _, _, t in sets:
            t["x"].normal_()
            t["par"].fill_(-5)
            t["tok"].fill_(-5)
        torch.cuda.synchronize()
        for g, s, _ in sets:
            with torch.cuda.stream(s):
                for _ in range(5):
                    g.replay()
        par, tok, _ = select(lib, torch, x, sc, n)
        torch.cuda.synchronize()
        assert np.array_equal(par, alone[0]) and np.array_equal(tok, alone[1])
        for _, _, t in sets:
            want = select_reference(t["x"], t["sc"], n)
            assert np.array_equal(t["par"].cpu().numpy(), want[0])
            assert np.array_equal(t["tok"].cpu().numpy(), want[1])


# ---- a run of them together: the decode driver --------------------------------------------
LOGITS = 1e-3  # the bar of this driver's logits between its batched and its one-token calls (relative L2)


def small_decoder(lib, torch, hd, max_seq=96, seed=7, **kw):
    import gncx_amd.decode as dec
    shape = dec.Qwen3Shape(n_layers=2, embed=256, n_heads=4, n_kv=2, head_dim=hd, ffn=512, vocab=600)
    model = dec.build_model(torch, shape, seed=seed)
    return dec, model, dec.Decoder(lib, torch, model, max_seq=max_seq, fused=True, **kw)


def distance(got, want):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    return np.linalg.norm(got - want) / np.linalg.norm(want)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_a_tree_is_its_branches_decoded_one_by_one(lib, torch_mod, hd):
    """Every node's logits, and after keep_path the next step's, against another
    decoder that steps along the node's branch alone."""
    torch = torch_mod
    dec, model, d = small_decoder(lib, torch, hd)
    prompt = [11, 22, 33, 44, 55, 66, 77]
    tokens, parents = [5, 6, 7, 8, 5, 9, 10, 599, 0], [-1, 0, 0, 1, 2, 4, 5, 3, -1]
    d.prefill(prompt)
    got = d.verify_tree(tokens, parents, len(prompt)).cpu().numpy()
    ref = dec.Decoder(lib, torch, model, max_seq=96, fused=True)
    for i in range(len(tokens)):
        branch, j = [], i
        while j >= 0:
            branch.insert(0, j)
            j = parents[j]
        ref.prefill(prompt)
        for at, j in enumerate(branch):
            want = ref.forward_token(tokens[j], len(prompt) + at).cpu().numpy()
        assert distance(got[i], want) < LOGITS, i
    path = [0, 2, 4, 5, 6]
    d.keep_path(len(prompt), path)
    ref.prefill(prompt)
    for at, j in enumerate(path):
        ref.forward_token(tokens[j], len(prompt) + at)
    pos = len(prompt) + len(path)
    assert distance(d.forward_token(17, pos).cpu(), ref.forward_token(17, pos).cpu()) < LOGITS
    for a, b in zip(d.kc + d.vc, ref.kc + ref.vc):
        assert distance(a[:pos].cpu(), b[:pos].cpu()) < LOGITS
    gncx.check(lib)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", ["none", "lookup", "right", "wide"])
def test_drafted_generation_is_greedy(lib, torch_mod, hd, kind):
    """Whatever the drafts, every new id is the largest logit (to the bar's
    width) of a decoder that steps along the ids one by one; right drafts are
    accepted, so they take few passes."""
    torch = torch_mod
    dec, model, d = small_decoder(lib, torch, hd)
    prompt, n_new = [3, 599, 17, 3, 599, 250, 3, 599], 24
    plain = d.generate(prompt, n_new)
    rng = np.random.default_rng(1)
    passes = []

    def draft(ids):
        at = len(ids) - len(prompt)
        passes.append(at)
        if kind == "none":
            return [], []
        rest = plain[at:at + 6]
        if kind == "right":
            return rest, list(range(-1, len(rest) - 1))
        tokens, parents = [], []  # wrong branches before, beside and below the right one
        last = -1
        for t in rest:
            for _ in range(20):
                tokens.append(int(rng.integers(600)))
                parents.append(int(rng.integers(-1, len(tokens) - 1)))
            tokens.append(t)
            parents.append(last)
            last = len(tokens) - 1
        return tokens[:60], parents[:60]

    new = d.generate_drafted(prompt, n_new, None if kind == "lookup" else draft)
    assert len(new) == n_new
    ref = dec.Decoder(lib, torch, model, max_seq=96, fused=True)
    logits, same = ref.prefill(prompt), 0
    for i, t in enumerate(new):
        x = logits.cpu().numpy().astype(np.float64)
        assert x[t] >= x.max() - 2 * LOGITS * np.linalg.norm(x), i
        logits = ref.forward_token(t, len(prompt) + i)
    while same < n_new and new[same] == plain[same]:
        same += 1
    if kind == "right" and same == n_new:
        assert passes == [1, 8, 15, 22]  # six accepted and one chosen a pass
    if kind == "none":
        assert passes == list(range(1, n_new))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("beams,end", [(1, -1), (4, -1), (5, 123), (32, -1)])
def test_beam_search(lib, torch_mod, hd, beams, end):
    """Scores against the ids' log probabilities by a decoder that steps along
    them one by one, and the ids against a beam search over that decoder
    wherever its decisions are wider than the bar."""
    torch = torch_mod
    dec, model, d = small_decoder(lib, torch, hd)
    prompt, n_new = [11, 22, 33, 44, 55], 5
    got = d.beam_search(prompt, beams, n_new, end)
    ref = dec.Decoder(lib, torch, model, max_seq=96, fused=True)
    memo = {}

    def log_probs(ids):  # and how far the bar lets each of them be off
        if ids not in memo:
            logits = ref.prefill(prompt)
            for i, t in enumerate(ids):
                logits = ref.forward_token(t, len(prompt) + i)
            x = logits.cpu().numpy().astype(np.float64)
            memo[ids] = (x - x.max() - np.log(np.exp(x - x.max()).sum()), 2 * LOGITS * np.linalg.norm(x))
        return memo[ids]

    def steps(ids):  # the tokens that count: up to the first end
        ids = tuple(ids)
        return ids[:ids.index(end) + 1] if end in ids else ids

    assert 1 <= len(got) <= beams
    assert [c for _, c in got] == sorted((c for _, c in got), reverse=True)
    for ids, score in got:
        want = bar = 0.0
        for i, t in enumerate(steps(ids)):
            lp, off = log_probs(tuple(ids[:i]))
            want, bar = want + lp[t], bar + off
        assert abs(score - want) <= bar + 1e-4
        assert all(t == end for t in ids[len(steps(ids)):])
    hyps, clear = [((), 0.0, 0.0)], True
    for _ in range(n_new):
        cand = []
        for ids, c, bar in hyps:
            if end in ids:
                cand.append((ids + (end,), c, bar))
                continue
            lp, off = log_probs(ids)
            cand += [(ids + (t,), c + lp[t], bar + off) for t in range(600)]
        cand.sort(key=lambda h: -h[1])
        for a, b in zip(cand[:beams], cand[1:beams + 1]):
            clear &= a[1] - b[1] > a[2] + b[2]
        hyps = cand[:beams]
    if clear:
        assert [tuple(i) for i, _ in got] == [h[0] for h in hyps]
    assert got[0][1] >= hyps[0][1] - 2 * hyps[0][2] - 1e-4 or not clear
    gncx.check(lib)


def test_driver_refusals(lib, torch_mod):
    _, _, d = small_decoder(lib, torch_mod, 64, max_seq=16)
    d.prefill([1, 2, 3])
    for tokens, parents, pos in (([], [], 3), ([1], [-1, 0], 3), ([1, 2], [-1, 0], 15), ([1], [-1], -1)):
        with pytest.raises(ValueError):
            d.verify_tree(tokens, parents, pos)
    with pytest.raises(RuntimeError, match="earlier node"):
        d.verify_tree([1, 2], [1, -1], 3)
    with pytest.raises(RuntimeError, match="ascend"):
        d.keep_path(3, [1, 0])
    for beams, n in ((0, 4), (33, 4), (2, 0), (2, 15)):
        with pytest.raises(ValueError):
            d.beam_search([1, 2, 3], beams, n)
    _, _, h = small_decoder(lib, torch_mod, 64, max_seq=16, device="cpu")
    with pytest.raises(ValueError):
        h.verify_tree([1], [-1], 0)
    with pytest.raises(ValueError):
        h.beam_search([1, 2, 3], 2, 2)
