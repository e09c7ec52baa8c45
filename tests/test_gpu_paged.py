"""GPU: many sequences at once through the C-ABI with device pointers, against
64-bit formulas: rotary positions of rows, appending to the paged cache of 8-bit
blocks, attention over it, and log probabilities."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest

from conftest import gncx

pytestmark = pytest.mark.gpu
U = 2.0 ** -24  # half a step of fp32
EPS = 1e-6
BLOCK = 16


def refused(lib, text):
    assert lib.gncx_hip_last_status() != 0
    assert text in lib.gncx_hip_last_error().decode()


def randn(torch, seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def whole(torch, values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- rotary positions ---------------------------------------------------------------
class Turn:
    """A rotation, and what it does in 64 bits."""

    def __init__(self, torch, n_rot, inter=0, magnitude=1.0, base=1e4):
        self.torch, self.n, self.inter, self.magnitude = torch, n_rot, inter, magnitude
        self.freqs = torch.from_numpy(base ** (-2.0 * np.arange(max(n_rot // 2, 1)) / max(n_rot, 1))).cuda()
        self.c = gncx.Rotation(self.freqs.data_ptr(), n_rot, inter, magnitude)
        self.magnitude = self.c.magnitude  # as a float

    def ref(self):
        return C.addressof(self.c)

    def __call__(self, x, at):
        """x [rows][heads][head_dim] (64 bits): the result, and how far 32 bits may be off
        from it.  A turn is off by half a step below 1/2, 2^-26 or 2 pi 2^-26 radians; the
        cosine and sine by four steps, the products and their sum by three roundings:
        under 2^-23.4 + 8 u + 3 u < 13 u of |a| + |b|."""
        torch, n = self.torch, self.n
        if n == 0:
            return x.clone(), torch.zeros_like(x)
        angle = at.double()[:, None, None] * self.freqs
        a, b = (x[..., 0:n:2], x[..., 1:n:2]) if self.inter else (x[..., :n // 2], x[..., n // 2:n])
        y, tol = x.clone(), torch.zeros_like(x)
        p = self.magnitude * (a * angle.cos() - b * angle.sin())
        q = self.magnitude * (b * angle.cos() + a * angle.sin())
        t = 13 * U * abs(self.magnitude) * (a.abs() + b.abs())
        if self.inter:
            y[..., 0:n:2], y[..., 1:n:2], tol[..., 0:n:2], tol[..., 1:n:2] = p, q, t, t
        else:
            y[..., :n // 2], y[..., n // 2:n], tol[..., :n // 2], tol[..., n // 2:n] = p, q, t, t
        return y, tol


@pytest.mark.parametrize("rows,heads,hd,n_rot,inter,mag,pad,shift", [
    (1, 40, 128, 128, 0, 1.0, 0, 0), (3, 5, 64, 64, 1, 1.0, 0, 0), (7, 3, 128, 32, 0, 1.25, 8, 4),
    (7, 3, 128, 32, 1, 1.25, 8, 4), (5, 2, 80, 80, 0, 1.0, 0, 0), (5, 2, 80, 20, 1, 0.5, 0, 0),
    (4, 3, 96, 70, 0, 1.0, 0, 0), (4, 3, 6, 2, 1, 1.0, 1, 0), (2, 70, 256, 256, 0, 1.0, 0, 0),
    (2, 1, 1024, 1024, 1, 1.0, 0, 0), (2, 3, 1024, 8, 0, 1.0, 0, 0), (300, 9, 128, 128, 0, 1.0, 3, 1),
    (6, 4, 64, 0, 0, 3.0, 0, 0), (6, 2, 2, 2, 0, 1.0, 0, 0), (1100, 2, 64, 48, 1, 1.0, 0, 0)])
def test_rope_rows(lib, torch_mod, rows, heads, hd, n_rot, inter, mag, pad, shift):
    torch = torch_mod
    width, t = heads * hd, Turn(torch, n_rot, inter, mag)
    held = randn(torch, rows, rows * (width + pad) + shift)
    x = held[shift:].view(rows, width + pad)
    at = torch.randint(-5000, 1000000, (rows,), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda",
                       dtype=torch.int32)
    at[0] = 0
    want, tol = t(x[:, :width].double().view(rows, heads, hd), at)
    out = torch.full((rows, width + pad + 4), 7.0, device="cuda")
    before = held.clone()
    lib.gncx_hip_rope_rows(x.data_ptr(), rows, width + pad, heads, hd, at.data_ptr(), t.ref(), width + pad + 4,
                           out.data_ptr())
    gncx.check(lib)
    assert torch.equal(held, before) and (out[:, width:] == 7.0).all()
    got = out[:, :width].reshape(rows, heads, hd)
    assert ((got.double() - want).abs() <= tol).all()
    assert torch.equal(got[..., n_rot:], x[:, :width].view(rows, heads, hd)[..., n_rot:])
    # in place: the same, and what lies between the rows stays
    lib.gncx_hip_rope_rows(x.data_ptr(), rows, width + pad, heads, hd, at.data_ptr(), t.ref(), width + pad, x.data_ptr())
    gncx.check(lib)
    assert torch.equal(x[:, :width].reshape(rows, heads, hd), got)
    assert torch.equal(x[:, width:], before[shift:].view(rows, width + pad)[:, width:])


def test_rope_turns_back_and_differentiates(lib, torch_mod):
    """Negative positions are the rotation's transpose, <R x, y> = <x, R' y>: its gradient."""
    torch, t = torch_mod, Turn(torch_mod, 64, 0, 1.2)
    x, y = randn(torch, 1, 9, 4 * 64), randn(torch, 2, 9, 4 * 64)
    at = whole(torch, [0, 1, 2, 77, 500, 4095, 4096, 100000, 7])
    back, rx, ry = -at, torch.empty_like(x), torch.empty_like(y)
    lib.gncx_hip_rope_rows(x.data_ptr(), 9, 256, 4, 64, at.data_ptr(), t.ref(), 256, rx.data_ptr())
    lib.gncx_hip_rope_rows(y.data_ptr(), 9, 256, 4, 64, back.data_ptr(), t.ref(), 256, ry.data_ptr())
    gncx.check(lib)
    _, tx = t(x.double().view(9, 4, 64), at)
    _, ty = t(y.double().view(9, 4, 64), back)
    off = (tx.view(9, -1) * y.double().abs() + ty.view(9, -1) * x.double().abs()).sum(1)
    assert (((rx.double() * y.double()).sum(1) - (x.double() * ry.double()).sum(1)).abs() <= off).all()


def test_rope_frequencies_on_the_device(lib, torch_mod):
    torch = torch_mod
    fac = np.linspace(1, 4, 32, dtype=np.float32)
    d_fac, mag = torch.from_numpy(fac).cuda(), C.c_float()
    out, host = torch.zeros(32, dtype=torch.float64, device="cuda"), np.zeros(32)
    for f, o in ((d_fac.data_ptr(), out.data_ptr()), (fac.ctypes.data, host.ctypes.data)):
        assert lib.gncx_hip_rope_frequencies(64, 1e4, gncx.ROPE_YARN, 4.0, 4096, 32.0, 1.0, f, o, C.addressof(mag)) == 0
    assert (out.cpu().numpy() == host).all() and host[0] == 1.0
    # memory that ends before the last of them, or lies between two
    end = torch.zeros(2 ** 22, dtype=torch.float64, device="cuda")  # (an allocation of its own)
    for f, o, text in ((None, end.data_ptr() + 8 * (2 ** 22 - 31), "past the end"), (None, out.data_ptr() + 4, "8-byte"),
                       (end.data_ptr() + 8 * 2 ** 22 - 4 * 31, host.ctypes.data, "past the end")):
        lib.gncx_hip_last_status()
        assert lib.gncx_hip_rope_frequencies(64, 1e4, gncx.ROPE_PLAIN, 1.0, 0, 0.0, 0.0, f, o, None) == -1
        refused(lib, text)
    assert (end == 0).all() and (out.cpu().numpy() == host).all()


def test_rope_refusals(lib, torch_mod):
    torch, t = torch_mod, Turn(torch_mod, 64)
    x, at = randn(torch, 1, 4, 128), whole(torch, [1, 2, 3, 4])
    before = x.clone()

    def call(rows=x.data_ptr(), n=4, stride=128, heads=2, hd=64, pos=at.data_ptr(), rot=t.ref(), ostride=128,
             out=x.data_ptr()):
        lib.gncx_hip_last_status()
        lib.gncx_hip_rope_rows(rows, n, stride, heads, hd, pos, rot, ostride, out)

    host = np.zeros(1000, np.float32)  # (kept: its address is passed)
    for kw, text in ((dict(rows=host.ctypes.data), "memory of the library's GPU"), (dict(out=host.ctypes.data), "GPU"),
                     (dict(pos=host.ctypes.data), "GPU"), (dict(rows=x.data_ptr() + 2), "4-byte aligned"),
                     (dict(n=2 ** 24), "past the end"), (dict(out=x.data_ptr() + 512), "overlaps"),
                     (dict(ostride=129), "overlap"), (dict(pos=x.data_ptr()), "overlaps"),
                     (dict(heads=4, hd=32), "multiple of 2 up to head_dim"),
                     (dict(rot=C.byref(gncx.Rotation(t.freqs.data_ptr(), 63, 0, 1.0))), "multiple of 2"),
                     (dict(rot=C.byref(gncx.Rotation(t.freqs.data_ptr(), -2, 0, 1.0))), "multiple of 2"),
                     (dict(rot=C.byref(gncx.Rotation(host.ctypes.data, 64, 0, 1.0))), "GPU"),
                     (dict(rot=C.byref(gncx.Rotation(t.freqs.data_ptr() + 4, 64, 0, 1.0))), "8-byte aligned")):
        call(**kw)
        refused(lib, text)
    assert torch.equal(x, before)
    call(rot=None)  # no rotation: a copy onto itself
    gncx.check(lib)
    assert torch.equal(x, before)


# ---- the paged cache ------------------------------------------------------------------
class Paged:
    """A layer's cache whose blocks hold values already (codes of N(0, 1) with scales to
    them, what lies behind the sequences' ends and in pages of nobody NaN codes and NaN
    scales), and the tables of some sequences.  held: tokens before the call, new: rows."""

    def __init__(self, torch, held, new, H=4, KV=2, hd=64, page=32, seed=0, spare=3, room=0, size=1.0):
        self.torch, self.held, self.new = torch, list(held), list(new)
        self.H, self.KV, self.hd, self.page = H, KV, hd, page
        need = [-(-(max(a, 0) + b) // page) for a, b in zip(held, new)]
        self.max_pages = max(max(need), 1) + room
        self.n_pages = sum(need) + spare
        rng = np.random.default_rng(seed)
        names = rng.permutation(self.n_pages)
        self.table = np.full((len(held), self.max_pages), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = names[at:at + n]
            at += n
        self.rows = sum(new)
        blocks = page // BLOCK
        self.k = torch.full((self.n_pages, KV, blocks, BLOCK, hd), 0x7f, dtype=torch.uint8, device="cuda")
        self.v = torch.full((self.n_pages, KV, blocks, hd, BLOCK), 0xff, dtype=torch.uint8, device="cuda")
        self.scales = torch.full((self.n_pages, KV, blocks, 2), float("nan"), device="cuda")
        for s, a in enumerate(held):
            if a <= 0:
                continue
            kk, vv = (size * randn(torch, 7 * s + i + seed, -(-a // BLOCK) * BLOCK, KV, hd) for i in (1, 2))
            for b in range(-(-a // BLOCK)):
                name, blk, n = int(self.table[s, b * BLOCK // page]), b * BLOCK % page // BLOCK, min(BLOCK, a - b * BLOCK)
                for x, codes, i in ((kk, self.k, 0), (vv, self.v, 1)):
                    y = x[b * BLOCK:b * BLOCK + n].transpose(0, 1)  # [KV][n][hd]
                    scale = torch.exp2(torch.ceil(torch.log2(y.abs().amax((1, 2)).double() / 448))).float()
                    q = (y / scale[:, None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
                    if i:
                        codes[name, :, blk, :, :n] = q.transpose(1, 2)
                    else:
                        codes[name, :, blk, :n] = q
                    self.scales[name, :, blk, i] = scale
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.q, self.kr, self.vr = (size * randn(torch, 90 + i + seed, max(self.rows, 1), n * hd)
                                    for i, n in enumerate((H, KV, KV)))
        self.gamma = 1 + 0.1 * randn(torch, 5 + seed, 2, hd)
        self.out = torch.full_like(self.q, float("nan"))
        self.scale = 1 / math.sqrt(hd)
        self.upload()

    def upload(self):
        torch = self.torch
        self.d_table, self.d_len, self.d_start = (torch.from_numpy(np.array(a, np.int32)).cuda()
                                                  for a in (self.table, self.held, self.starts))
        self.cache = gncx.PagedCache(self.k.data_ptr(), self.v.data_ptr(), self.scales.data_ptr(), self.n_pages,
                                     self.page, self.KV, self.hd)
        self.batch = gncx.PagedBatch(len(self.held), self.q.shape[0], self.max_pages, self.d_start.data_ptr(),
                                     self.d_len.data_ptr(), self.d_table.data_ptr())

    def append(self, lib, turn=None, norm=-1, q=True, check=True, out=None):
        out = self.out if out is None else out
        lib.gncx_hip_kv_append_paged(C.byref(self.cache), C.byref(self.batch), self.q.data_ptr() if q else None,
                                     self.kr.data_ptr(), self.vr.data_ptr(), self.H, self.gamma.data_ptr(), 0,
                                     4 * self.hd, norm, EPS, turn.ref() if turn else None, out.data_ptr() if q else None)
        if check:
            gncx.check(lib)

    def attend(self, lib, sw=0, check=True, q=None, out=None):
        q, out = self.q if q is None else q, self.out if out is None else out
        lib.gncx_hip_attention_paged(C.byref(self.cache), C.byref(self.batch), q.data_ptr(), self.H, self.scale, sw,
                                     out.data_ptr())
        if check:
            gncx.check(lib)

    def tokens(self, s, end):
        """Keys and values [end][KV][hd] (64 bits) of sequence s, and which of them are there."""
        torch = self.torch
        names = self.table[s, [t // self.page for t in range(end)]]
        there = torch.from_numpy((names >= 0) & (names < self.n_pages)).cuda()
        names = torch.from_numpy(np.where((names >= 0) & (names < self.n_pages), names, 0)).cuda().long()
        t = torch.arange(end, device="cuda")
        blk, tok = t % self.page // BLOCK, t % BLOCK
        f8 = torch.float8_e4m3fn
        k = self.k.view(f8).float().double()[names, :, blk, tok] * self.scales.double()[names, :, blk, 0, None]
        v = self.v.view(f8).float().double()[names, :, blk, :, tok] * self.scales.double()[names, :, blk, 1, None]
        return k, v, there

    def check_attention(self, q=None, out=None, sw=0):
        """out against 64 bits.  A score is off by ds <= (2^-21 + 8 sqrt(hd) u) max_j scale
        sum_d |q_d k_jd| (queries kept to 2^-22 each, roundings of the sum taken as
        independent), and by 2^-23 of the row's largest |q| for elements far below it; the
        weights are exact pieces of fp32 exponentials of 2 steps, so an output is off by
        (2 ds + 2^-20 + 8 sqrt(N) u) sum_j w_j |v_j| / l."""
        torch = self.torch
        q, out = self.q if q is None else q, self.out if out is None else out
        G = self.H // self.KV
        for s, (a, n) in enumerate(zip(self.held, self.new)):
            r0 = int(self.starts[s])
            n = min(n, self.max_pages * self.page - a)
            if n <= 0 or a < 0:
                continue
            k, v, there = self.tokens(s, a + n)
            at = torch.arange(a, a + n, device="cuda")
            key = torch.arange(a + n, device="cuda")
            see = there[None, :] & (key[None, :] <= at[:, None])
            if sw:
                see &= key[None, :] > at[:, None] - sw
            for h in range(self.H):
                qh = q[r0:r0 + n].view(n, self.H, self.hd)[:, h].double().contiguous()
                kh, vh = k[:, h // G].contiguous(), v[:, h // G].contiguous()
                # a key or value may be NaN where nobody of these rows sees it, and only there
                seen = see.any(0)[:, None]
                kh, vh = torch.where(seen, kh, 0.0), torch.where(seen, vh, 0.0)
                sc = torch.where(see, qh @ kh.t().contiguous() * self.scale, -math.inf)
                size = torch.where(see, qh.abs() @ kh.abs().t().contiguous(), 0.0).amax(1, keepdim=True) * abs(self.scale)
                far = torch.where(see, kh.abs().sum(1)[None, :], 0.0).amax(1, keepdim=True) * abs(self.scale)
                w = torch.exp(sc - sc.amax(1, keepdim=True).clamp(min=-1e300))
                l = w.sum(1, keepdim=True).clamp(min=1e-300)
                want = w @ vh / l
                ds = (2.0 ** -21 + 8 * math.sqrt(self.hd) * U) * size + 2.0 ** -36 * qh.abs().amax(1, keepdim=True) * far
                tol = (2 * ds + 2.0 ** -20 + 8 * math.sqrt(a + n) * U) * (w @ vh.abs() / l) + 1e-37
                got = out[r0:r0 + n].view(n, self.H, self.hd)[:, h].double()
                assert ((got - want).abs() <= tol).all(), (s, h, float(((got - want).abs() / tol).max()))


def nearest_e4m3(x):
    """How far a stored value may be from x / scale: half a step, 2^-4 of the power of two
    below it, 2^-10 below the normal ones."""
    return power_below(x).clamp(min=2.0 ** -6) / 16


def power_below(x):
    m, e = x.abs().frexp()
    return (0 * x + 1).ldexp(e - 1) * (m != 0)


def check_append(p, before, turn=None, norm=-1, q=True):
    """The cache after p.append(): scales, kept and new codes, and everything else as it was;
    out_q against the formula."""
    torch, f8 = p.torch, p.torch.float8_e4m3fn
    k0, v0, s0 = before
    k, v, scales = k0.clone(), v0.clone(), s0.clone()
    turn = turn or Turn(torch, 0)

    def head(x, n, gamma, at, bits=32):
        """64-bit result and how far 32 bits may be off (64: 2^-14 of that, as
        the kernel's cosine and sine, to 2^-41 of 1, count the most).  A norm's sum (positive terms) is off
        by at most 14 of its roundings, its root by half of that; with the root, the
        division and the products, 12 u of an element, and 12 u mag (|a| + |b|) turned."""
        x = x.double().view(-1, n, p.hd)
        less = 2.0 ** -14 if bits == 64 else 1.0
        if norm < 0:
            y, tol = turn(x, at)
            return y, tol * less
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
        x = x * gamma.double() if norm > 0 else x
        y, tol = turn(x, at)
        return y, (tol * (25 / 13) + 12 * U * x.abs()) * less

    for s, (a, n) in enumerate(zip(p.held, p.new)):
        room = p.max_pages * p.page
        n = min(n, room - a) if 0 <= a <= room else 0
        r0 = int(p.starts[s])
        if n <= 0:
            continue
        at = torch.arange(a, a + n, device="cuda", dtype=torch.int32)
        rows = slice(r0, r0 + n)
        if q:
            want, tol = head(p.q[rows], p.H, p.gamma[0], at)
            assert ((p.out[rows].double().view(n, p.H, p.hd) - want).abs() <= tol).all()
        wk, tk = head(p.kr[rows], p.KV, p.gamma[1], at, 64)
        wv = p.vr[rows].double().view(n, p.KV, p.hd)
        pos = a
        while pos < a + n:
            end = min(a + n, pos // BLOCK * BLOCK + BLOCK)
            name, blk = int(p.table[s, pos // p.page]), pos % p.page // BLOCK
            lo, hi = pos % BLOCK, pos % BLOCK + end - pos
            if 0 <= name < p.n_pages:
                for i, (x, tol, codes, got) in enumerate(((wk, tk, k, p.k), (wv, 0 * wv, v, p.v))):
                    y, t = (z[pos - a:end - a].transpose(0, 1) for z in (x, tol))  # [KV][tokens][hd]
                    fin = torch.where(y.isfinite(), y.abs(), 0.0)
                    most = fin.amax((1, 2))
                    scale = torch.exp2(torch.ceil(torch.log2(most / 448)).clamp(min=-100, max=120))
                    old = s0[name, :, blk, i].double()
                    if lo:
                        scale = torch.maximum(scale, old)
                    new_scale = p.scales[name, :, blk, i].double()
                    # (a rotated maximum within its error of the border may take either)
                    slack = torch.where(y.isfinite(), t, 0.0).amax((1, 2))
                    assert ((new_scale == scale) | ((most + slack > 448 * scale) & (new_scale == 2 * scale)) |
                            ((most - slack <= 224 * scale) & (2 * new_scale == scale))).all()
                    scales[name, :, blk, i] = p.scales[name, :, blk, i]
                    g = got[name, :, blk].view(f8).float()
                    c = codes[name, :, blk].view(f8).float()
                    if i:
                        g, c = g.transpose(1, 2), c.transpose(1, 2)
                    if lo:
                        kept = (c[:, :lo] * (old / new_scale).float()[:, None, None]).to(f8).float()
                        assert torch.equal(kept.nan_to_num(nan=1e9), g[:, :lo].nan_to_num(nan=1e9))
                    z = y / new_scale[:, None, None]
                    off = (g[:, lo:hi].double() - z).abs()
                    ok = torch.where(y.isfinite(), off <= nearest_e4m3(z) + t / new_scale[:, None, None], g[:, lo:hi].isnan())
                    assert ok.all()
                    full = got[name, :, blk].clone()
                    if i:
                        codes[name, :, blk, :, :hi] = full[:, :, :hi]
                    else:
                        codes[name, :, blk, :hi] = full[:, :hi]
            pos = end
    # nothing else has changed
    assert torch.equal(k, p.k) and torch.equal(v, p.v)
    assert torch.equal(scales.nan_to_num(nan=-1.0), p.scales.nan_to_num(nan=-1.0))


def state(p):
    return p.k.clone(), p.v.clone(), p.scales.clone()


@pytest.mark.parametrize("held,new", [
    ([0], [1]), ([5], [1]), ([15], [1]), ([16], [1]), ([31], [2]), ([0], [100]), ([7, 0, 33], [40, 0, 3]),
    ([0, 16, 1, 47, 100, 3], [16, 16, 15, 1, 33, 0]), ([300] * 70, [1] * 70), (list(range(67)), [1 + i % 3 for i in range(67)])])
@pytest.mark.parametrize("H,KV,hd,page,n_rot,inter,norm", [(4, 2, 64, 16, 64, 0, 1), (33, 3, 128, 32, 64, 1, 0),
                                                            (2, 1, 256, 64, 256, 0, -1), (8, 8, 128, 128, 0, 0, 1)])
def test_append(lib, torch_mod, held, new, H, KV, hd, page, n_rot, inter, norm):
    p = Paged(torch_mod, held, new, H=H, KV=KV, hd=hd, page=page)
    turn = Turn(torch_mod, n_rot, inter, 1.1) if n_rot else None
    before = state(p)
    p.append(lib, turn, norm)
    check_append(p, before, turn, norm)
    # without queries the cache is the same
    after = state(p)
    p.k, p.v, p.scales = (x.clone() for x in before)
    p.upload()
    p.append(lib, turn, norm, q=False)
    for x, y in zip(state(p), after):
        assert torch_mod.equal(x.nan_to_num(nan=-1.0) if x.is_floating_point() else x,
                               y.nan_to_num(nan=-1.0) if y.is_floating_point() else y)


def test_append_grows_a_blocks_scale_and_keeps_what_is_held(lib, torch_mod):
    """Tokens of growing size one by one: each is there to half a step of the last scale,
    as if all had come at once (codes above the subnormal ones move exactly)."""
    torch = torch_mod
    p = Paged(torch, [0], [16], H=2, KV=2, hd=64)
    rows = (p.kr.clone(), p.vr.clone())
    for x in rows:
        x.mul_(2.0 ** torch.arange(16, device="cuda")[:, None] / 64)
    p.kr, p.vr = rows
    p.append(lib)
    at_once = state(p)
    p.scales.fill_(float("nan"))
    p.starts = np.array([0, 1], np.int32)
    for t in range(16):
        p.held, p.new = [t], [1]
        p.kr, p.vr = (x[t:t + 1].clone() for x in rows)
        p.q = p.q[:1].clone()
        p.upload()
        p.append(lib)
    assert torch.equal(p.scales.nan_to_num(nan=-1), at_once[2].nan_to_num(nan=-1))
    f8 = torch.float8_e4m3fn
    for got, want in ((p.k, at_once[0]), (p.v, at_once[1])):
        a, b = got.view(f8).float(), want.view(f8).float()
        same = (a == b) | (a.isnan() & b.isnan())
        # (subnormal codes: a second rounding moves them by a step of 2^-9 at most)
        assert (same | ((b.abs() < 2.0 ** -6) & ((a - b).abs() <= 2.0 ** -9))).all()


def test_append_zeros_tiny_huge_and_non_finite_values(lib, torch_mod):
    torch = torch_mod
    p = Paged(torch, [0, 3, 0, 0, 20], [5, 4, 6, 18, 1], H=2, KV=2, hd=64)
    r = p.starts
    for x in (p.kr, p.vr):
        x[r[0]:r[1]] = 0.0                       # zeros only: the least scale
        x[r[1]:r[2]] *= 2.0 ** -120              # below the least scale's codes
        x[r[2]:r[3]] = torch.sign(x[r[2]:r[3]]) * 3.4e38
        x[r[3] + 2, 7] = float("inf")
        x[r[3] + 2, 8] = float("-inf")
        x[r[3] + 3] = float("nan")
        x[r[3] + 17, 70] = float("nan")
        x[r[4]] *= 1e-30                         # beside larger ones that are held
    before = state(p)
    p.append(lib)
    check_append(p, before)
    assert (p.scales[int(p.table[0, 0]), :, 0] == 2.0 ** -100).all()
    assert (p.scales[int(p.table[2, 0]), :, 0] == 2.0 ** 120).all()


def test_append_at_the_border_of_a_scale(lib, torch_mod):
    """448 times a power of two is reached, the next float is not; the third row's largest
    is 1, from the clamp, and 448 2^-8 is the first to reach it."""
    torch = torch_mod
    up = float(np.nextafter(np.float32(448), np.float32(1000)))
    p = Paged(torch, [0, 0, 0], [1, 1, 1], H=2, KV=1, hd=64)
    for x in (p.kr, p.vr):
        x.clamp_(-1, 1)
        x[0, 3], x[1, 3], x[2, 3] = 448.0, -up, 224.0 * 2.0 ** -10
    p.append(lib)
    for s, want in enumerate((1.0, 2.0, 2.0 ** -8)):
        assert (p.scales[int(p.table[s, 0]), :, 0] == want).all()


def test_append_of_keys_past_the_floats(lib, torch_mod):
    """A rotated key above the largest float is stored as NaN, as an infinite one is."""
    torch = torch_mod
    p = Paged(torch, [0, 5], [4, 9], H=2, KV=2, hd=64)
    turn = Turn(torch, 64)
    p.kr[2, 3] = p.kr[2, 35] = 3e38  # (pair 3 at position 2: (cos - sin, cos + sin) of 0.84)
    before = state(p)
    p.append(lib, turn)
    codes = p.k[int(p.table[0, 0]), 0, 0, 2].view(torch.float8_e4m3fn).float()
    assert codes.isnan().nonzero().view(-1).tolist() == [35]
    p.held, p.new, p.starts = [-1, 5], [4, 9], p.starts  # (the other sequence, as ever)
    p.k[int(p.table[0, 0])], p.v[int(p.table[0, 0])] = before[0][int(p.table[0, 0])], before[1][int(p.table[0, 0])]
    p.scales[int(p.table[0, 0])] = before[2][int(p.table[0, 0])]
    check_append(p, before, turn, q=False)


def test_append_leaves_rows_and_pages_that_are_not_there(lib, torch_mod):
    """Lengths outside the table, rows past its end, pages outside the pool, rows behind the
    last sequence: nothing of them is touched."""
    torch = torch_mod
    p = Paged(torch, [10, 20, 30, 76], [3, 4, 5, 8], H=4, KV=2, hd=64, page=16)
    p.max_pages, p.table = 5, p.table[:, :5].copy()  # 80 positions: room for four of the last sequence's rows
    p.q = randn(torch, 3, p.rows + 6, 4 * 64)
    p.kr, p.vr = (randn(torch, 4 + i, p.rows + 6, 2 * 64) for i in range(2))
    p.out = torch.full_like(p.q, 7.0)
    p.held[0] = -1
    p.table[1, 1] = p.n_pages
    p.table[2, 2] = -2 ** 31
    p.upload()
    before = state(p)
    p.append(lib)
    keep = p.out.clone()
    check_append(p, before)
    assert (keep[:3] == 7).all() and (keep[12 + 4:] == 7).all() and (keep[3:16] != 7).any(1).all()


def test_append_out_q_in_place_and_refusals(lib, torch_mod):
    torch = torch_mod
    p = Paged(torch, [5, 0], [2, 30], H=8, KV=2, hd=64)
    turn = Turn(torch, 64)
    before = state(p)
    p.append(lib, turn, 1)
    q, after = p.out.clone(), state(p)
    keep = p.q.clone()
    p.append(lib, turn, 1, out=p.q)
    assert torch.equal(p.q, q)
    p.q.copy_(keep)
    base = dict(cache=p.cache, batch=p.batch, q=p.q.data_ptr(), k=p.kr.data_ptr(), v=p.vr.data_ptr(),
                g=p.gamma.data_ptr(), rot=turn.ref(), out=p.out.data_ptr())

    def call(**kw):
        a = {**base, **kw}
        lib.gncx_hip_last_status()
        lib.gncx_hip_kv_append_paged(C.byref(a["cache"]), C.byref(a["batch"]), a["q"], a["k"], a["v"], 8, a["g"], 0,
                                     256, 1, EPS, a["rot"], a["out"])

    def with_(struct, **kw):
        c = type(struct)()
        C.pointer(c)[0] = struct
        for n, v in kw.items():
            setattr(c, n, v)
        return c

    memory = np.zeros(100000, np.float32)
    host = memory.ctypes.data
    for kw, text in ((dict(q=host), "GPU"), (dict(k=host), "GPU"), (dict(v=None), "GPU"), (dict(out=None), "GPU"),
                     (dict(out=p.q.data_ptr() + 16), "overlaps"), (dict(k=p.kr.data_ptr() + 4), "16-byte"),
                     (dict(out=p.kr.data_ptr()), "overlaps"),
                     (dict(cache=with_(p.cache, scales=host)), "GPU"),
                     (dict(cache=with_(p.cache, scales=p.scales.data_ptr() + 4)), "8-byte"),
                     (dict(cache=with_(p.cache, n_pages=p.n_pages + 10000)), "past the end"),
                     (dict(cache=with_(p.cache, v_pages=p.k.data_ptr())), "overlap"),
                     (dict(cache=with_(p.cache, k_pages=p.k.data_ptr() + 8)), "16-byte"),
                     (dict(batch=with_(p.batch, lengths=None)), "GPU"),
                     (dict(batch=with_(p.batch, n_rows=10 ** 6)), "past the end"),
                     (dict(batch=with_(p.batch, max_pages=10 ** 6)), "past the end"),
                     (dict(batch=with_(p.batch, pages=p.scales.data_ptr())), "overlaps an input"),
                     (dict(g=p.gamma.data_ptr() + 4), "16-byte"),
                     (dict(rot=C.byref(gncx.Rotation(turn.freqs.data_ptr(), 60, 0, 1.0))), "multiple of 8"),
                     (dict(rot=C.byref(gncx.Rotation(turn.freqs.data_ptr(), 72, 0, 1.0))), "multiple of 8")):
        call(**kw)
        refused(lib, text)
    assert torch.equal(p.k, after[0]) and torch.equal(p.v, after[1])
    assert not torch.equal(before[0], after[0])


@pytest.mark.parametrize("H,KV,hd,page", [(4, 2, 64, 16), (32, 8, 128, 64), (8, 2, 256, 32), (5, 1, 128, 256),
                                           (12, 4, 128, 128), (16, 16, 64, 32), (64, 1, 64, 16)])
@pytest.mark.parametrize("held,new", [([0], [1]), ([63], [1]), ([64], [1]), ([1, 500, 17, 0], [1, 1, 1, 1]),
                                       ([1000], [1]), ([130, 0, 700], [1, 0, 3]), ([0], [200]), ([77, 0, 300], [64, 90, 0]),
                                       ([3000, 5], [2, 1])])
@pytest.mark.parametrize("sw", [0, 100])
def test_attention(lib, torch_mod, H, KV, hd, page, held, new, sw):
    p = Paged(torch_mod, held, new, H=H, KV=KV, hd=hd, page=page, seed=3)
    p.append(lib)
    p.out.fill_(float("nan"))
    p.attend(lib, sw)
    p.check_attention(sw=sw)


@pytest.mark.parametrize("sw", [1, 16, 17, 64, 65, 10000])
@pytest.mark.parametrize("held,new", [([200, 40], [1, 1]), ([200, 40], [70, 33])])
def test_attention_windows(lib, torch_mod, sw, held, new):
    p = Paged(torch_mod, held, new, H=4, KV=2, hd=64, seed=4)
    p.append(lib)
    p.attend(lib, sw)
    p.check_attention(sw=sw)


@pytest.mark.parametrize("rows", [1, 40])
def test_attention_sees_nothing_of_hidden_places(lib, torch_mod, rows):
    """NaN and infinity-like keys and values behind a row's position, before its window, and
    in pages that are not there; a row that sees them gets NaN."""
    torch = torch_mod
    p = Paged(torch, [90, 10], [rows, rows], H=4, KV=2, hd=64, page=16, seed=5)
    p.append(lib)
    p.attend(lib, 64)
    clean = p.out.clone()
    # before every window of sequence 0
    for t in range(90 - 64 - 11, 90 - 64 + 1):
        name, blk, tok = int(p.table[0, t // 16]), 0, t % 16
        p.k[name, :, blk, tok] = 0x7f
        p.v[name, :, blk, :, tok] = 0xff
    p.attend(lib, 64)
    assert torch.equal(p.out, clean)
    # the last row's own key and value: NaN for that row alone, value: those floats alone
    last = 90 + rows - 1
    name, tok = int(p.table[0, last // 16]), last % 16
    p.v[name, 1, 0, 5, tok] = 0x7f
    p.k[name, 0, 0, tok, 9] = 0xff
    p.attend(lib, 64)
    got, want = p.out.view(2 * rows, 4, 64), clean.view(2 * rows, 4, 64)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[rows - 1, :2] = True
    bad[rows - 1, 2:, 5] = True
    assert torch.equal(got.isnan(), bad)
    assert torch.equal(got[~bad], want[~bad])


def test_attention_rows_without_anything_and_rows_that_are_none(lib, torch_mod):
    torch = torch_mod
    p = Paged(torch, [40, 50, 60, 70], [1, 3, 2, 2], H=4, KV=2, hd=64, page=16, seed=6)
    p.append(lib)
    p.q = randn(torch, 3, p.rows + 4, 4 * 64)
    p.out = torch.full_like(p.q, 7.0)
    p.table[0] = -1                         # nothing is there: zeros
    p.table[1, 1] = p.n_pages               # a hole
    p.held[2] = -5                          # no sequence
    p.held[3] = p.max_pages * 16 - 1        # the second row is past the table
    p.upload()
    p.attend(lib)
    assert (p.out[0] == 0).all()
    assert (p.out[4:6] == 7).all() and (p.out[7:] == 7).all()
    p.new = [0, 3, 0, 0]
    p.check_attention()


def test_attention_of_large_and_small_numbers(lib, torch_mod):
    """Scores of 2^24 and more, values near the largest and the least scale, queries of very
    different sizes, a row of zeros."""
    torch = torch_mod
    p = Paged(torch, [100, 100, 100, 100, 100], [1, 1, 1, 1, 2], H=4, KV=2, hd=64, seed=8)
    p.append(lib)
    p.q[0] *= 1e7
    p.q[1] *= 1e-20
    p.q[2] = 0.0
    p.q[3, ::2] *= 1e-6
    for s, e in ((2, 110), (3, -90)):
        for b in range(7):
            p.scales[int(p.table[s, b * 16 // 32]), :, b * 16 % 32 // 16, 1] *= 2.0 ** e
    p.attend(lib)
    p.check_attention()
    # a block of large values that is hidden beside small ones that are seen
    p.attend(lib, 10)
    p.check_attention(sw=10)


@pytest.mark.parametrize("bad", ["inf", "nan"])
def test_attention_of_a_query_that_is_not_finite(lib, torch_mod, bad):
    torch = torch_mod
    p = Paged(torch, [100, 20], [1, 30], H=8, KV=2, hd=64, seed=9)
    p.append(lib)
    p.attend(lib)
    want = p.out.clone()
    p.q.view(31, 8, 64)[3, 2, 7] = float(bad)
    p.attend(lib)
    hit = torch.zeros(31, 8, dtype=torch.bool, device="cuda")
    hit[3, 2] = True
    assert p.out.view(31, 8, 64)[hit].isnan().all()
    assert torch.equal(p.out.view(31, 8, 64)[~hit], want.view(31, 8, 64)[~hit])


def test_shared_pages_and_reordered_sequences(lib, torch_mod):
    """Sequences with a common beginning in the same pages, in another order: the same rows."""
    torch = torch_mod
    p = Paged(torch, [64, 64], [5, 5], H=4, KV=2, hd=64, seed=10)
    p.table[1, :2] = p.table[0, :2]
    p.upload()
    p.append(lib)
    p.attend(lib)
    p.check_attention()
    first = p.out.clone()
    p.table = p.table[::-1].copy()
    p.q, p.kr, p.vr = (torch.cat([x[5:], x[:5]]) for x in (p.q, p.kr, p.vr))
    p.upload()
    p.attend(lib)
    assert torch.equal(torch.cat([p.out[5:], p.out[:5]]), first)


def test_one_call_is_the_rows_of_many(lib, torch_mod):
    """A prompt in one call, and token by token: the same cache but for a second rounding of
    subnormal codes, outputs that agree with the cache they saw."""
    torch = torch_mod
    p = Paged(torch, [0, 0], [37, 20], H=4, KV=2, hd=64, seed=11)
    turn = Turn(torch, 64)
    p.append(lib, turn, 1)
    rq, out, at_once = p.out.clone(), torch.empty_like(p.out), state(p)
    p.attend(lib, q=rq, out=out)
    p.check_attention(q=rq, out=out)
    rows, starts, f8 = (p.kr.clone(), p.vr.clone(), p.q.clone()), p.starts, torch.float8_e4m3fn
    p.k.fill_(0x7f)
    p.v.fill_(0x7f)
    for t in range(37):
        now = [s for s in range(2) if starts[s] + t < starts[s + 1]]
        pick = [int(starts[s]) + t for s in now]
        p.held, p.new = [t if s in now else int(starts[s + 1] - starts[s]) for s in range(2)], [int(s in now) for s in range(2)]
        p.starts = np.concatenate([[0], np.cumsum(p.new)]).astype(np.int32)
        p.kr, p.vr, p.q = (x[pick].clone() for x in rows)
        p.out = torch.empty_like(p.q)
        p.upload()
        p.append(lib, turn, 1)
        assert torch.equal(p.out, rq[pick])
        p.attend(lib, q=rq[pick].clone(), out=p.q)
        p.check_attention(q=rq[pick], out=p.q)
    assert torch.equal(p.scales.nan_to_num(nan=-1), at_once[2].nan_to_num(nan=-1))
    for got, was in ((p.k, at_once[0]), (p.v, at_once[1])):
        a, b = got.view(f8).float(), was.view(f8).float()
        assert ((a == b) | (a.isnan() & b.isnan()) | ((b.abs() < 2.0 ** -6) & ((a - b).abs() <= 2.0 ** -9)) | b.isnan()).all()


def test_offsets_past_4_gib(lib, torch_mod):
    """A pool of 4.5 GiB for K and as much for V; the sequence's pages are its last ones."""
    torch = torch_mod
    n_pages = 9 * 2 ** 29 // (2 * 128 * 128) + 1
    p = Paged(torch, [300], [2], H=4, KV=2, hd=128, page=128, seed=12)
    k, v = (torch.zeros(n_pages, 2, 8, 16 * 128, dtype=torch.uint8, device="cuda") for _ in range(2))
    scales = torch.ones(n_pages, 2, 8, 2, device="cuda")
    assert k.numel() > 2 ** 32
    used = [int(x) for x in p.table[0]]
    for i, name in enumerate(used):
        k[n_pages - 1 - i] = p.k[name].view(2, 8, -1)
        v[n_pages - 1 - i] = p.v[name].view(2, 8, -1)
        scales[n_pages - 1 - i] = p.scales[name]
    want = Paged.__new__(Paged)
    want.__dict__.update(p.__dict__)
    want.append(lib)
    want.out = torch.empty_like(p.q)
    want.attend(lib)
    p.k, p.v, p.scales, p.n_pages = k, v, scales, n_pages
    p.table = np.array([[n_pages - 1 - i for i in range(len(used))]], np.int32)
    p.upload()
    p.append(lib)
    p.attend(lib)
    assert torch.equal(p.out, want.out)
    for i, name in enumerate(used):
        assert torch.equal(k[n_pages - 1 - i].view(-1), want.k[name].reshape(-1))
    assert int(k[:n_pages - len(used)].count_nonzero()) == 0


def test_attention_refusals(lib, torch_mod):
    torch = torch_mod
    p = Paged(torch, [40], [2], H=4, KV=2, hd=64)
    p.append(lib)
    p.out.fill_(7.0)
    memory = np.zeros(10000, np.float32)
    host = memory.ctypes.data

    def call(q=p.q.data_ptr(), out=p.out.data_ptr(), **kw):
        b = gncx.PagedBatch()
        C.pointer(b)[0] = p.batch
        for n, v in kw.items():
            setattr(b, n, v)
        lib.gncx_hip_last_status()
        lib.gncx_hip_attention_paged(C.byref(p.cache), C.byref(b), q, 4, p.scale, 0, out)

    for kw, text in ((dict(q=host), "GPU"), (dict(out=host), "GPU"), (dict(out=p.q.data_ptr()), "overlaps"),
                     (dict(q=p.q.data_ptr() + 4), "16-byte"), (dict(n_rows=10 ** 6), "past the end"),
                     (dict(out=p.scales.data_ptr()), "overlaps"), (dict(pages=host), "GPU"),
                     (dict(row_start=None), "GPU"), (dict(max_pages=10 ** 7), "past the end")):
        call(**kw)
        refused(lib, text)
    assert (p.out == 7.0).all()


def test_captured_decode_steps(lib, torch_mod):
    """A decode step captured once and replayed, its lengths moved on by a kernel in the
    graph, against the same steps eagerly, with other work between the replays."""
    torch = torch_mod
    turn = Turn(torch, 64)
    p = Paged(torch, [5, 40, 700], [1, 1, 1], H=4, KV=2, hd=64, page=16, room=3, seed=13)
    names = sorted(set(range(p.n_pages)) - set(p.table[p.table >= 0].tolist()))
    p.table[2, 44] = names[0] if p.table[2, 44] < 0 else p.table[2, 44]
    p.upload()
    steps = [tuple(randn(torch, 50 + 3 * i + j, 3, n * 64) for j, n in enumerate((4, 2, 2))) for i in range(4)]
    start = state(p)

    def step(i):
        for x, y in zip((p.q, p.kr, p.vr), steps[i]):
            x.copy_(y)

    rq, out = torch.empty_like(p.q), torch.empty_like(p.q)
    want = []
    for i in range(4):
        step(i)
        p.append(lib, turn, 1, out=rq)
        p.attend(lib, q=rq, out=out)
        p.d_len.add_(1)
        want.append(out.clone())
    cache = state(p)
    for x, y in zip((p.k, p.v, p.scales), start):
        x.copy_(y)
    p.d_len.copy_(whole(torch, p.held))
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    lib.gncx_hip_set_stream(stream.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            p.append(lib, turn, 1, out=rq)
            p.attend(lib, q=rq, out=out)
            p.d_len.add_(1)
        lib.gncx_hip_set_stream(None)
        other = Paged(torch, [900, 30], [1, 1], H=32, KV=8, hd=128, seed=14)
        for i in range(4):
            step(i)
            torch.cuda.synchronize()
            graph.replay()
            other.append(lib)  # eager calls beside the replay
            other.attend(lib)
            torch.cuda.synchronize()
            assert torch.equal(out, want[i])
            other.check_attention()
        for x, y in zip(state(p), cache):
            assert torch.equal(x.float().nan_to_num(nan=-1), y.float().nan_to_num(nan=-1))
    finally:
        lib.gncx_hip_set_stream(None)


def test_two_captured_graphs_beside_one_another(lib, torch_mod):
    """Two graphs of attention and log probabilities, replayed at once on two streams with
    eager calls (that grow the eager workspaces) between: each has its own parts."""
    torch = torch_mod
    sets = []
    for i, (held, new) in enumerate((([5000, 300], [1, 1]), ([2500], [40]))):
        p = Paged(torch, held, new, H=32, KV=8, hd=128, seed=40 + i)
        p.append(lib)
        p.attend(lib)
        x = 3 * randn(torch, 50 + i, 3, 60000 + 7000 * i)
        sets.append((p, p.out.clone(), x, logprobs(lib, torch, x, whole(torch, [5, 6, 7]), 9)))
    streams, graphs, outs = [torch.cuda.Stream() for _ in sets], [], []
    torch.cuda.synchronize()
    try:
        for (p, _, x, _), stream in zip(sets, streams):
            lib.gncx_hip_set_stream(stream.cuda_stream)
            graph, tokens = torch.cuda.CUDAGraph(), whole(torch, [5, 6, 7])
            out = [torch.empty(3, device="cuda"), torch.empty(3, device="cuda"),
                   torch.empty(3, 9, dtype=torch.int32, device="cuda"), torch.empty(3, 9, device="cuda")]
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=stream):
                p.attend(lib)
                lib.gncx_hip_token_logprobs(x.data_ptr(), 3, x.shape[1], tokens.data_ptr(), 9,
                                            *(t.data_ptr() for t in out))
            graphs.append(graph)
            outs.append((out, tokens))
        lib.gncx_hip_set_stream(None)
        for i in range(4):
            for (p, *_), (out, _) in zip(sets, outs):
                p.out.zero_()
                for t in out:
                    t.zero_()
            torch.cuda.synchronize()
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
            other = Paged(torch, [3000] * (1 + i), [1 + 20 * i] * (1 + i), H=32, KV=8, hd=128, seed=60 + i)
            other.append(lib)
            other.attend(lib)
            torch.cuda.synchronize()
            for (p, want, _, answer), (out, _) in zip(sets, outs):
                assert torch.equal(p.out, want) and all(torch.equal(a, b) for a, b in zip(out, answer))
            other.check_attention()
    finally:
        lib.gncx_hip_set_stream(None)


def test_calls_on_another_stream(lib, torch_mod):
    torch = torch_mod
    p = Paged(torch, [2000, 3], [1, 1], H=32, KV=8, hd=128, seed=15)
    p.append(lib)
    p.attend(lib)
    want = p.out.clone()
    stream = torch.cuda.Stream()
    try:
        for i in range(4):
            lib.gncx_hip_set_stream(stream.cuda_stream if i % 2 == 0 else None)
            p.out.fill_(0.0)
            torch.cuda.synchronize()
            p.attend(lib)
            torch.cuda.synchronize()
            assert torch.equal(p.out, want)
    finally:
        lib.gncx_hip_set_stream(None)


@pytest.mark.parametrize("seqs,most", [(65, 90), (300, 40), (2100, 0), (4200, 0)])
@pytest.mark.parametrize("new", [1, 3])
def test_many_sequences(lib, torch_mod, seqs, most, new):
    """More sequences than a wave has lanes, some without rows; 2100 without a split."""
    rng = np.random.default_rng(seqs)
    held = rng.integers(0, most + 1, seqs).tolist()
    p = Paged(torch_mod, held, [0 if i % 7 == 3 else new for i in range(seqs)], H=2, KV=1, hd=64, page=16, seed=30)
    p.append(lib)
    p.attend(lib)
    p.check_attention()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new,sw,bad", [(1, 0, False), (3, 40, False), (2, 0, True)])
def test_many_short_sequences(lib, torch_mod, hd, new, sw, bad):
    """More than 2048 (sequence, KV head) pairs of few steps: a wave each; with NaN codes in
    held tokens of some sequences, which only those meet."""
    torch = torch_mod
    rng = np.random.default_rng(hd)
    held = rng.integers(0, 400, 300).tolist()
    p = Paged(torch, held, [0 if i % 9 == 4 else new for i in range(300)], H=16, KV=8, hd=hd, page=32, seed=35)
    p.append(lib)
    if bad:
        for s in range(0, 300, 50):
            if held[s]:
                p.v[int(p.table[s, 0]), 3, 0, 5, 0] = 0x7f
    p.attend(lib, sw)
    if bad:
        seen = torch.zeros_like(p.out, dtype=torch.bool).view(-1, 16, hd)
        for s in range(0, 300, 50):
            if held[s]:
                seen[int(p.starts[s]):int(p.starts[s + 1]), 6:8, 5] = True
        rows = int(p.starts[-1])
        assert torch.equal(p.out.view(-1, 16, hd)[:rows].isnan(), seen[:rows])
        p.out.nan_to_num_(nan=0.0)
        for s in range(0, 300, 50):
            if held[s]:
                p.v[int(p.table[s, 0]), 3, 0, 5, 0] = 0
                p.out.view(-1, 16, hd)[int(p.starts[s]):int(p.starts[s + 1]), 6:8, 5] = math.nan
        p.held = [-1 if s % 50 == 0 else a for s, a in enumerate(held)]  # (checked above)
    p.check_attention(sw=sw)


@pytest.mark.parametrize("sw", [1, 70, 300, 2 ** 31 - 1])
@pytest.mark.parametrize("H,KV,hd", [(8, 2, 128), (3, 1, 64), (6, 2, 256)])
def test_windows_of_long_prompts(lib, torch_mod, sw, H, KV, hd):
    p = Paged(torch_mod, [2000, 0], [600, 130], H=H, KV=KV, hd=hd, seed=31)
    p.append(lib)
    p.attend(lib, sw)
    p.check_attention(sw=sw)


@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0])
@pytest.mark.parametrize("new", [1, 50])
def test_scales_of_the_scores(lib, torch_mod, scale, new):
    p = Paged(torch_mod, [300], [new], H=4, KV=2, hd=64, seed=32)
    p.scale = scale
    p.append(lib)
    p.attend(lib)
    p.check_attention()


@pytest.mark.parametrize("starts", [[0, 60, 20, 90], [90, 60, 30, 0], [-5, 1000000, -7, 90], [0, 90, 0, 90]])
@pytest.mark.parametrize("held", [[10, 700, 3], [2000, 2000, 2000]])
def test_row_starts_that_do_not_ascend(lib, torch_mod, starts, held):
    """What such rows receive is open; rows that are not the call's, and pages that no table
    names, stay as they are, and the next call is answered."""
    torch = torch_mod
    p = Paged(torch, held, [30, 30, 30], H=8, KV=2, hd=64, seed=33, room=3)
    free = sorted(set(range(p.n_pages)) - set(p.table.ravel().tolist()))
    p.starts = np.array(starts, np.int32)
    p.upload()
    behind = torch.full((40, 8 * 64), 7.0, device="cuda")
    buffers = [torch.cat([x, behind]) for x in (p.q, p.out)]
    p.batch.n_rows = 90
    before = state(p)
    p.append(lib, Turn(torch, 64), 1, out=buffers[0][:90])
    p.attend(lib, out=buffers[1][:90])
    torch.cuda.synchronize()
    assert torch.equal(buffers[0][90:], behind) and torch.equal(buffers[1][90:], behind)
    for now, was in zip(state(p), before):
        assert torch.equal(now[free].float().nan_to_num(nan=-1), was[free].float().nan_to_num(nan=-1))
    other = Paged(torch, [100], [1], seed=34)
    other.append(lib)
    other.attend(lib)
    other.check_attention()


def check_around_nan(lib, p, places, sw=0):
    """Attention with NaN codes at places (sequence, position, KV head, float) among the
    values: NaN in that float of the rows that see it, everything else against 64 bits."""
    torch, G = p.torch, p.H // p.KV
    bad = torch.zeros(p.out.shape[0], p.H, p.hd, dtype=torch.bool, device="cuda")
    codes = []
    for s, t, b, d in places:
        codes.append((int(p.table[s, t // p.page]), b, t % p.page // BLOCK, d, t % BLOCK))
        r0, a = int(p.starts[s]), p.held[s]
        last = min(p.new[s], t + sw - a) if sw else p.new[s]
        bad[r0 + max(t - a, 0):r0 + last, b * G:(b + 1) * G, d] = True
    for at in codes:
        p.v[at] = 0x7f
    p.attend(lib, sw)
    got = p.out.clone()
    assert torch.equal(got.isnan().view(bad.shape), bad)
    for at in codes:
        p.v[at] = 0
    p.attend(lib, sw)
    p.check_attention(out=torch.where(bad.view(got.shape), p.out, got), sw=sw)


def grow_values(p, s, t, e):
    """The values of the block of sequence s's position t times 2^e."""
    p.scales[int(p.table[s, t // p.page]), :, t % p.page // BLOCK, 1] *= 2.0 ** e


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("held,new,sw", [([600, 30], [1, 1], 0), ([600, 620], [3, 3], 0), ([610], [3], 500),
                                         ([1000, 20], [90, 70], 0)])
def test_nan_values_in_a_step_whose_scale_grows(lib, torch_mod, hd, held, new, sw):
    """A NaN code among the values of the last, partial step, whose scale is above those of
    the wave's steps before: other floats, and rows that do not see it, are as without it."""
    p = Paged(torch_mod, held, new, H=4, KV=2, hd=hd, page=32, seed=70)
    p.append(lib)
    ends = [a + n - 1 for a, n in zip(held, new)]
    for s, t in enumerate(ends):
        grow_values(p, s, t, 3)
    check_around_nan(lib, p, [(s, t, 1, 5 + s) for s, t in enumerate(ends)], sw)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 3])
def test_nan_values_of_many_short_sequences_whose_scales_grow(lib, torch_mod, hd, new):
    """The same where each sequence and KV head is a wave's."""
    held = np.random.default_rng(hd).integers(100, 400, 300).tolist()
    p = Paged(torch_mod, held, [new] * 300, H=16, KV=8, hd=hd, page=32, seed=71)
    p.append(lib)
    places = [(s, held[s] + new - 1, s % 8, s % hd) for s in range(0, 300, 7)]
    for s, t, _, _ in places:
        grow_values(p, s, t, 3)
    check_around_nan(lib, p, places)


def check_around_nan(lib, p, places, sw=0):
    """Attention with NaN codes at places (sequence, position, KV head, float) among the
    values: NaN in that float of the rows that see it, everything else against 64 bits."""
    torch, G = p.torch, p.H // p.KV
    bad = torch.zeros(p.out.shape[0], p.H, p.hd, dtype=torch.bool, device="cuda")
    codes = []
    for s, t, b, d in places:
        codes.append((int(p.table[s, t // p.page]), b, t % p.page // BLOCK, d, t % BLOCK))
        r0, a = int(p.starts[s]), p.held[s]
        last = min(p.new[s], t + sw - a) if sw else p.new[s]
        bad[r0 + max(t - a, 0):r0 + last, b * G:(b + 1) * G, d] = True
    for at in codes:
        p.v[at] = 0x7f
    p.attend(lib, sw)
    got = p.out.clone()
    assert torch.equal(got.isnan().view(bad.shape), bad)
    for at in codes:
        p.v[at] = 0
    p.attend(lib, sw)
    p.check_attention(out=torch.where(bad.view(got.shape), p.out, got), sw=sw)


def grow_values(p, s, t, e):
    """The values of the block of sequence s's position t times 2^e."""
    p.scales[int(p.table[s, t // p.page]), :, t % p.page // BLOCK, 1] *= 2.0 ** e


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("held,new,sw", [([600, 30], [1, 1], 0), ([600, 620], [3, 3], 0), ([610], [3], 500),
                                         ([1000, 20], [90, 70], 0)])
def test_nan_values_in_a_step_whose_scale_grows(lib, torch_mod, hd, held, new, sw):
    """A NaN code among the values of the last, partial step, whose scale is above those of
    the wave's steps before: other floats, and rows that do not see it, are as without it."""
    p = Paged(torch_mod, held, new, H=4, KV=2, hd=hd, page=32, seed=70)
    p.append(lib)
    ends = [a + n - 1 for a, n in zip(held, new)]
    for s, t in enumerate(ends):
        grow_values(p, s, t, 3)
    check_around_nan(lib, p, [(s, t, 1, 5 + s) for s, t in enumerate(ends)], sw)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 3])
def test_nan_values_of_many_short_sequences_whose_scales_grow(lib, torch_mod, hd, new):
    """The same where each sequence and KV head is a wave's."""
    held = np.random.default_rng(hd).integers(100, 400, 300).tolist()
    p = Paged(torch_mod, held, [new] * 300, H=16, KV=8, hd=hd, page=32, seed=71)
    p.append(lib)
    places = [(s, held[s] + new - 1, s % 8, s % hd) for s in range(0, 300, 7)]
    for s, t, _, _ in places:
        grow_values(p, s, t, 3)
    check_around_nan(lib, p, places)


# held, new, H, KV: decode rows, prompts, and a wave for each sequence and KV head
FORMS = [([100, 700], [1, 1], 4, 2), ([600], [70], 4, 2), ([70 + 2 * i for i in range(130)], [1] * 130, 16, 16)]


@pytest.mark.parametrize("held,new,H,KV", FORMS)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_of_very_small_and_very_large_factors(lib, torch_mod, held, new, H, KV, hd):
    """Queries near the least float, beside keys of zeros, of ordinary size and near the
    largest; a tiny scale of the scores."""
    torch = torch_mod
    p = Paged(torch, held, new, H=H, KV=KV, hd=hd, page=16, seed=74)
    p.append(lib)
    q, scales = p.q.clone(), p.scales.clone()
    for big in (1.0, 1e-10, 1e-20, 1e-38):
        p.q = big * q
        p.attend(lib)
        p.check_attention()
    # products that are ordinary numbers: 2^-125 2^125
    p.q = q * 2.0 ** -125
    p.scales[..., 0] *= 2.0 ** 125
    p.attend(lib)
    p.check_attention()
    p.scales.copy_(scales)
    # keys of zeros: the first two blocks' and every third one's
    for s, (a, n) in enumerate(zip(held, new)):
        for t in range(0, a + n, BLOCK):
            if t < 2 * BLOCK or t // BLOCK % 3 == 0:
                p.k[int(p.table[s, t // 16])] = 0
                p.scales[int(p.table[s, t // 16]), ..., 0] = 2.0 ** -100
    for big in (1.0, 1e-10, 1e-20, 1e-38):
        p.q = big * q
        p.attend(lib)
        p.check_attention()
    p.q, p.scale = q, 1e-30
    p.attend(lib)
    p.check_attention()


@pytest.mark.parametrize("new", [1, 70])
def test_attention_of_large_queries_and_keys_that_do_not_meet(lib, torch_mod, new):
    """Queries with one large float, keys that are zero there and large elsewhere: every
    score is zero, and the output the mean of the values."""
    torch = torch_mod
    p = Paged(torch, [200], [new], H=4, KV=2, hd=64, page=16, seed=75)
    p.append(lib)
    p.k[..., 7] = 0
    p.scales[..., 0] *= 2.0 ** 90
    p.q.zero_().view(new, 4, 64)[..., 7] = 2.0 ** 100
    p.attend(lib)
    _, v, _ = p.tokens(0, 200 + new)
    v = v.repeat_interleave(2, 1)
    for i in range(new):
        x = v[:201 + i]
        assert ((p.out.view(new, 4, 64)[i] - x.mean(0)).abs() <= 2.0 ** -20 * x.abs().mean(0)).all()


def check_around_nan(lib, p, places, sw=0):
    """Attention with NaN codes at places (sequence, position, KV head, float) among the
    values: NaN in that float of the rows that see it, everything else against 64 bits."""
    torch, G = p.torch, p.H // p.KV
    bad = torch.zeros(p.out.shape[0], p.H, p.hd, dtype=torch.bool, device="cuda")
    codes = []
    for s, t, b, d in places:
        codes.append((int(p.table[s, t // p.page]), b, t % p.page // BLOCK, d, t % BLOCK))
        r0, a = int(p.starts[s]), p.held[s]
        last = min(p.new[s], t + sw - a) if sw else p.new[s]
        bad[r0 + max(t - a, 0):r0 + last, b * G:(b + 1) * G, d] = True
    for at in codes:
        p.v[at] = 0x7f
    p.attend(lib, sw)
    got = p.out.clone()
    assert torch.equal(got.isnan().view(bad.shape), bad)
    for at in codes:
        p.v[at] = 0
    p.attend(lib, sw)
    p.check_attention(out=torch.where(bad.view(got.shape), p.out, got), sw=sw)


def grow_values(p, s, t, e):
    """The values of the block of sequence s's position t times 2^e."""
    p.scales[int(p.table[s, t // p.page]), :, t % p.page // BLOCK, 1] *= 2.0 ** e


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("held,new,sw", [([600, 30], [1, 1], 0), ([600, 620], [3, 3], 0), ([610], [3], 500),
                                         ([1000, 20], [90, 70], 0)])
def test_nan_values_in_a_step_whose_scale_grows(lib, torch_mod, hd, held, new, sw):
    """A NaN code among the values of the last, partial step, whose scale is above those of
    the wave's steps before: other floats, and rows that do not see it, are as without it."""
    p = Paged(torch_mod, held, new, H=4, KV=2, hd=hd, page=32, seed=70)
    p.append(lib)
    ends = [a + n - 1 for a, n in zip(held, new)]
    for s, t in enumerate(ends):
        grow_values(p, s, t, 3)
    check_around_nan(lib, p, [(s, t, 1, 5 + s) for s, t in enumerate(ends)], sw)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 3])
def test_nan_values_of_many_short_sequences_whose_scales_grow(lib, torch_mod, hd, new):
    """The same where each sequence and KV head is a wave's."""
    held = np.random.default_rng(hd).integers(100, 400, 300).tolist()
    p = Paged(torch_mod, held, [new] * 300, H=16, KV=8, hd=hd, page=32, seed=71)
    p.append(lib)
    places = [(s, held[s] + new - 1, s % 8, s % hd) for s in range(0, 300, 7)]
    for s, t, _, _ in places:
        grow_values(p, s, t, 3)
    check_around_nan(lib, p, places)


# held, new, H, KV: decode rows, prompts, and a wave for each sequence and KV head
FORMS = [([100, 700], [1, 1], 4, 2), ([600], [70], 4, 2), ([70 + 2 * i for i in range(130)], [1] * 130, 16, 16)]


@pytest.mark.parametrize("held,new,H,KV", FORMS)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_of_very_small_and_very_large_factors(lib, torch_mod, held, new, H, KV, hd):
    """Queries near the least float, beside keys of zeros, of ordinary size and near the
    largest; a tiny scale of the scores."""
    torch = torch_mod
    p = Paged(torch, held, new, H=H, KV=KV, hd=hd, page=16, seed=74)
    p.append(lib)
    q, scales = p.q.clone(), p.scales.clone()
    for big in (1.0, 1e-10, 1e-20, 1e-38):
        p.q = big * q
        p.attend(lib)
        p.check_attention()
    # products that are ordinary numbers: 2^-125 2^125
    p.q = q * 2.0 ** -125
    p.scales[..., 0] *= 2.0 ** 125
    p.attend(lib)
    p.check_attention()
    p.scales.copy_(scales)
    # keys of zeros: the first two blocks' and every third one's
    for s, (a, n) in enumerate(zip(held, new)):
        for t in range(0, a + n, BLOCK):
            if t < 2 * BLOCK or t // BLOCK % 3 == 0:
                p.k[int(p.table[s, t // 16])] = 0
                p.scales[int(p.table[s, t // 16]), ..., 0] = 2.0 ** -100
    for big in (1.0, 1e-10, 1e-20, 1e-38):
        p.q = big * q
        p.attend(lib)
        p.check_attention()
    p.q, p.scale = q, 1e-30
    p.attend(lib)
    p.check_attention()


@pytest.mark.parametrize("new", [1, 70])
def test_attention_of_large_queries_and_keys_that_do_not_meet(lib, torch_mod, new):
    """Queries with one large float, keys that are zero there and large elsewhere: every
    score is zero, and the output the mean of the values."""
    torch = torch_mod
    p = Paged(torch, [200], [new], H=4, KV=2, hd=64, page=16, seed=75)
    p.append(lib)
    p.k[..., 7] = 0
    p.scales[..., 0] *= 2.0 ** 90
    p.q.zero_().view(new, 4, 64)[..., 7] = 2.0 ** 100
    p.attend(lib)
    _, v, _ = p.tokens(0, 200 + new)
    v = v.repeat_interleave(2, 1)
    for i in range(new):
        x = v[:201 + i]
        assert ((p.out.view(new, 4, 64)[i] - x.mean(0)).abs() <= 2.0 ** -20 * x.abs().mean(0)).all()


@pytest.mark.parametrize("e", [22, 24, 25, 27, 31, 60])
@pytest.mark.parametrize("held,new,H,KV", FORMS)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_of_large_scores(lib, torch_mod, e, held, new, H, KV, hd):
    """Queries of 2^e: where one key's score is above all others by more than both may be off
    (check_attention's ds) and 30, it has all the weight, and the output is its value."""
    torch = torch_mod
    p = Paged(torch, held, new, H=H, KV=KV, hd=hd, seed=72)
    p.append(lib)
    p.q *= 2.0 ** e
    p.attend(lib)
    assert p.out.isfinite().all()
    rows = clear = 0
    for s in range(0, len(held), 1 + len(held) // 40):
        a, n, r0 = held[s], new[s], int(p.starts[s])
        k, v, _ = p.tokens(s, a + n)
        hidden = torch.arange(a + n, device="cuda")[None, :] > torch.arange(a, a + n, device="cuda")[:, None]
        for h in range(H):
            q = p.q[r0:r0 + n].view(n, H, hd)[:, h].double().contiguous()
            kh, vh = k[:, h // (H // KV)].contiguous(), v[:, h // (H // KV)].contiguous()
            sc = (q @ kh.t().contiguous() * p.scale).masked_fill(hidden, -math.inf)
            size = (q.abs() @ kh.abs().t().contiguous() * p.scale).amax(1)
            far = kh.abs().sum(1).amax() * p.scale
            ds = (2.0 ** -21 + 8 * math.sqrt(hd) * U) * size + 2.0 ** -36 * q.abs().amax(1) * far
            top = sc.topk(2, dim=1)
            lead = top.values[:, 0] - top.values[:, 1] > 2 * ds + 30
            want = vh[top.indices[:, 0]]
            off = (p.out[r0:r0 + n].view(n, H, hd)[:, h].double() - want).abs()
            assert (off <= 2.0 ** -20 * want.abs())[lead].all()
            rows, clear = rows + n, clear + int(lead.sum())
    assert 2 * clear > rows


@pytest.mark.parametrize("e", range(18, 32))
@pytest.mark.parametrize("new", [1, 70])
def test_equal_large_scores_weigh_the_same(lib, torch_mod, e, new):
    """Two blocks of the same keys whose values' scales differ by odd powers of two: the
    query's best keys, one of each, have half the weight each."""
    torch = torch_mod
    p = Paged(torch, [200], [new], H=2, KV=2, hd=64, page=16, seed=73)
    p.append(lib)
    one, two = int(p.table[0, 3]), int(p.table[0, 8])
    p.k[two], p.scales[two, ..., 0] = p.k[one], p.scales[one, ..., 0]
    grow_values(p, 0, 8 * 16, -3)
    k, v, _ = p.tokens(0, 200)
    p.q.view(new, 2, 64).copy_(2.0 ** e * k[3 * 16 + 5])  # (its score is |k|^2 2^e / 8, 2^(e + 3), far above the others)
    p.attend(lib)
    want = (v[3 * 16 + 5] + v[8 * 16 + 5]) / 2
    size = (v[3 * 16 + 5].abs() + v[8 * 16 + 5].abs()) / 2
    assert ((p.out.view(new, 2, 64).double() - want).abs() <= 2.0 ** -20 * size).all()


def check_around_nan(lib, p, places, sw=0):
    """Attention with NaN codes at places (sequence, position, KV head, float) among the
    values: NaN in that float of the rows that see it, everything else against 64 bits."""
    torch, G = p.torch, p.H // p.KV
    bad = torch.zeros(p.out.shape[0], p.H, p.hd, dtype=torch.bool, device="cuda")
    codes = []
    for s, t, b, d in places:
        codes.append((int(p.table[s, t // p.page]), b, t % p.page // BLOCK, d, t % BLOCK))
        r0, a = int(p.starts[s]), p.held[s]
        last = min(p.new[s], t + sw - a) if sw else p.new[s]
        bad[r0 + max(t - a, 0):r0 + last, b * G:(b + 1) * G, d] = True
    for at in codes:
        p.v[at] = 0x7f
    p.attend(lib, sw)
    got = p.out.clone()
    assert torch.equal(got.isnan().view(bad.shape), bad)
    for at in codes:
        p.v[at] = 0
    p.attend(lib, sw)
    p.check_attention(out=torch.where(bad.view(got.shape), p.out, got), sw=sw)


def grow_values(p, s, t, e):
    """The values of the block of sequence s's position t times 2^e."""
    p.scales[int(p.table[s, t // p.page]), :, t % p.page // BLOCK, 1] *= 2.0 ** e


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("held,new,sw", [([600, 30], [1, 1], 0), ([600, 620], [3, 3], 0), ([610], [3], 500),
                                         ([1000, 20], [90, 70], 0)])
def test_nan_values_in_a_step_whose_scale_grows(lib, torch_mod, hd, held, new, sw):
    """A NaN code among the values of the last, partial step, whose scale is above those of
    the wave's steps before: other floats, and rows that do not see it, are as without it."""
    p = Paged(torch_mod, held, new, H=4, KV=2, hd=hd, page=32, seed=70)
    p.append(lib)
    ends = [a + n - 1 for a, n in zip(held, new)]
    for s, t in enumerate(ends):
        grow_values(p, s, t, 3)
    check_around_nan(lib, p, [(s, t, 1, 5 + s) for s, t in enumerate(ends)], sw)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 3])
def test_nan_values_of_many_short_sequences_whose_scales_grow(lib, torch_mod, hd, new):
    """The same where each sequence and KV head is a wave's."""
    held = np.random.default_rng(hd).integers(100, 400, 300).tolist()
    p = Paged(torch_mod, held, [new] * 300, H=16, KV=8, hd=hd, page=32, seed=71)
    p.append(lib)
    places = [(s, held[s] + new - 1, s % 8, s % hd) for s in range(0, 300, 7)]
    for s, t, _, _ in places:
        grow_values(p, s, t, 3)
    check_around_nan(lib, p, places)


# held, new, H, KV: decode rows, prompts, and a wave for each sequence and KV head
FORMS = [([100, 700], [1, 1], 4, 2), ([600], [70], 4, 2), ([70 + 2 * i for i in range(130)], [1] * 130, 16, 16)]


@pytest.mark.parametrize("held,new,H,KV", FORMS)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_of_very_small_and_very_large_factors(lib, torch_mod, held, new, H, KV, hd):
    """Queries near the least float, beside keys of zeros, of ordinary size and near the
    largest; a tiny scale of the scores."""
    torch = torch_mod
    p = Paged(torch, held, new, H=H, KV=KV, hd=hd, page=16, seed=74)
    p.append(lib)
    q, scales = p.q.clone(), p.scales.clone()
    for big in (1.0, 1e-10, 1e-20, 1e-38):
        p.q = big * q
        p.attend(lib)
        p.check_attention()
    # products that are ordinary numbers: 2^-125 2^125
    p.q = q * 2.0 ** -125
    p.scales[..., 0] *= 2.0 ** 125
    p.attend(lib)
    p.check_attention()
    p.scales.copy_(scales)
    # keys of zeros: the first two blocks' and every third one's
    for s, (a, n) in enumerate(zip(held, new)):
        for t in range(0, a + n, BLOCK):
            if t < 2 * BLOCK or t // BLOCK % 3 == 0:
                p.k[int(p.table[s, t // 16])] = 0
                p.scales[int(p.table[s, t // 16]), ..., 0] = 2.0 ** -100
    for big in (1.0, 1e-10, 1e-20, 1e-38):
        p.q = big * q
        p.attend(lib)
        p.check_attention()
    p.q, p.scale = q, 1e-30
    p.attend(lib)
    p.check_attention()


@pytest.mark.parametrize("new", [1, 70])
def test_attention_of_large_queries_and_keys_that_do_not_meet(lib, torch_mod, new):
    """Queries with one large float, keys that are zero there and large elsewhere: every
    score is zero, and the output the mean of the values."""
    torch = torch_mod
    p = Paged(torch, [200], [new], H=4, KV=2, hd=64, page=16, seed=75)
    p.append(lib)
    p.k[..., 7] = 0
    p.scales[..., 0] *= 2.0 ** 90
    p.q.zero_().view(new, 4, 64)[..., 7] = 2.0 ** 100
    p.attend(lib)
    _, v, _ = p.tokens(0, 200 + new)
    v = v.repeat_interleave(2, 1)
    for i in range(new):
        x = v[:201 + i]
        assert ((p.out.view(new, 4, 64)[i] - x.mean(0)).abs() <= 2.0 ** -20 * x.abs().mean(0)).all()


@pytest.mark.parametrize("e", [22, 24, 25, 27, 31, 60])
@pytest.mark.parametrize("held,new,H,KV", FORMS)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_of_large_scores(lib, torch_mod, e, held, new, H, KV, hd):
    """Queries of 2^e: where one key's score is above all others by more than both may be off
    (check_attention's ds) and 30, it has all the weight, and the output is its value."""
    torch = torch_mod
    p = Paged(torch, held, new, H=H, KV=KV, hd=hd, seed=72)
    p.append(lib)
    p.q *= 2.0 ** e
    p.attend(lib)
    assert p.out.isfinite().all()
    rows = clear = 0
    for s in range(0, len(held), 1 + len(held) // 40):
        a, n, r0 = held[s], new[s], int(p.starts[s])
        k, v, _ = p.tokens(s, a + n)
        hidden = torch.arange(a + n, device="cuda")[None, :] > torch.arange(a, a + n, device="cuda")[:, None]
        for h in range(H):
            q = p.q[r0:r0 + n].view(n, H, hd)[:, h].double().contiguous()
            kh, vh = k[:, h // (H // KV)].contiguous(), v[:, h // (H // KV)].contiguous()
            sc = (q @ kh.t().contiguous() * p.scale).masked_fill(hidden, -math.inf)
            size = (q.abs() @ kh.abs().t().contiguous() * p.scale).amax(1)
            far = kh.abs().sum(1).amax() * p.scale
            ds = (2.0 ** -21 + 8 * math.sqrt(hd) * U) * size + 2.0 ** -36 * q.abs().amax(1) * far
            top = sc.topk(2, dim=1)
            lead = top.values[:, 0] - top.values[:, 1] > 2 * ds + 30
            want = vh[top.indices[:, 0]]
            off = (p.out[r0:r0 + n].view(n, H, hd)[:, h].double() - want).abs()
            assert (off <= 2.0 ** -20 * want.abs())[lead].all()
            rows, clear = rows + n, clear + int(lead.sum())
    assert 2 * clear > rows


@pytest.mark.parametrize("e", range(18, 32))
@pytest.mark.parametrize("new", [1, 70])
def test_equal_large_scores_weigh_the_same(lib, torch_mod, e, new):
    """Two blocks of the same keys whose values' scales differ by odd powers of two: the
    query's best keys, one of each, have half the weight each."""
    torch = torch_mod
    p = Paged(torch, [200], [new], H=2, KV=2, hd=64, page=16, seed=73)
    p.append(lib)
    one, two = int(p.table[0, 3]), int(p.table[0, 8])
    p.k[two], p.scales[two, ..., 0] = p.k[one], p.scales[one, ..., 0]
    grow_values(p, 0, 8 * 16, -3)
    k, v, _ = p.tokens(0, 200)
    p.q.view(new, 2, 64).copy_(2.0 ** e * k[3 * 16 + 5])  # (its score is |k|^2 2^e / 8, 2^(e + 3), far above the others)
    p.attend(lib)
    want = (v[3 * 16 + 5] + v[8 * 16 + 5]) / 2
    size = (v[3 * 16 + 5].abs() + v[8 * 16 + 5].abs()) / 2
    assert ((p.out.view(new, 2, 64).double() - want).abs() <= 2.0 ** -20 * size).all()


def grow_all_values(p, exponents):
    """Every held or new block's values times 2^e, e = exponents(sequence, block)."""
    for s, (a, n) in enumerate(zip(p.held, p.new)):
        for t in range(0, a + n, BLOCK):
            grow_values(p, s, t, exponents(s, t // BLOCK))


@pytest.mark.parametrize("held,new,H,KV", FORMS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("sw", [0, 90])
def test_values_of_scales_far_apart(lib, torch_mod, held, new, H, KV, hd, sw):
    """Blocks of values more than 2^16 apart, near and far, in any order; blocks of zeros."""
    torch = torch_mod
    p = Paged(torch, held, new, H=H, KV=KV, hd=hd, page=16, seed=76)
    p.append(lib)
    kept = p.scales.clone()
    rng = np.random.default_rng(hd)
    for span in (17, 40, 110):
        p.scales.copy_(kept)
        grow_all_values(p, lambda s, b: int(rng.integers(-min(span, 90), span)))
        p.attend(lib, sw)
        p.check_attention(sw=sw)
    for first in (True, False):  # (rising and falling through the sequence)
        p.scales.copy_(kept)
        grow_all_values(p, lambda s, b: min(6 * b - 90, 110) if first else max(110 - 6 * b, -90))
        p.attend(lib, sw)
        p.check_attention(sw=sw)
    p.scales.copy_(kept)
    for s, (a, n) in enumerate(zip(held, new)):
        for t in range(16 * (s % 3), a + n, 48):
            p.v[int(p.table[s, t // 16])] = 0
            p.scales[int(p.table[s, t // 16]), ..., 1] = 2.0 ** -100
    p.attend(lib, sw)
    p.check_attention(sw=sw)


@pytest.mark.parametrize("held,new,H,KV", FORMS)
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("low", [-30.0, -45.0, -300.0])
def test_large_values_of_little_weight(lib, torch_mod, held, new, H, KV, hd, low):
    """Blocks of values of 2^110 whose keys have weights of about e^low, beside blocks of small
    values: what the large ones leave of the sum, nothing for e^-300, is what counts."""
    torch = torch_mod
    p = Paged(torch, held, new, H=H, KV=KV, hd=hd, page=16, seed=77)
    p.append(lib)
    p.q.view(-1, H, hd)[..., 3] = 128.0 * math.sqrt(hd)  # (scores are 128 k_3 and an ordinary rest)
    big, small = {-30.0: (50, 0), -45.0: (80, 0), -300.0: (110, -80)}[low]
    grow_all_values(p, lambda s, b: big if b % 5 == 2 else small)
    f8 = torch.float8_e4m3fn
    k = p.k.view(f8).float()
    k[..., 3] = 0
    for s, (a, n) in enumerate(zip(held, new)):
        for t in range(2 * BLOCK, a + n, 5 * BLOCK):
            name = int(p.table[s, t // 16])
            k[name, ..., 3] = low / 128.0 / p.scales[name, :, 0, 0][:, None, None]
    assert (k[..., 3].nan_to_num() >= -448).all()
    p.k.copy_(k.to(f8).view(torch.uint8))
    p.attend(lib)
    p.check_attention()


@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("held,new", [([600, 620], [3, 3]), ([1000, 20], [90, 70])])
def test_nan_values_among_scales_far_apart(lib, torch_mod, hd, held, new):
    p = Paged(torch_mod, held, new, H=4, KV=2, hd=hd, page=16, seed=78)
    p.append(lib)
    grow_all_values(p, lambda s, b: (0, 30, -40, 3, 60)[b % 5])
    places = [(s, a + n - 1, 1, 5) for s, (a, n) in enumerate(zip(held, new))]
    check_around_nan(lib, p, places + [(0, held[0], 0, 9), (1, held[1] + 1, 0, 40)])


def test_scores_past_the_floats(lib, torch_mod):
    """A row with a score above the largest float is NaN, others are as ever."""
    torch = torch_mod
    p = Paged(torch, [100, 30], [1, 40], H=4, KV=2, hd=64, seed=83)
    p.append(lib)
    p.q *= 2.0 ** -20
    p.scale *= 2.0 ** 20
    p.attend(lib)
    want = p.out.clone()
    p.check_attention()
    k, _, _ = p.tokens(0, 101)
    p.q.view(41, 4, 64)[0, 1] = (k[50, 0] * 2.0 ** 120).float()  # (a score of |k|^2 2^137)
    p.attend(lib)
    bad = torch.zeros(41, 4, 64, dtype=torch.bool, device="cuda")
    bad[0, 1] = True
    bad = bad.view(want.shape)
    assert torch.equal(p.out.isnan(), bad)
    assert (p.out - want)[~bad].abs().max() <= 2.0 ** -19 * want[~bad].abs().max()


# ---- log probabilities ------------------------------------------------------------------
def logprobs(lib, torch, x, tokens, n_top, entropy=True):
    rows, vocab = x.shape
    lp, en = (torch.full((rows,), 7.0, device="cuda") for _ in range(2))
    words = torch.full((rows, n_top), 7, dtype=torch.int32, device="cuda")
    best = torch.full((rows, n_top), 7.0, device="cuda")
    lib.gncx_hip_token_logprobs(x.data_ptr(), rows, vocab, None if tokens is None else tokens.data_ptr(), n_top,
                                None if tokens is None else lp.data_ptr(), en.data_ptr() if entropy else None,
                                words.data_ptr() if n_top else None, best.data_ptr() if n_top else None)
    gncx.check(lib)
    return lp, en, words, best


def check_logprobs(torch, x, tokens, n_top, got):
    """Against 64 bits.  An exponential is off by 2 steps and by u |d| of its argument's
    rounding, so log S by 4 u + u sum p |d|, a result besides by its own rounding, and the
    entropy's sum by sum p |d| (5 u + u |d|)."""
    lp, en, words, best = got
    rows, vocab = x.shape
    y = torch.where(x.isnan(), -math.inf, x.double())
    m = y.amax(1, keepdim=True)
    d = torch.where(y == m, 0.0, y - m).clamp(min=-1000)
    none = (m == -math.inf)[:, 0]
    e = torch.where(y == -math.inf, 0.0, d.exp())
    s = e.sum(1, keepdim=True).clamp(min=1e-300)
    p = e / s
    lpr = torch.where(y == -math.inf, -math.inf, torch.where(y == m, 0.0, y - m) - s.log())
    h = torch.where(none, 0.0, -(p * torch.where(p > 0, d, 0.0)).sum(1) + s.log()[:, 0])
    spread = (p * d.abs()).sum(1)
    t1 = 4 * U + U * spread
    if en is not None:
        assert ((en.double() - h).abs() <= t1 + 5 * U * spread + U * (p * d * d).sum(1) + 2 * U * h.abs()).all()
    if tokens is not None:
        inside = (tokens >= 0) & (tokens < vocab)
        want = lpr.gather(1, tokens.long().clamp(0, vocab - 1)[:, None])[:, 0]
        want = torch.where(inside, want, -math.inf)
        fin = want.isfinite()
        assert torch.equal(lp[~fin].double(), want[~fin])
        assert ((lp.double() - want).abs() <= t1 + 2 * U * want.abs())[fin].all()
    if n_top:
        z = torch.where(x.isnan(), -math.inf, x) + 0.0
        order = torch.sort(z, dim=1, descending=True, stable=True)
        k = min(n_top, vocab)
        v, i = order.values[:, :k], order.indices[:, :k]
        miss = v == -math.inf
        assert torch.equal(words[:, :k].long(), torch.where(miss, -1, i))
        w = torch.where(miss, -math.inf, lpr.gather(1, i))
        fin = w.isfinite()
        assert torch.equal(best[:, :k].double()[~fin], w[~fin])
        assert ((best[:, :k].double() - w).abs() <= t1[:, None] + 2 * U * w.abs())[fin].all()
        assert (words[:, k:] == -1).all() and (best[:, k:] == -math.inf).all()


@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 2), (3, 5), (2, 300), (3, 1023), (2, 1024), (2, 1025), (5000, 700), (1, 2047), (1, 2048), (1, 2049), (5, 4097),
                                         (1, 50257), (64, 32000), (300, 1000), (700, 16385), (1, 151936), (9, 151936),
                                         (1, 2 ** 22)])
@pytest.mark.parametrize("n_top", [0, 1, 20, 64])
def test_logprobs(lib, torch_mod, rows, vocab, n_top):
    torch = torch_mod
    x = 3 * randn(torch, rows + vocab, rows, vocab)
    tokens = torch.randint(0, vocab, (rows,), device="cuda", dtype=torch.int32,
                           generator=torch.Generator(device="cuda").manual_seed(1))
    check_logprobs(torch, x, tokens, n_top, logprobs(lib, torch, x, tokens, n_top))


@pytest.mark.parametrize("rows,vocab", [(1, 7), (3, 900), (4, 3000), (2, 60000), (700, 20000)])
@pytest.mark.parametrize("kind", ["equal", "masked", "none", "nan", "inf", "steep", "flat", "ties", "lowest"])
def test_logprobs_of_odd_rows(lib, torch_mod, rows, vocab, kind):
    torch = torch_mod
    x = 3 * randn(torch, rows + vocab, rows, vocab)
    g = torch.Generator(device="cuda").manual_seed(2)
    if kind == "equal":
        x.fill_(1.5)
    elif kind == "masked":
        x.masked_fill_(torch.rand(rows, vocab, generator=g, device="cuda") < 0.999, -math.inf)
        x[:, 3] = 1.0
    elif kind == "none":
        x.fill_(-math.inf)
        x[0, vocab - 1] = -3.0 if rows > 1 else -math.inf
    elif kind == "nan":
        x[:, 1::3] = math.nan
    elif kind == "inf":
        x[:, vocab // 2] = math.inf
        x[0, vocab - 1] = math.inf
    elif kind == "steep":
        x *= 1e4
    elif kind == "flat":
        x *= 1e-6
    elif kind == "ties":
        x = (x * 2).round() / 2 * torch.where(x > 0, 1.0, -0.0)
    else:
        x[:, ::2] = torch.finfo(torch.float32).min
    tokens = torch.randint(-2, vocab + 2, (rows,), device="cuda", dtype=torch.int32, generator=g)
    tokens[0] = 3
    for n_top in (0, 5, 64):
        check_logprobs(torch, x, tokens, n_top, logprobs(lib, torch, x, tokens, n_top))


def test_logprobs_without_some_outputs_and_refusals(lib, torch_mod):
    torch = torch_mod
    x = randn(torch, 1, 3, 5000)
    tokens = whole(torch, [4, 4999, 0])
    full = logprobs(lib, torch, x, tokens, 4)
    lp, en, words, best = logprobs(lib, torch, x, None, 4)
    assert (lp == 7).all() and torch.equal(en, full[1]) and torch.equal(words, full[2]) and torch.equal(best, full[3])
    lp, en, _, _ = logprobs(lib, torch, x, tokens, 0, entropy=False)
    assert torch.equal(lp, full[0]) and (en == 7).all()
    memory = np.zeros(20000, np.float32)
    out, host = torch.full((64,), 7.0, device="cuda"), memory.ctypes.data
    o = out.data_ptr()

    def call(logits=x.data_ptr(), rows=3, vocab=5000, toks=tokens.data_ptr(), top=4, lp=o, en=o + 12, w=o + 24, b=o + 72):
        lib.gncx_hip_last_status()
        lib.gncx_hip_token_logprobs(logits, rows, vocab, toks, top, lp, en, w, b)

    for kw, text in ((dict(logits=host), "GPU"), (dict(toks=host), "GPU"), (dict(lp=host), "GPU"),
                     (dict(rows=10 ** 5), "past the end"), (dict(en=o + 4), "two of the outputs"),
                     (dict(w=o + 20), "two of the outputs"), (dict(b=x.data_ptr()), "overlaps an input"),
                     (dict(lp=tokens.data_ptr()), "overlaps an input"), (dict(logits=x.data_ptr() + 2), "4-byte")):
        call(**kw)
        refused(lib, text)
    assert (out == 7.0).all()
    call()
    gncx.check(lib)
    assert torch.equal(out[:3], full[0]) and torch.equal(out[18:30].view(3, 4), full[3])


def test_logprobs_captured(lib, torch_mod):
    torch = torch_mod
    x = torch.empty(3, 70001, device="cuda")
    tokens = whole(torch, [0, 70000, 5])
    outs = (torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda"),
            torch.zeros(3, 8, dtype=torch.int32, device="cuda"), torch.zeros(3, 8, device="cuda"))

    def call():
        lib.gncx_hip_token_logprobs(x.data_ptr(), 3, 70001, tokens.data_ptr(), 8, *(o.data_ptr() for o in outs))
        gncx.check(lib)

    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    lib.gncx_hip_set_stream(stream.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        lib.gncx_hip_set_stream(None)
        for i in range(4):
            x.copy_(3 * randn(torch, i, 3, 70001))
            torch.cuda.synchronize()
            graph.replay()
            eager = logprobs(lib, torch, 3 * randn(torch, 100 + i, 40, 30000), None, 4)
            torch.cuda.synchronize()
            check_logprobs(torch, x, tokens, 8, outs)
            assert eager[1].isfinite().all()
    finally:
        lib.gncx_hip_set_stream(None)


# ---- more work-groups than a launch has place for (2^32 threads) ---------------------------
def test_rope_of_2_24_rows(lib, torch_mod):
    torch, t, rows = torch_mod, Turn(torch_mod, 2), 2 ** 24 + 3
    x = randn(torch, 1, rows, 2)
    at = torch.arange(rows, dtype=torch.int32, device="cuda") % 4096
    out = torch.full_like(x, math.nan)
    lib.gncx_hip_rope_rows(x.data_ptr(), rows, 2, 1, 2, at.data_ptr(), t.ref(), 2, out.data_ptr())
    gncx.check(lib)
    want, tol = t(x.double().view(rows, 1, 2), at)
    assert ((out.double().view(rows, 1, 2) - want).abs() <= tol).all()


def test_append_of_2_25_rows(lib, torch_mod):
    """One sequence's rows in one call, and in two."""
    torch, rows, page = torch_mod, 2 ** 25 + 40, 256
    n_pages = -(-rows // page)
    q, k, v = (randn(torch, i, rows, 64) for i in range(3))
    table = torch.arange(n_pages, dtype=torch.int32, device="cuda")
    turn = Turn(torch, 64)

    def append(parts):
        codes = [torch.zeros(n_pages * page * 64, dtype=torch.uint8, device="cuda") for _ in range(2)]
        scales, out = torch.zeros(n_pages * page // 8, device="cuda"), torch.zeros_like(q)
        cache = gncx.PagedCache(codes[0].data_ptr(), codes[1].data_ptr(), scales.data_ptr(), n_pages, page, 1, 64)
        first = 0
        for n in parts:
            starts, length = whole(torch, [0, n]), whole(torch, [first])
            batch = gncx.PagedBatch(1, n, n_pages, starts.data_ptr(), length.data_ptr(), table.data_ptr())
            a = 256 * first
            lib.gncx_hip_kv_append_paged(C.byref(cache), C.byref(batch), q.data_ptr() + a, k.data_ptr() + a,
                                         v.data_ptr() + a, 1, None, 0, 0, 0, EPS, turn.ref(), out.data_ptr() + a)
            gncx.check(lib)
            first += n
        torch.cuda.synchronize()
        return *codes, scales, out

    one, two = append([rows]), append([rows // 3, rows - rows // 3])
    for a, b in zip(one, two):
        assert torch.equal(a, b)
    assert one[3].any(1).all()


@pytest.mark.parametrize("max_pages", [1, 40])
def test_attention_of_2_24_sequences_and_heads(lib, torch_mod, max_pages):
    """A wave, and a work-group, for each sequence and KV head: both more than 2^24."""
    torch, S, H, hd = torch_mod, 16500, 1024, 64
    if max_pages == 1:
        S = 65536
    p = Paged(torch, [15], [1], H=H, KV=H, hd=hd, page=16, seed=79)
    p.append(lib)
    table = torch.full((S, max_pages), int(p.table[0, 0]), dtype=torch.int32, device="cuda")
    lengths = torch.arange(S, dtype=torch.int32, device="cuda") % 16
    starts = torch.arange(S + 1, dtype=torch.int32, device="cuda")
    q = randn(torch, 80, S, H * hd)

    def attend(parts):
        out = torch.full((S, H * hd), math.nan, device="cuda")
        for lo, hi in parts:
            batch = gncx.PagedBatch(hi - lo, hi - lo, max_pages, starts.data_ptr(), lengths[lo:hi].data_ptr(),
                                    table.data_ptr())
            lib.gncx_hip_attention_paged(C.byref(p.cache), C.byref(batch), q[lo:hi].data_ptr(), H, p.scale, 0,
                                         out[lo:hi].data_ptr())
            gncx.check(lib)
        return out

    out = attend([(0, S)])
    assert out.isfinite().all()
    assert torch.equal(out, attend([(i, min(i + 7000, S)) for i in range(0, S, 7000)]))
    # the last sequence
    p.held, p.new, p.starts = [int(lengths[-1])], [1], np.arange(2, dtype=np.int32)
    p.check_attention(q=q[-1:], out=out[-1:])


@pytest.mark.parametrize("rows,n_top", [(2 ** 26 + 5, 0), (2 ** 26 + 5, 1), (2 ** 24 + 5, 33)])
def test_logprobs_of_2_26_rows(lib, torch_mod, rows, n_top):
    torch = torch_mod
    x = randn(torch, 81, rows, 2)
    tokens = torch.arange(rows, dtype=torch.int32, device="cuda") % 2
    got = logprobs(lib, torch, x, tokens, n_top)
    for i in list(range(0, rows - 2 ** 22, 2 ** 23)) + [rows - 2 ** 22]:
        n = slice(i, i + 2 ** 22)
        check_logprobs(torch, x[n], tokens[n], n_top, tuple(t[n] for t in got))


# ---- a run of them together: the decode driver --------------------------------------------
LOGITS = 1e-3  # the bar of this driver's logits between its batched and its one-token calls (relative L2)


def small_decoder(lib, torch, hd, max_seq=200, **kw):
    import gncx_amd.decode as dec
    shape = dec.Qwen3Shape(n_layers=2, embed=256, n_heads=4, n_kv=2, head_dim=hd, ffn=512, vocab=600)
    model = dec.build_model(torch, shape, seed=7)
    return dec, model, dec.Decoder(lib, torch, model, max_seq=max_seq, fused=True, **kw)


def watch(dec, d, monkeypatch, yarn=None):
    """Every append and attention of d.generate_batch against the formulas, on what they were
    given; the logits it answered from."""
    torch, seen = d.torch, []

    class Watched(dec.PagedSequences):
        def attention(self, l, q, k, v, out, scale):
            s, m = self.m.shape, self.m
            p = object.__new__(Paged)
            p.torch, p.held, p.new, p.H, p.KV, p.hd, p.page = torch, self.lengths, self.counts, s.n_heads, s.n_kv, \
                s.head_dim, self.page
            p.table, p.max_pages, p.n_pages, p.scale = self.table.cpu().numpy(), self.max_pages, self.n_pages, scale
            p.starts = np.concatenate([[0], np.cumsum(self.counts)])
            shape = self.n_pages, s.n_kv, self.page // BLOCK
            p.k, p.v = self.k[l].view(*shape, BLOCK, s.head_dim), self.v[l].view(*shape, s.head_dim, BLOCK)
            p.scales = self.scales[l].view(*shape, 2)
            at = [m.off(f"blk.{l}.attn_{n}_norm.weight") for n in "qk"]
            p.gamma = [m.blob[a:a + 4 * s.head_dim].view(torch.float32) for a in at]
            p.q, p.kr, p.vr, p.out = q.clone(), k, v, q
            before = state(p)
            super().attention(l, q, k, v, out, scale)
            turn = Turn(torch, s.head_dim, base=s.rope_base)
            if yarn:
                turn.freqs, turn.magnitude = self.freqs, self.rotation.magnitude
                assert math.isclose(turn.magnitude, 0.1 * math.log(yarn) + 1, rel_tol=1e-6)
            check_append(p, before, turn, 1)
            p.check_attention(q=q, out=out)

    answers = d._logprobs

    def logprobs_of(logits, tokens=None, n_top=0):
        got = answers(logits, tokens, n_top)
        seen.append(logits.clone())
        check_logprobs(torch, logits, None, n_top, (None, None, got[2], got[3]))
        return got

    monkeypatch.setattr(dec, "PagedSequences", Watched)
    monkeypatch.setattr(d, "_logprobs", logprobs_of)
    return seen


@pytest.mark.parametrize("hd,page,at_once,scaling", [(64, 16, 50, False), (128, 64, 4096, False), (256, 32, 1, False),
                                                     (128, 32, 70, True)])
def test_generate_batch(lib, torch_mod, monkeypatch, hd, page, at_once, scaling):
    """Each operator of the run on its own inputs, and the run's logits against a decoder
    that steps along each sequence alone over fp32 caches: a code is off by 0.026 of its
    value (root mean square of 2^-4 at most), which moves scores of N(0, 1) and outputs as
    much, under 0.1 of the logits in two layers; those of another place are sqrt(2) away."""
    torch = torch_mod
    dec, model, d = small_decoder(lib, torch, hd)
    rng = np.random.default_rng(hd)
    lens, n_new = ([1, 3, 2] if at_once == 1 else [1, 40, 7, 130, 16]), 6
    prompts = [rng.integers(0, 600, n).tolist() for n in lens]
    kw = dict(n_top=3, page=page, rows_at_once=at_once)
    if scaling:
        kw["scaling"] = dict(scaling=gncx.ROPE_YARN, factor=4.0, trained_context=64)
    with monkeypatch.context() as patch:
        seen = watch(dec, d, patch, 4.0 if scaling else None)
        got = d.generate_batch(prompts, n_new, **kw)
    assert [len(ids) for ids, _, _ in got] == [n_new] * len(lens) and len(seen) == n_new
    ref = dec.Decoder(lib, torch, model, max_seq=200, fused=True)
    for i, (ids, lps, tops) in enumerate(got):
        if not scaling:
            want = ref.prefill(prompts[i])
        for j, (t, lp, top) in enumerate(zip(ids, lps, tops)):
            assert top[0] == (t, lp) and len(top) == 3
            x = seen[j][i].double()
            assert x[t] == x.max() and abs(lp - float(x[t] - x.logsumexp(0))) < 1e-5
            if not scaling:
                assert (x - want.double()).norm() < 0.3 * want.double().norm(), (i, j)
                want = ref.forward_token(t, lens[i] + j)
    # the second sequence's second token as the end: the same up to it, wherever it comes
    end = got[1][0][1]
    with monkeypatch.context() as patch:
        watch(dec, d, patch, 4.0 if scaling else None)
        ended = d.generate_batch(prompts, n_new, end=end, **kw)
    first = min(ids.index(end) for ids, _, _ in got if end in ids)
    for (ids, lps, tops), (all_ids, all_lps, all_tops) in zip(ended, got):
        n = first + 1  # (behind it the passes have other rows)
        assert ids[:n] == all_ids[:n] and lps[:n] == all_lps[:n] and tops[:n] == all_tops[:n]
        assert len(ids) == len(lps) == len(tops) == (ids.index(end) + 1 if end in ids else n_new)
    assert [len(t) for _, _, t in d.generate_batch(prompts[:2], 2)] == [2, 2]


@pytest.mark.parametrize("hd,n", [(64, 2), (128, 50), (64, 1030)])
def test_score(lib, torch_mod, hd, n):
    torch = torch_mod
    dec, model, d = small_decoder(lib, torch, hd, max_seq=1100)
    ids = np.random.default_rng(n).integers(0, 600, n).tolist()
    lps, ents, tops = d.score(ids, n_top=2)
    assert len(lps) == len(ents) == len(tops) == n - 1
    ref = dec.Decoder(lib, torch, model, max_seq=1100, fused=True)
    for i in range(n - 1):
        x = ref.forward_token(ids[i], i).double()
        if 3 < i < n - 8:
            continue
        # logits off by the bar: a log probability by twice it; the entropy's slope in a
        # logit is p (log p + H), so it by (log V + H) times it
        bar = float(LOGITS * x.norm())
        p = x.log_softmax(0)
        assert abs(lps[i] - float(p[ids[i + 1]])) <= 2 * bar + 1e-5
        assert abs(ents[i] + float((p.exp() * p).sum())) <= 2 * math.log(600) * bar + 1e-5
        for t, lp in tops[i]:
            assert abs(lp - float(p[t])) <= 2 * bar + 1e-5
        assert tops[i][0][1] >= float(p.max()) - 2 * bar - 1e-5
    assert d.score(ids)[2] == [[]] * (n - 1)
    gncx.check(lib)
